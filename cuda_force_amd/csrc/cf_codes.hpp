// Rows held in 8 bits: a scale per row and a code per value, int8 or OCP
// e4m3fn, for caches and for the int8 product's activations.
//
//   s = absmax (1 / M), both in fp32 (M = 127 or 448, the largest code); 1 where
//       that is 0; NaN where the row holds a NaN or an infinity
//   code = the code nearest to x / s, ties to the even code, at most M either
//       way; 0 where s is NaN
//
// Nearest is meant exactly: a rounded quotient can fall on the middle between
// two codes where x / s itself does not (81 of 64000 e4m3 codes of bf16
// normals would differ), so the quotient is rounded to odd: its last bit is set
// where it is not exact, and rounding that to a code's few bits gives what
// rounding x / s would. The remainder x - q s has the sign of what is missing
// (one fma, rounded once, and scales are kept in the normal range for it).
#pragma once

#include "cf_common.hpp"

namespace cf {

/// The larger code's magnitude: of int8 and of e4m3fn.
template <cf_cache_format kFormat>
constexpr float kLargestCode = kFormat == CF_CACHE_INT8 ? 127.0f : 448.0f;

/// What the codes of one row are made with. x is multiplied by `lift` first, a
/// power of two that keeps quotients and remainders of rows below 2^-80 in the
/// normal range (1 else).
struct RowScale {
    float s;        // as stored
    float lift;
    float lifted;   // s lift
    float inverse;  // 1 / (s lift), to a unit in the last place
    uint32_t keep;  // of the codes' bits: none for a row that is not finite
};

/// From the bits of the row's largest magnitude (as integers they are ordered
/// like the magnitudes, infinity and NaN last).
template <cf_cache_format kFormat>
__device__ __forceinline__ RowScale row_scale(uint32_t absmax_bits) {
    RowScale r;
    const float s = __uint_as_float(absmax_bits) * (1.0f / kLargestCode<kFormat>);
    const bool finite = absmax_bits < 0x7F800000u;
    const float used = s > 0.0f ? s : 1.0f;
    r.lift = used < 0x1p-80f ? 0x1p100f : 1.0f;
    r.lifted = used * r.lift;
    r.inverse = __builtin_amdgcn_rcpf(r.lifted);
    r.s = finite ? used : __uint_as_float(0x7FC00000u);
    r.keep = finite ? 0xFFFFFFFFu : 0u;
    return r;
}

/// x / s rounded to odd, x finite.
template <bool kLift>
__device__ __forceinline__ float odd_quotient(float x, const RowScale& r) {
    const float y = __builtin_fabsf(kLift ? x * r.lift : x);
    const float q0 = y * r.inverse;
    const float q = fmaf(fmaf(-q0, r.lifted, y), r.inverse, q0);  // within a unit in the last place
    const float rest = fmaf(-q, r.lifted, y);
    // Below 0: q lies past the quotient.
    const uint32_t odd = (__float_as_uint(q) - (__float_as_uint(rest) >> 31)) | 1u;
    return __builtin_copysignf(rest == 0.0f ? q : __uint_as_float(odd), x);
}

/// Whether every row of the wave goes without a lift (uniform).
__device__ __forceinline__ bool ordinary_rows(const RowScale& r) {
    return __builtin_amdgcn_ballot_w64(r.lift != 1.0f) == 0;
}

/// Four codes, the first in the low byte.
template <cf_cache_format kFormat, bool kLift>
__device__ __forceinline__ uint32_t pack4_codes(const float* x, const RowScale& r) {
    float q[4];
    if constexpr (kFormat == CF_CACHE_INT8) {
        // |q| < 2^22: the spacing of sums with 3 2^22 is 1, so the add rounds q to an
        // integer, ties to even, and leaves it in the low byte.
        constexpr float kShift = 12582912.0f;
        bool near = kLift;
        if constexpr (!kLift) {
            // Rounding a quotient that is off by up to 127 2^-23 = 1.6e-5 is right unless
            // x lies next to the middle of two codes, which its distance from the code
            // shows: about one in 2^13 does.
            const float middle = 0.49995f * r.s;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                q[i] = fmaf(x[i], r.inverse, kShift);
                near = near || __builtin_fabsf(fmaf(kShift - q[i], r.s, x[i])) > middle;
            }
            near = __builtin_amdgcn_ballot_w64(near) != 0;
        }
        if (near) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // Past the largest code only where s is subnormal and so rounded far.
                const float odd = odd_quotient<kLift>(x[i], r);
                q[i] = (kLift ? __builtin_amdgcn_fmed3f(odd, -127.0f, 127.0f) : odd) + kShift;
            }
        }
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(q[1]), __float_as_uint(q[0]), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(q[3]), __float_as_uint(q[2]), 0x0c0c0400u);
        return __builtin_amdgcn_perm(hi, lo, 0x05040100u) & r.keep;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = odd_quotient<kLift>(x[i], r);
            if constexpr (kLift) q[i] = __builtin_amdgcn_fmed3f(q[i], -448.0f, 448.0f);
        }
        int packed = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        packed = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], packed, true);
        return static_cast<uint32_t>(packed) & r.keep;
    }
}

/// The largest magnitude's bits of 16 bytes of T.
template <typename T>
__device__ __forceinline__ uint32_t largest16(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t top = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) top = MaxU32::apply(top, w[i] & 0x7FFFFFFFu);
        return top;
    } else {
        // Two at a time: 16-bit magnitudes are ordered like their bits, too.
        typedef uint16_t u16x2_v __attribute__((ext_vector_type(2)));
        u16x2_v both = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            both = __builtin_elementwise_max(both, __builtin_bit_cast(u16x2_v, w[i] & 0x7FFF7FFFu));
        }
        return __float_as_uint(Storage<T>::from_bits(both[0] > both[1] ? both[0] : both[1]));
    }
}

/// The numbers that four codes stand for, without the scale.
template <cf_cache_format kFormat>
__device__ __forceinline__ void unpack4_codes(uint32_t w, float* x) {
    if constexpr (kFormat == CF_CACHE_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
    } else {
        typedef float f32x2_v __attribute__((ext_vector_type(2)));
        const f32x2_v lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
        const f32x2_v hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
        x[0] = lo[0];
        x[1] = lo[1];
        x[2] = hi[0];
        x[3] = hi[1];
    }
}

inline bool valid_format(cf_cache_format f) {
    return f == CF_CACHE_PLAIN || f == CF_CACHE_INT8 || f == CF_CACHE_E4M3;
}

}  // namespace cf
