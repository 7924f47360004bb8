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
    float inverse;  // 1 / (s lift), 0 for a row that is not finite
};

/// From the bits of the row's largest magnitude (as integers they are ordered
/// like the magnitudes, infinity and NaN last).
template <cf_cache_format kFormat>
__device__ __forceinline__ RowScale row_scale(uint32_t absmax_bits) {
    RowScale r;
    const float s = __uint_as_float(absmax_bits) * (1.0f / kLargestCode<kFormat>);
    r.s = s > 0.0f ? s : 1.0f;
    r.lift = r.s < 0x1p-80f ? 0x1p100f : 1.0f;
    r.lifted = r.s * r.lift;
    r.inverse = 1.0f / r.lifted;
    if (absmax_bits >= 0x7F800000u) {
        r.s = __uint_as_float(0x7FC00000u);
        r.inverse = 0.0f;
    }
    return r;
}

/// x / s rounded to odd, x finite.
__device__ __forceinline__ float odd_quotient(float x, const RowScale& r) {
    const float y = x * r.lift;
    const float q0 = y * r.inverse;
    const float q = fmaf(fmaf(-q0, r.lifted, y), r.inverse, q0);  // within a unit in the last place
    const float rest = fmaf(-q, r.lifted, y);
    const uint32_t bits = __float_as_uint(q);
    // A remainder of the other sign than q: q lies past x / s.
    const uint32_t back = (__float_as_uint(rest) ^ bits) >> 31;
    return rest == 0.0f ? q : __uint_as_float((bits - back) | 1u);
}

/// Four codes, the first in the low byte. Values of a row whose scale is NaN may
/// be anything.
template <cf_cache_format kFormat>
__device__ __forceinline__ uint32_t pack4_codes(const float* x, const RowScale& r) {
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // Past the largest code only where s is subnormal and so rounded far.
        const float top = kLargestCode<kFormat>;
        q[i] = r.inverse == 0.0f ? 0.0f : __builtin_amdgcn_fmed3f(odd_quotient(x[i], r), -top, top);
        // Zeros keep their sign (the fma above gives +0 for -0).
        if constexpr (kFormat == CF_CACHE_E4M3) q[i] = r.inverse == 0.0f ? 0.0f : __builtin_copysignf(q[i], x[i]);
    }
    if constexpr (kFormat == CF_CACHE_INT8) {
        // |q| < 2^22: the sum's spacing is 1, so the add rounds q to an integer,
        // ties to even, and leaves it in the low byte.
        uint32_t t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = __float_as_uint(q[i] + 12582912.0f);  // 3 2^22
        const uint32_t lo = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(t[3], t[2], 0x0c0c0400u);
        return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    } else {
        int packed = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        packed = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], packed, true);
        return static_cast<uint32_t>(packed);
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
