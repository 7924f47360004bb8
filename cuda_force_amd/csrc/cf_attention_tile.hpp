// Tiles of attention over a cache on the matrix cores, for the kernels that
// form scores transposed, S^T = K Q^T: a lane holds one query row and several
// tokens, and the probabilities are in place as the B operand of O^T += V^T P^T.
// Also the copies to LDS and waits that such kernels order by hand.
#pragma once

#include <type_traits>

#include "cf_common.hpp"
#include "cf_lds_dma.hpp"

namespace cf {
namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
typedef __attribute__((address_space(3))) uint8_t lds_u8_t;

/// LDS byte address of a pointer into shared memory.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8_t*)(const_cast<void*>(p))));
}

/// 16 bytes per lane from `from` (a lane's own address) to LDS bytes
/// dst + 16 lane. In inline assembly for the reason given at dma16_m0; it has no
/// register output.
__device__ __forceinline__ void copy16_to_lds(const void* from, uint32_t dst) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, off"
                 :
                 : "v"(from), "{m0}"(__builtin_amdgcn_readfirstlane(dst))
                 : "memory");
}

/// The same from a base that all lanes share, and each lane's offset from it.
__device__ __forceinline__ void copy16_to_lds(const uint8_t* base, uint32_t offset, uint32_t dst) {
    const uint64_t address = reinterpret_cast<uint64_t>(base);
    const uint64_t low = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(address)));
    const uint64_t high = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(address >> 32)));
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(offset), "s"(high << 32 | low), "{m0}"(__builtin_amdgcn_readfirstlane(dst))
                 : "memory");
}

/// Four copies like the first, to LDS bytes dst + kCopyBytes n + 16 lane: the
/// instruction's offset counts for both addresses, so the sources are given less
/// kCopyBytes n.
constexpr int kCopyBytes = 16 * kWaveSize;
__device__ __forceinline__ void copy16x4_to_lds(const uint8_t* from0, const uint8_t* from1, const uint8_t* from2,
                                                const uint8_t* from3, uint32_t dst) {
    asm volatile(
        "s_nop 4\n\tglobal_load_lds_dwordx4 %0, off\n\tglobal_load_lds_dwordx4 %1, off offset:%5\n\t"
        "global_load_lds_dwordx4 %2, off offset:%6\n\tglobal_load_lds_dwordx4 %3, off offset:%7"
        :
        : "v"(from0), "v"(from1), "v"(from2), "v"(from3), "{m0}"(__builtin_amdgcn_readfirstlane(dst)), "n"(kCopyBytes),
          "n"(2 * kCopyBytes), "n"(3 * kCopyBytes)
        : "memory");
}

/// Waits until at most n vector-memory operations of the wave are in flight.
template <int n>
__device__ __forceinline__ void wait_vm() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(n));
    asm volatile("" ::: "memory");
}

/// Waits for the wave's LDS operations.
__device__ __forceinline__ void wait_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xF | (7 << 4) | (0 << 8) | (3 << 14));
    asm volatile("" ::: "memory");
}

/// The larger of each lane's value and that of the lanes with the same place
/// in the other groups of kGroup (32 or 16) lanes, exchanged in registers.
template <int kGroup>
__device__ __forceinline__ float groups_max(float v) {
    if constexpr (kGroup == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

/// What depends on the cache's type: rows and tokens of a tile, fragments,
/// products. kD: head size rounded up to 64, 128 or 256.
template <typename T, int kD>
struct Tile {
    static constexpr bool kWide = sizeof(T) == 4;
    static constexpr int kRows = kWide ? 16 : 32;    // query rows per wave
    static constexpr int kTokens = kWide ? 16 : 32;  // tokens per tile
    static constexpr int kPerVec = 16 / static_cast<int>(sizeof(T));
    static constexpr int kRowBytes = kD * static_cast<int>(sizeof(T));
    static constexpr int kChunks = kRowBytes / 16;
    static constexpr int kBytes = kTokens * kRowBytes;            // K or V of one tile
    static constexpr int kCopies = kBytes / (16 * kWaveSize);     // wave-wide copies of it
    static constexpr int kScores = kRows * kTokens / kWaveSize;   // scores per lane
    static constexpr int kAcc = kRows * kD / kWaveSize;           // output values per lane
    static constexpr int kOutPitch = kD + 4;                      // floats per row of the output area
    /// A row's maximum may lag the true one by up to kLag (base 2): sums and
    /// outputs are rescaled only when it would lag more. Probabilities, and with
    /// them weighted values and sums, are kept 2^kLift times as large: fp16
    /// holds them up to 2^15, so one is a full number down to 2^-27 of the row's
    /// largest, and off by at most 2^-38 of that below (kept at most 1, one
    /// below 2^-25 was 0: 32767 tokens 17.5 nats behind a leading one without
    /// a value gave 0 for 8.2e-4). A lag of 2 against 8 costs nothing, none at
    /// all 5% (128 sequences behind 32768 tokens in fp16: 125, 125 and 131 us).
    static constexpr float kLag = std::is_same<T, f16_t>::value ? 2.0f : 8.0f;
    static constexpr float kLift = std::is_same<T, f16_t>::value ? 13.0f : 0.0f;

    /// Order of the 16-byte pieces of a K row: a fragment read takes the same
    /// piece of 16 rows.
    __device__ __forceinline__ static int k_swizzle(int row) {
        return kChunks >= 16 ? (row & 15) : ((row >> 1) & 7);
    }
    /// And of a V row: a transposed (fp32: plain) read takes 64 bytes of four
    /// rows, neighbours (fp32: four apart).
    __device__ __forceinline__ static int v_swizzle(int row) {
        if constexpr (kWide) return row & 12;
        return kChunks >= 16 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
    }

    using Query = std::conditional_t<kWide, f32x4_t, u32x4_t>;
    static constexpr int kQueries = kWide ? kD / 16 : kD / 16;  // 16-byte query pieces per lane
    using Score = std::conditional_t<kWide, f32x4_t, f32x16_t>;

    /// Query row of a lane, and its half or quarter.
    __device__ __forceinline__ static int row_of(int lane) { return lane & (kRows - 1); }
    __device__ __forceinline__ static int part_of(int lane) { return lane / kRows; }
    /// First dim of a lane's query piece u.
    __device__ __forceinline__ static int query_dim(int u, int lane) {
        return 16 * u + kPerVec * part_of(lane);
    }
    /// A lane's score i is token 4 part + token_of(i) of the tile.
    __device__ __forceinline__ static constexpr int token_of(int i) { return kWide ? i : 8 * (i >> 2) + (i & 3); }
    /// Dim of a lane's output value i: four neighbours from each i % 4 == 0.
    __device__ __forceinline__ static int dim_of(int i, int lane) {
        if constexpr (kWide) return 16 * (i >> 2) + 4 * part_of(lane) + (i & 3);
        return 32 * (i >> 4) + 8 * ((i >> 2) & 3) + 4 * part_of(lane) + (i & 3);
    }

    __device__ __forceinline__ static Score scores(const uint8_t* k, const Query (&q)[kQueries], int lane) {
        Score s;
#pragma unroll
        for (int i = 0; i < kScores; ++i) s[i] = 0.0f;
        const int row = lane & (kTokens - 1);
        const int sw = k_swizzle(row);
#pragma unroll
        for (int u = 0; u < kQueries; ++u) {
            // 16-bit: 16 dims a step, 8 per half; fp32: 16 dims, 4 per quarter.
            const int piece = (kWide ? 4 : 2) * u + part_of(lane);
            const u32x4_t raw = *reinterpret_cast<const u32x4_t*>(k + row * kRowBytes + ((piece ^ sw) << 4));
            if constexpr (kWide) {
                const f32x4_t kk = __builtin_bit_cast(f32x4_t, raw);
#pragma unroll
                for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[e], q[u][e], s, 0, 0, 0);
            } else if constexpr (std::is_same<T, bf16_t>::value) {
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, raw),
                                                            __builtin_bit_cast(bf16x8_t, q[u]), s, 0, 0, 0);
            } else {
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, raw),
                                                           __builtin_bit_cast(f16x8_t, q[u]), s, 0, 0, 0);
            }
        }
        return s;
    }

    /// acc += V^T P^T for the tile's probabilities p.
    __device__ __forceinline__ static void values(const uint8_t* v, const Score& p, Score (&acc)[kAcc / kScores],
                                                  int lane) {
        if constexpr (kWide) {
            const int g = lane >> 4;
            const int j = lane & 15;
#pragma unroll
            for (int b = 0; b < kD / 16; ++b) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = 4 * g + e;
                    const int piece = (4 * b + (j >> 2)) ^ v_swizzle(row);
                    const float x = *reinterpret_cast<const float*>(v + row * kRowBytes + (piece << 4) + (j & 3) * 4);
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, p[e], acc[b], 0, 0, 0);
                }
            }
        } else {
            const int half = lane >> 5;
            const int quad = (lane >> 4) & 1;
            const int j = lane & 15;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t bits[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (std::is_same<T, bf16_t>::value) {
                        bits[e] = f32x2_to_bf16x2_bits(p[8 * u + 2 * e], p[8 * u + 2 * e + 1]);
                    } else {
                        bits[e] = Storage<T>::to_bits2(p[8 * u + 2 * e], p[8 * u + 2 * e + 1]);
                    }
                }
                const u32x4_t pb = {bits[0], bits[1], bits[2], bits[3]};
                // Tokens 16 u + 4 half .. + 3, then the same 8 further on.
                const int row = 16 * u + 4 * half + (j >> 2);
                const int sw = v_swizzle(row);
#pragma unroll
                for (int b = 0; b < kD / 32; ++b) {
                    const int piece = (4 * b + 2 * quad + ((j & 3) >> 1)) ^ sw;
                    const uint8_t* at = v + row * kRowBytes + (piece << 4) + (j & 1) * 8;
                    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4_t*)(lds_u8_t*)(const_cast<uint8_t*>(at)));
                    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4_t*)(lds_u8_t*)(const_cast<uint8_t*>(at + 8 * kRowBytes)));
                    const auto vv = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    if constexpr (std::is_same<T, bf16_t>::value) {
                        acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vv),
                                                                         __builtin_bit_cast(bf16x8_t, pb), acc[b], 0,
                                                                         0, 0);
                    } else {
                        acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, vv),
                                                                        __builtin_bit_cast(f16x8_t, pb), acc[b], 0, 0,
                                                                        0);
                    }
                }
            }
        }
    }
};

}  // namespace
}  // namespace cf
