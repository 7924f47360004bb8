// Products of 8-bit integers, with a scale for each row of the one and each row
// of the other operand, and the row-wise quantisation that makes the operand of
// activations:
//
//   y[i, j] = T(x_scales[i] w_scales[j] sum_k x[i, k] w[j, k] + bias[j])
//
// x [m, k] and w [n, k] are int8, both dense along k (w is a torch Linear's
// weight), sums exact in int32.
//
// Few rows are bound by w, which is read once: its rows go from memory straight to
// the matrix cores, 16 of them a workgroup, whose waves split k (8 rows by 11008
// columns of 4096: 14.1 us, 3.2 TB/s; sending the next loads ahead of the products
// changed nothing). Middling batches are bound by the steps of the loop over k,
// each a barrier, copies, LDS reads and a short chain of products: small tiles,
// and two groups of waves on one, give the CUs enough to do beside them (333 x
// 4096 x 4096: 15 us by kernel time, 11 TB/s from L2 to LDS at 15% of the matrix
// cores' rate; neither a fifth stage of LDS nor steps in another order for every
// tile changed anything). Large ones are bound by the matrix cores and the
// power they draw: 8192 x 4096 x 4096 takes 115 to 128 us by the card, 2.1 to 2.4 POP/s, with
// the matrix cores 56% busy at 1.6 to 1.8 GHz.
//
// The quantiser is bound by memory: a row is read once and held in registers
// (8192 rows of 4096 in bf16: 17.8 us, 5.7 TB/s).
#include "cf_codes.hpp"
#include "cf_common.hpp"
#include "cf_lds_dma.hpp"

#include <type_traits>

namespace cf {
namespace {

typedef int i32x4v_t __attribute__((ext_vector_type(4)));
typedef int i32x16v_t __attribute__((ext_vector_type(16)));
typedef float f32x4v_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8_t;

// ---- quantisation of rows ------------------------------------------------------

struct RowsArgs {
    const void* x;
    int8_t* codes;
    float* scales;
    int64_t rows;
    int64_t cols;
    int64_t stride;
};

constexpr int kRowThreads = 256;

/// kVecs 16-byte vectors per thread of kPerRow; the row stays in registers.
template <typename T, int kPerRow, int kVecs>
__global__ __launch_bounds__(kPerRow < kRowThreads ? kRowThreads : kPerRow) void quantize_rows_kernel(RowsArgs a) {
    constexpr int kThreads = kPerRow < kRowThreads ? kRowThreads : kPerRow;
    constexpr int kRows = kThreads / kPerRow;
    constexpr int kWaves = kPerRow / kWaveSize;
    constexpr int kPer = Storage<T>::kPerVec;
    __shared__ uint32_t tops[kWaves];
    const int tid = static_cast<int>(threadIdx.x);
    const int part = tid % kPerRow;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + tid / kPerRow; row < a.rows;
         row += static_cast<int64_t>(gridDim.x) * kRows) {
        const T* x = static_cast<const T*>(a.x) + row * a.stride;
        float f[kVecs][kPer];
        uint4 raw[kVecs];
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const int d = (v * kPerRow + part) * kPer;
            raw[v] = d < a.cols ? *reinterpret_cast<const uint4*>(x + d) : make_uint4(0, 0, 0, 0);
        }
        uint32_t top = 0;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            top = MaxU32::apply(top, largest16<T>(raw[v]));
            unpack16<T>(raw[v], f[v]);
        }
        top = group_reduce_u32<16, MaxU32>(top);
        // Bits of finite magnitudes, infinities and NaN: never negative as integers.
        int wave_top = __builtin_amdgcn_readlane(static_cast<int>(top), 0);
#pragma unroll
        for (int l = 16; l < kWaveSize; l += 16) {
            const int o = __builtin_amdgcn_readlane(static_cast<int>(top), l);
            wave_top = o > wave_top ? o : wave_top;
        }
        top = static_cast<uint32_t>(wave_top);
        if constexpr (kWaves > 1) {  // a row per workgroup: all its threads are here
            if ((tid & (kWaveSize - 1)) == 0) tops[tid / kWaveSize] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = MaxU32::apply(top, tops[w]);
            __syncthreads();
        }
        const RowScale s = row_scale<CF_CACHE_INT8>(top);
        const bool ordinary = ordinary_rows(s);
        int8_t* to = a.codes + row * a.cols;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const int d = (v * kPerRow + part) * kPer;
            uint32_t w[kPer / 4];
#pragma unroll
            for (int e = 0; e < kPer / 4; ++e) {
                w[e] = ordinary ? pack4_codes<CF_CACHE_INT8, false>(f[v] + 4 * e, s)
                                : pack4_codes<CF_CACHE_INT8, true>(f[v] + 4 * e, s);
            }
            if (d < a.cols) {
                if constexpr (kPer == 8) {
                    *reinterpret_cast<uint2*>(to + d) = make_uint2(w[0], w[1]);
                } else {
                    *reinterpret_cast<uint32_t*>(to + d) = w[0];
                }
            }
        }
        if (part == 0) a.scales[row] = s.s;
    }
}

/// Rows of any length and alignment, read twice.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void quantize_rows_any_kernel(RowsArgs a) {
    constexpr int kWaves = kRowThreads / kWaveSize;
    __shared__ uint32_t tops[kWaves];
    const int tid = static_cast<int>(threadIdx.x);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.stride;
        uint32_t top = 0;
        for (int64_t d = tid; d < a.cols; d += kRowThreads) {
            top = MaxU32::apply(top, __float_as_uint(Storage<T>::load(x + d)) & 0x7FFFFFFFu);
        }
#pragma unroll
        for (int d = 1; d < kWaveSize; d <<= 1) {
            top = MaxU32::apply(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
        }
        if ((tid & (kWaveSize - 1)) == 0) tops[tid / kWaveSize] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = MaxU32::apply(top, tops[w]);
        __syncthreads();
        const RowScale s = row_scale<CF_CACHE_INT8>(top);
        for (int64_t d = tid; d < a.cols; d += kRowThreads) {
            const float f[4] = {Storage<T>::load(x + d), 0.0f, 0.0f, 0.0f};
            a.codes[row * a.cols + d] = static_cast<int8_t>(pack4_codes<CF_CACHE_INT8, true>(f, s));
        }
        if (tid == 0) a.scales[row] = s.s;
    }
}

template <typename T>
void launch_rows(const RowsArgs& a, hipStream_t stream) {
    constexpr int kPer = Storage<T>::kPerVec;
    const int64_t vecs = a.cols / kPer;
    // (Rows beyond a launch's workgroups go in turn.)
    auto capped = [](int64_t n, int threads = kRowThreads) {
        const int64_t most = UINT32_MAX / threads;
        return dim3(static_cast<unsigned>(n < most ? n : most));
    };
    const bool vectors = a.cols % kPer == 0 && host_aligned(a.x, 16) && a.stride % kPer == 0 &&
                         host_aligned(a.codes, kPer) && vecs <= 1024 * 8;
    if (!vectors) {
        launch(quantize_rows_any_kernel<T>, capped(a.rows), dim3(kRowThreads), 0, stream, a);
        return;
    }
    // A wave per row where rows are short and enough to fill the GPU with that (4096
    // rows of 1024 in bf16 6.6 us, a workgroup per row 7.8; 2048 of them 6.4 either
    // way; 4096 rows of 4096 would take 13.7 us against 12.3).
    if (vecs <= 64 * 2 && a.rows >= 2048) {
        const dim3 grid = capped(ceil_div<int64_t>(a.rows, 4));
        auto* kernel = vecs <= 64 ? quantize_rows_kernel<T, 64, 1> : quantize_rows_kernel<T, 64, 2>;
        launch(kernel, grid, dim3(kRowThreads), 0, stream, a);
    } else if (vecs <= 256 * 8) {
        auto* kernel = vecs <= 256    ? quantize_rows_kernel<T, 256, 1>
                       : vecs <= 512  ? quantize_rows_kernel<T, 256, 2>
                       : vecs <= 1024 ? quantize_rows_kernel<T, 256, 4>
                                      : quantize_rows_kernel<T, 256, 8>;
        launch(kernel, capped(a.rows), dim3(256), 0, stream, a);
    } else {
        launch(quantize_rows_kernel<T, 1024, 8>, capped(a.rows, 1024), dim3(1024), 0, stream, a);
    }
}

// ---- products -------------------------------------------------------------------

struct Int8Args {
    const int8_t* x;
    const int8_t* w;
    const float* x_scales;
    const float* w_scales;
    const void* bias;
    void* y;
    int m;
    int n;
    int k;
    int tiles_m;
    int tiles_n;
};

constexpr int kStep = 128;  // bytes of k per stage: a line of every row

/// Order of the 16-byte pieces of a row of 128: a fragment read takes the same
/// piece of 32 rows, eight rows and those 24 further on (or eight apart) at a
/// time, which bit 3 of the row sends to different halves.
__device__ __forceinline__ int swizzle(int row) { return (row & 7) ^ ((row >> 3) & 1); }

/// One result: as the header has it.
__device__ __forceinline__ float result(int sum, float xs, float ws, float bias) {
    return fmaf(static_cast<float>(sum) * xs, ws, bias);
}

template <typename T>
__device__ __forceinline__ float bias_at(const Int8Args& a, int j) {
    return a.bias != nullptr ? Storage<T>::load(static_cast<const T*>(a.bias) + j) : 0.0f;
}

/// Four neighbouring columns j .. j + 3 of row i.
template <typename T>
__device__ __forceinline__ void store4(const Int8Args& a, int i, int j, const int (&sum)[4], float xs, bool vectors) {
    T* y = static_cast<T*>(a.y) + static_cast<int64_t>(i) * a.n + j;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int col = j + e < a.n ? j + e : a.n - 1;
        v[e] = result(sum[e], xs, a.w_scales[col], bias_at<T>(a, col));
    }
    if (vectors && j + 3 < a.n) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            *reinterpret_cast<uint2*>(y) = make_uint2(Storage<T>::to_bits2(v[0], v[1]), Storage<T>::to_bits2(v[2], v[3]));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (j + e < a.n) Storage<T>::store(y + e, v[e]);
        }
    }
}

/// kBM x kBN results per workgroup, kWM x kWN per wave, kStages stages of 128
/// bytes of k in LDS. The product is formed transposed (w the first operand), so
/// a lane holds runs of four columns of one row. With two groups each of them has
/// the whole tile, stages of its own and every other 128 bytes of k, and the
/// second hands its sums over at the end: half as many barriers, whose steps are
/// what a workgroup that is alone on its CU waits for.
template <typename T, int kBM, int kBN, int kWM, int kWN, int kStages, int kGroups>
__global__ __launch_bounds__(kGroups * (kBM / kWM) * (kBN / kWN) * kWaveSize) void matmul_int8_kernel(Int8Args a) {
    constexpr int kWavesM = kBM / kWM;
    constexpr int kWavesN = kBN / kWN;
    constexpr int kWaves = kWavesM * kWavesN;
    // Copies of 1 KiB per wave and stage; the last waves may have none.
    constexpr int kCopies = ((kBM + kBN) / 8 + kWaves - 1) / kWaves;
    constexpr int kStageBytes = (kBM + kBN) * kStep;
    static_assert((kBM + kBN) / 8 % kCopies == 0 && kBM / 8 % kCopies == 0, "a wave copies rows of one operand");
    __shared__ __attribute__((aligned(16))) uint8_t lds[kGroups * kStages * kStageBytes];
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63;
    const int group = kGroups == 1 ? 0 : __builtin_amdgcn_readfirstlane((tid >> 6) / kWaves);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) - group * kWaves;
    uint8_t* const own = lds + group * kStages * kStageBytes;
    int tm;
    int tn;
    tile_of(static_cast<int>(blockIdx.x), a.tiles_m, a.tiles_n, tm, tn);
    const int m0 = tm * kBM;
    const int n0 = tn * kBN;

    // This wave's copies: rows 8 c .. + 7 of one operand, lane l row l / 8 and
    // piece l % 8 as it lies in LDS.
    const bool of_x = wave * kCopies < kBM / 8;
    const int first_copy = of_x ? wave * kCopies : wave * kCopies - kBM / 8;
    const int rows_here = of_x ? (a.m - m0 < kBM ? a.m - m0 : kBM) : (a.n - n0 < kBN ? a.n - n0 : kBN);
    const int8_t* base = of_x ? a.x + static_cast<int64_t>(m0) * a.k : a.w + static_cast<int64_t>(n0) * a.k;
    const i32x4_t buffer = uniform(raw_buffer_words(base, static_cast<uint32_t>(rows_here) * static_cast<uint32_t>(a.k)));
    uint32_t offset[2];  // of even and odd copies
    uint32_t tail[2];    // in the last stage: zeros behind the end of x's rows
    const int steps = (a.k + kStep - 1) / kStep;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int piece = (lane & 7) ^ (lane >> 3) ^ b;
        offset[b] = static_cast<uint32_t>((lane >> 3) * a.k + piece * 16);
        tail[b] = of_x && (steps - 1) * kStep + piece * 16 >= a.k ? kOutOfRange : offset[b];
    }
    const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<size_t>((lds_u8_t*)own)) +
                              static_cast<uint32_t>(wave * kCopies) * 1024;
    const int turns = (steps - group + kGroups - 1) / kGroups;  // this group's steps
    const bool copies = (kBM + kBN) / 8 == kCopies * kWaves || wave * kCopies < (kBM + kBN) / 8;
    auto issue = [&](int turn) {
        if (!copies) return;
        const int step = turn * kGroups + group;
        const uint32_t dst = lds_base + static_cast<uint32_t>(turn % kStages) * kStageBytes;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            const uint32_t at = static_cast<uint32_t>((first_copy + c) * 8) * static_cast<uint32_t>(a.k) +
                                static_cast<uint32_t>(step) * kStep;
            const int odd = (first_copy + c) & 1;
            const uint32_t lane_at = step == steps - 1 ? (odd ? tail[1] : tail[0]) : (odd ? offset[1] : offset[0]);
            dma16_m0(buffer, dst + static_cast<uint32_t>(c) * 1024, lane_at, at);
        }
    };

    constexpr int kM = kWM / 32;
    constexpr int kN = kWN / 32;
    const int wm = wave / kWavesN;
    const int wn = wave % kWavesN;
    i32x16v_t acc[kN][kM];
#pragma unroll
    for (int j = 0; j < kN; ++j) {
#pragma unroll
        for (int i = 0; i < kM; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] = 0;
        }
    }
    const int row = lane & 31;
    const int sw = swizzle(row);
    const int h = lane >> 5;

#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        if (s < turns) issue(s);
    }
    // (The first group has as many turns as the other or one more.)
    for (int turn = 0; turn < (steps + kGroups - 1) / kGroups; ++turn) {
        // This wave's copies of the turn have landed, then everyone's.
        if (turn + kStages - 2 < turns) {
            __builtin_amdgcn_s_waitcnt(vmcnt_imm((kStages - 2) * kCopies));
        } else {
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        }
        bare_barrier();
        if (turn >= turns) break;  // the last barrier is passed
        if (turn + kStages - 1 < turns) issue(turn + kStages - 1);
        const uint8_t* xs = own + turn % kStages * kStageBytes + wm * kWM * kStep;
        const uint8_t* ws = own + turn % kStages * kStageBytes + (kBM + wn * kWN) * kStep;
#pragma unroll
        for (int u = 0; u < kStep / 32; ++u) {
            const int at = row * kStep + (((2 * u + h) ^ sw) << 4);
            i32x4v_t xf[kM];
            i32x4v_t wf[kN];
#pragma unroll
            for (int i = 0; i < kM; ++i) xf[i] = *reinterpret_cast<const i32x4v_t*>(xs + i * 32 * kStep + at);
#pragma unroll
            for (int j = 0; j < kN; ++j) wf[j] = *reinterpret_cast<const i32x4v_t*>(ws + j * 32 * kStep + at);
#pragma unroll
            for (int j = 0; j < kN; ++j) {
#pragma unroll
                for (int i = 0; i < kM; ++i) {
                    acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[j], xf[i], acc[j][i], 0, 0, 0);
                }
            }
        }
        __builtin_amdgcn_s_waitcnt(0xF | (3 << 14) | (7 << 4));  // LDS reads are done before the next barrier
    }

    if constexpr (kGroups == 2) {
        // 16 sums a lane and block; the first group's stages take the second one's.
        __syncthreads();
        i32x4v_t* sums = reinterpret_cast<i32x4v_t*>(lds) + wave * (kM * kN * 4 * kWaveSize) + lane;
        static_assert(kWaves * kM * kN * 64 * kWaveSize <= kGroups * kStages * kStageBytes, "room for the sums");
#pragma unroll
        for (int j = 0; j < kN; ++j) {
#pragma unroll
            for (int i = 0; i < kM; ++i) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    i32x4v_t& at = sums[((j * kM + i) * 4 + q) * kWaveSize];
                    if (group == 1) {
                        at = i32x4v_t{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
                    }
                }
            }
        }
        __syncthreads();
        if (group == 1) return;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
#pragma unroll
            for (int i = 0; i < kM; ++i) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const i32x4v_t at = sums[((j * kM + i) * 4 + q) * kWaveSize];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][i][4 * q + e] += at[e];
                }
            }
        }
    }

    const bool vectors = a.n % 4 == 0;
#pragma unroll
    for (int i = 0; i < kM; ++i) {
        const int gi = m0 + wm * kWM + 32 * i + (lane & 31);
        if (gi >= a.m) continue;
        const float xs = a.x_scales[gi];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int gj = n0 + wn * kWN + 32 * j + 8 * q + 4 * h;
                if (gj >= a.n) continue;
                const int sum[4] = {acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
                store4<T>(a, gi, gj, sum, xs, vectors);
            }
        }
    }
}

// ---- products with one wave per SIMD ----------------------------------------------
// 256 x 256 results per workgroup of four waves, 128 x 128 each as 4 x 4 blocks in
// the accumulation registers (a wave has 512 registers when it is alone on its
// SIMD): per MFMA half of the LDS reads that a 64 x 128 wave tile needs.
//   * Stages of 128 bytes of k, two in LDS, of 32 KiB for either operand. Every
//     wave copies a quarter of each: 16 copies.
//   * Fragments are double-buffered in registers by halves of 64 bytes: the 32
//     MFMAs of one half issue while the next half's fragments are read.
//   * One barrier per stage, between its halves: by then every wave has read all
//     of it, so the stage after next takes its place, a copy behind every second
//     MFMA of the second half; and the next stage, sent one stage ago, has landed.
//     (Waiting for it twelve MFMAs later, at a second barrier, was 7% slower.)
constexpr int kBigTile = 256;
constexpr int kBigOperand = kBigTile * kStep;  // 32 KiB
constexpr int kBigLds = 4 * kBigOperand;       // x of both stages, then w

template <typename T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
void matmul_int8_big_kernel(Int8Args a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBigLds];
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1;
    const int wn = wave & 1;
    int tm;
    int tn;
    tile_of(static_cast<int>(blockIdx.x), a.tiles_m, a.tiles_n, tm, tn);
    const int m0 = tm * kBigTile;
    const int n0 = tn * kBigTile;
    const uint32_t k = static_cast<uint32_t>(a.k);
    const int rows_here = a.m - m0 < kBigTile ? a.m - m0 : kBigTile;
    const int cols_here = a.n - n0 < kBigTile ? a.n - n0 : kBigTile;
    const i32x4_t xbuf = uniform(raw_buffer_words(a.x + static_cast<int64_t>(m0) * a.k, static_cast<uint32_t>(rows_here) * k));
    const i32x4_t wbuf = uniform(raw_buffer_words(a.w + static_cast<int64_t>(n0) * a.k, static_cast<uint32_t>(cols_here) * k));
    // Copy i (0 .. 7) of an operand: rows 64 wave + 8 i + l / 8, piece l % 8 as it
    // lies in LDS. The row's swizzle takes l / 8 and bit 0 of i, so two lane offsets
    // serve all eight; 16 (i / 2) rows go into the scalar offset.
    const int steps = (a.k + kStep - 1) / kStep;
    uint32_t offset[2];
    uint32_t tail[2];  // of x in the last stage: zeros behind the rows' end
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int row = 64 * wave + 8 * b + (lane >> 3);
        const int piece = (lane & 7) ^ swizzle(row);
        offset[b] = static_cast<uint32_t>(row) * k + static_cast<uint32_t>(piece) * 16;
        tail[b] = (steps - 1) * kStep + piece * 16 >= a.k ? kOutOfRange : offset[b];
    }
    const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<size_t>((lds_u8_t*)lds)) +
                              static_cast<uint32_t>(wave) * 8192;
    // Copy s (0 .. 15) of a stage: x's for even s, w's for odd ones.
    auto issue = [&](int step, int s, bool last) {
        const int i = s >> 1;
        const uint32_t dst = lds_base + static_cast<uint32_t>((step & 1) * kBigOperand + i * 1024) + ((s & 1) ? 2 * kBigOperand : 0);
        const uint32_t at = static_cast<uint32_t>(step) * kStep + static_cast<uint32_t>(i >> 1) * 16 * k;
        const uint32_t lane_at = (s & 1) == 0 && last ? tail[i & 1] : offset[i & 1];
        dma16_m0((s & 1) ? wbuf : xbuf, dst, lane_at, at);
    };

    // Block i of x (second operand): rows wm 128 + 32 i + l % 32; of w (first): wn
    // 128 + 32 j + l % 32. A lane takes bytes 32 (l / 32) .. + 31 of a half, 16 to
    // an MFMA: whatever the order along k, it is the same for both.
    const int h = lane >> 5;
    const int sw = swizzle(lane & 31);
    const int rd0 = (lane & 31) * kStep + (((2 * h) ^ sw) << 4);
    const int rd1 = (lane & 31) * kStep + (((2 * h + 1) ^ sw) << 4);
    struct Pair {
        i32x4v_t lo, hi;
    };
    struct Frags {
        Pair w[4];
        Pair x[4];
    };
    auto read_pair = [&](int base, int half) {
        return Pair{*reinterpret_cast<const i32x4v_t*>(lds + base + (rd0 ^ (half << 6))),
                    *reinterpret_cast<const i32x4v_t*>(lds + base + (rd1 ^ (half << 6)))};
    };
    // Fragment r (0 .. 7) of a half in the order in which the MFMAs use them: w0, x0
    // .. x3, w1 .. w3.
    auto read_frag = [&](Frags& f, int stage, int half, int r) {
        if (r >= 1 && r <= 4) {
            f.x[r - 1] = read_pair(stage * kBigOperand + (wm * 128 + (r - 1) * 32) * kStep, half);
        } else {
            const int j = r == 0 ? 0 : r - 4;
            f.w[j] = read_pair((2 + stage) * kBigOperand + (wn * 128 + j * 32) * kStep, half);
        }
    };
    i32x16v_t acc[4][4];  // [w block][x block]
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] = 0;
        }
    }
    // The 32 MFMAs of a half, `between(s)` behind MFMA s; the scheduling barriers
    // keep the order. The two MFMAs of a block lie four apart: the second needs the
    // first's sums.
    auto multiply = [&](const Frags& f, auto between) {
#pragma unroll
        for (int s = 0; s < 32; ++s) {
            const int j = s >> 3;
            const int i = s & 3;
            if ((s & 4) == 0) {
                acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[j].lo, f.x[i].lo, acc[j][i], 0, 0, 0);
            } else {
                acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[j].hi, f.x[i].hi, acc[j][i], 0, 0, 0);
            }
            between(s);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

#pragma unroll
    for (int s = 0; s < 16; ++s) issue(0, s, steps == 1);
    if (steps > 1) {
#pragma unroll
        for (int s = 0; s < 16; ++s) issue(1, s, steps == 2);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(16));
    } else {
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    }
    bare_barrier();
    Frags f0;
    Frags f1;
#pragma unroll
    for (int r = 0; r < 8; ++r) read_frag(f0, 0, 0, r);
    using yes = std::true_type;
    using no = std::false_type;
    auto stage = [&](int step, auto send, auto more) {
        multiply(f0, [&](int s) {
            if (s % 4 == 0) read_frag(f1, step & 1, 1, s >> 2);
        });
        // Every wave has read all of the stage; the next one has landed.
        __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));
        if constexpr (decltype(more)::value) {
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            bare_barrier();
        }
        multiply(f1, [&](int s) {
            if constexpr (decltype(more)::value) {
                if (s % 4 == 0) read_frag(f0, (step & 1) ^ 1, 0, s >> 2);
            }
            if constexpr (decltype(send)::value) {
                if (s & 1) issue(step + 2, s >> 1, step + 3 == steps);
            }
        });
    };
    // The last two stages apart, so that the loop has no branch to move MFMAs across.
    int step = 0;
    for (; step + 2 < steps; ++step) stage(step, yes{}, yes{});
    if (steps >= 2) stage(step++, no{}, yes{});
    stage(step, no{}, no{});

    // acc[j][i] element 4 q + e of lane l: row wm 128 + 32 i + l % 32, column wn 128 +
    // 32 j + 8 q + 4 (l / 32) + e. 32 rows at a time go through the wave's part of LDS
    // to be stored as whole pieces of rows.
    __syncthreads();
    constexpr int kPer = Storage<T>::kPerVec;
    const int col0 = n0 + wn * 128;
    float4 ws[4][4];
    float4 bias[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = col0 + 32 * j + 8 * q + 4 * h;
            float w4[4];
            float b4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = col + e < a.n ? col + e : a.n - 1;
                w4[e] = a.w_scales[at];
                b4[e] = bias_at<T>(a, at);
            }
            ws[j][q] = make_float4(w4[0], w4[1], w4[2], w4[3]);
            bias[j][q] = make_float4(b4[0], b4[1], b4[2], b4[3]);
        }
    }
    uint8_t* stage_out = lds + wave * (32 * 128 * 4);
    const bool whole = a.n % kPer == 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = lane & 31;
        const int row0 = m0 + wm * 128 + 32 * i;
        const float xs = a.x_scales[row0 + r < a.m ? row0 + r : a.m - 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const i32x16v_t& c = acc[j][i];
                const float v[4] = {result(c[4 * q], xs, ws[j][q].x, bias[j][q].x),
                                    result(c[4 * q + 1], xs, ws[j][q].y, bias[j][q].y),
                                    result(c[4 * q + 2], xs, ws[j][q].z, bias[j][q].z),
                                    result(c[4 * q + 3], xs, ws[j][q].w, bias[j][q].w)};
                if constexpr (sizeof(T) == 4) {
                    const int piece = 8 * j + 2 * q + h;
                    *reinterpret_cast<float4*>(stage_out + r * 512 + ((piece ^ r) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    const int piece = 4 * j + q;
                    *reinterpret_cast<uint2*>(stage_out + r * 256 + ((piece ^ (r & 15)) << 4) + ((h ^ (r >> 4)) << 3)) =
                        make_uint2(Storage<T>::to_bits2(v[0], v[1]), Storage<T>::to_bits2(v[2], v[3]));
                }
            }
        }
        // Only this wave reads what it wrote.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        constexpr int kPieces = 128 / kPer;          // of 16 bytes per row
        constexpr int kRowsAt = kWaveSize / kPieces;  // per store
        const int piece = lane % kPieces;
        const int col = col0 + piece * kPer;
#pragma unroll
        for (int s = 0; s < 32 / kRowsAt; ++s) {
            const int out = s * kRowsAt + lane / kPieces;
            uint4 v;
            if constexpr (sizeof(T) == 4) {
                v = *reinterpret_cast<const uint4*>(stage_out + out * 512 + ((piece ^ out) << 4));
            } else {
                v = *reinterpret_cast<const uint4*>(stage_out + out * 256 + ((piece ^ (out & 15)) << 4));
                if (out >> 4) v = make_uint4(v.z, v.w, v.x, v.y);
            }
            if (row0 + out >= a.m || col >= a.n) continue;
            T* y = static_cast<T*>(a.y) + static_cast<int64_t>(row0 + out) * a.n + col;
            if (whole) {
                store_stream16(y, v);
            } else {
                const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    if (col + e >= a.n) continue;
                    if constexpr (sizeof(T) == 4) {
                        reinterpret_cast<uint32_t*>(y)[e] = words[e];
                    } else {
                        reinterpret_cast<uint16_t*>(y)[e] = static_cast<uint16_t>(words[e / 2] >> (16 * (e & 1)));
                    }
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

/// Few rows: 16 columns per workgroup, whose waves split k; w goes from memory
/// to the matrix cores without LDS.
template <typename T, int kM>
__global__ __launch_bounds__(512) void matmul_int8_rows_kernel(Int8Args a) {
    constexpr int kWaves = 8;
    constexpr int kAhead = 4;
    __shared__ i32x4v_t sums[kWaves][kM][kWaveSize];
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = static_cast<int>(blockIdx.x) * 16;
    const int g = lane >> 4;
    const int col = n0 + (lane & 15) < a.n ? n0 + (lane & 15) : a.n - 1;
    const int8_t* w = a.w + static_cast<int64_t>(col) * a.k;
    const int8_t* x[kM];
    i32x4v_t acc[kM];
#pragma unroll
    for (int i = 0; i < kM; ++i) {
        const int r = 16 * i + (lane & 15) < a.m ? 16 * i + (lane & 15) : a.m - 1;
        x[i] = a.x + static_cast<int64_t>(r) * a.k;
        acc[i] = i32x4v_t{0, 0, 0, 0};
    }
    const i32x4v_t none = {0, 0, 0, 0};
    // Steps of 64 bytes, a quarter for each 16 lanes; waves take runs of kAhead.
    for (int k0 = wave * kAhead * 64; k0 < a.k; k0 += kWaves * kAhead * 64) {
        i32x4v_t wf[kAhead];
        i32x4v_t xf[kAhead][kM];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int at = k0 + u * 64 + g * 16;
            const bool in = at < a.k;
            wf[u] = in ? *reinterpret_cast<const i32x4v_t*>(w + at) : none;
#pragma unroll
            for (int i = 0; i < kM; ++i) xf[u][i] = in ? *reinterpret_cast<const i32x4v_t*>(x[i] + at) : none;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
#pragma unroll
            for (int i = 0; i < kM; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], xf[u][i], acc[i], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < kM; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    // Row tile i of the results: wave i adds the waves' parts.
    for (int i = wave; i < kM; i += kWaves) {
        int sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            const i32x4v_t part = sums[v][i][lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += part[e];
        }
        const int gi = 16 * i + (lane & 15);
        const int gj = n0 + 4 * g;
        if (gi < a.m && gj < a.n) store4<T>(a, gi, gj, sum, a.x_scales[gi], a.n % 4 == 0);
    }
}

/// Any k and alignment. Tiles beyond the grid's number go in turn. Slow: 333 rows by
/// 4096 columns of 4095 take 335 us.
template <typename T>
__global__ __launch_bounds__(256) void matmul_int8_any_kernel(Int8Args a) {
    constexpr int kTile = 16;
    constexpr int kDeep = 64;
    __shared__ __attribute__((aligned(4))) int8_t xs[kTile][kDeep + 4];
    __shared__ __attribute__((aligned(4))) int8_t ws[kTile][kDeep + 4];
    const int tid = static_cast<int>(threadIdx.x);
    for (int64_t tile = blockIdx.x; tile < static_cast<int64_t>(a.tiles_m) * a.tiles_n; tile += gridDim.x) {
        const int tm = static_cast<int>(tile / a.tiles_n);
        const int tn = static_cast<int>(tile % a.tiles_n);
        const int i = tm * kTile + tid / kTile;
        const int j = tn * kTile + tid % kTile;
        int sum = 0;
        for (int k0 = 0; k0 < a.k; k0 += kDeep) {
            for (int c = tid; c < kTile * kDeep; c += 256) {
                const int r = c / kDeep;
                const int k = k0 + c % kDeep;
                const int xr = tm * kTile + r;
                const int wr = tn * kTile + r;
                xs[r][c % kDeep] = xr < a.m && k < a.k ? a.x[static_cast<int64_t>(xr) * a.k + k] : static_cast<int8_t>(0);
                ws[r][c % kDeep] = wr < a.n && k < a.k ? a.w[static_cast<int64_t>(wr) * a.k + k] : static_cast<int8_t>(0);
            }
            __syncthreads();
#pragma unroll 4
            for (int k = 0; k < kDeep; k += 4) {
                sum = __builtin_amdgcn_sdot4(*reinterpret_cast<const int*>(&xs[tid / kTile][k]),
                                             *reinterpret_cast<const int*>(&ws[tid % kTile][k]), sum, false);
            }
            __syncthreads();
        }
        if (i < a.m && j < a.n) {
            Storage<T>::store(static_cast<T*>(a.y) + static_cast<int64_t>(i) * a.n + j,
                              result(sum, a.x_scales[i], a.w_scales[j], bias_at<T>(a, j)));
        }
    }
}

// ---- host -----------------------------------------------------------------------

enum class Way { kAny, kRows, kTile64, kSplit64, kSplit96, kTile128, kTile256 };

Way way_of(const Int8Args& a) {
    if (a.k == 0 || a.k % 16 != 0 || !host_aligned(a.x, 16) || !host_aligned(a.w, 16) || !host_aligned(a.y, 16)) return Way::kAny;
    // Up to 16 rows w streams by. Up to 64 it still may, where there are too few tiles of
    // 64 columns to fill the GPU: 32 rows of 4096 by 4096 columns take 12 us against
    // 14.5 in tiles (64 of them), 64 rows 16 against 15; but by 11008 columns (172
    // tiles) 22 and 33 us against 15 and 16, and 17 rows 18 against 15.
    // (The general kernel takes columns past one launch.)
    if (ceil_div<int64_t>(a.n, 16) > kMaxWorkgroups / 2 && a.m <= 16) return Way::kAny;
    if (a.m <= 16 || (a.m <= 64 && ceil_div<int64_t>(a.n, 64) < 128)) return Way::kRows;
    // Tiles of 128 x 128 run two a CU, 512 at once. Fewer than 192 leave too many CUs
    // idle (96 and 160 of them, k 4096: 30 and 32 us against 20 and 30 in tiles of 64;
    // 192 and 256: 32 and 33 against 32 and 36). More than 512 take a second round, and
    // tiles of 256 are faster (384 and 512: 40 and 45 us against 46 and 47; 516 and
    // 640: 73 and 65 against 47 and 49).
    const int64_t mid = ceil_div<int64_t>(a.m, 128) * ceil_div<int64_t>(a.n, 128);
    if (mid >= 192) return mid > 512 ? Way::kTile256 : Way::kTile128;
    auto small = [&](int bm) { return ceil_div<int64_t>(a.m, bm) * ceil_div<int64_t>(a.n, 64); };
    // Where a CU has one tile of 64 x 64, or one of 96 x 64 instead of two, two groups of
    // waves share its k: 128 rows by 4096 columns of 4096 13.0 us against 15.3; 333 rows
    // 16.1 us against 19.4 in tiles of 64 and 18.0 with one group, of 11008 32 us against
    // 49 and 37.
    if (small(64) <= 256) return Way::kSplit64;
    return small(96) <= 256 ? Way::kSplit96 : Way::kTile64;
}

void tiles(Int8Args& a, int bm, int bn) {
    a.tiles_m = (a.m + bm - 1) / bm;
    a.tiles_n = (a.n + bn - 1) / bn;
}

template <typename T>
cf_status run(Int8Args a, hipStream_t stream) {
    const Way way = way_of(a);
    int threads = 256;
    void (*kernel)(Int8Args) = nullptr;
    switch (way) {
        case Way::kAny: tiles(a, 16, 16); kernel = matmul_int8_any_kernel<T>; break;
        case Way::kRows:
            tiles(a, a.m, 16);
            threads = 512;
            kernel = a.m <= 16   ? matmul_int8_rows_kernel<T, 1>
                     : a.m <= 32 ? matmul_int8_rows_kernel<T, 2>
                                 : matmul_int8_rows_kernel<T, 4>;
            break;
        case Way::kTile64: tiles(a, 64, 64); kernel = matmul_int8_kernel<T, 64, 64, 32, 32, 4, 1>; break;
        case Way::kSplit64:
            tiles(a, 64, 64);
            threads = 512;
            kernel = matmul_int8_kernel<T, 64, 64, 32, 32, 4, 2>;
            break;
        case Way::kSplit96:
            tiles(a, 96, 64);
            threads = 768;
            kernel = matmul_int8_kernel<T, 96, 64, 32, 32, 3, 2>;
            break;
        case Way::kTile128: tiles(a, 128, 128); kernel = matmul_int8_kernel<T, 128, 128, 64, 64, 2, 1>; break;
        case Way::kTile256: tiles(a, 256, 256); kernel = matmul_int8_big_kernel<T>; break;
    }
    int64_t grid = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
    if (way == Way::kAny && grid > kMaxWorkgroups) grid = kMaxWorkgroups;
    CF_REQUIRE(grid <= UINT32_MAX / threads, "cf_matmul_int8: %d x %d results are too many for a launch", a.m, a.n);
    launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(threads), 0, stream, a);
    return check_launch("launching the int8 product", stream);
}

}  // namespace
}  // namespace cf

extern "C" {

cf_status cf_quantize_int8_rows(const void* x, cf_dtype dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                int8_t* codes, float* scales, void* stream) {
    CF_ENTRY();
    const char* who = "cf_quantize_int8_rows";
    if (rows <= 0 || cols <= 0) return CF_OK;
    CF_REQUIRE(cf::valid_dtype(dtype), "%s: unknown dtype %d", who, static_cast<int>(dtype));
    CF_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, "%s: null pointer", who);
    CF_REQUIRE(row_stride >= cols || rows == 1, "%s: rows of %lld are %lld apart", who, static_cast<long long>(cols),
               static_cast<long long>(row_stride));
    CF_REQUIRE(cf::host_aligned(x, cf::dtype_size(dtype)) && cf::host_aligned(scales, 4), "%s: misaligned pointer", who);
    const cf::RowsArgs a{x, codes, scales, rows, cols, row_stride};
    auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case CF_F32: cf::launch_rows<float>(a, s); break;
        case CF_F16: cf::launch_rows<cf::f16_t>(a, s); break;
        case CF_BF16: cf::launch_rows<cf::bf16_t>(a, s); break;
    }
    return cf::check_launch("launching the row quantiser", s);
}

cf_status cf_matmul_int8(const int8_t* x, const int8_t* w, const float* x_scales, const float* w_scales,
                         const void* bias, void* y, cf_dtype dtype, int64_t m, int64_t n, int64_t k, void* stream) {
    CF_ENTRY();
    const char* who = "cf_matmul_int8";
    if (m <= 0 || n <= 0) return CF_OK;
    CF_REQUIRE(cf::valid_dtype(dtype), "%s: unknown dtype %d", who, static_cast<int>(dtype));
    CF_REQUIRE(k >= 0 && k <= 131071 && m <= INT32_MAX - 256 && n <= INT32_MAX - 256,
               "%s: %lld x %lld results of %lld products (at most 131071)", who, static_cast<long long>(m),
               static_cast<long long>(n), static_cast<long long>(k));
    CF_REQUIRE((x != nullptr && w != nullptr) || k == 0, "%s: null pointer", who);
    CF_REQUIRE(x_scales != nullptr && w_scales != nullptr && y != nullptr, "%s: null pointer", who);
    const size_t size = cf::dtype_size(dtype);
    CF_REQUIRE(cf::host_aligned(y, size) && cf::host_aligned(bias, size) && cf::host_aligned(x_scales, 4) &&
                   cf::host_aligned(w_scales, 4),
               "%s: misaligned pointer", who);
    cf::Int8Args a{};
    a.x = x;
    a.w = w;
    a.x_scales = x_scales;
    a.w_scales = w_scales;
    a.bias = bias;
    a.y = y;
    a.m = static_cast<int>(m);
    a.n = static_cast<int>(n);
    a.k = static_cast<int>(k);
    auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case CF_F32: return cf::run<float>(a, s);
        case CF_F16: return cf::run<cf::f16_t>(a, s);
        case CF_BF16: return cf::run<cf::bf16_t>(a, s);
    }
    return CF_OK;
}

}  // extern "C"
