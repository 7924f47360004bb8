// Causal attention of the newest tokens of every sequence over a paged cache,
// in the query's type or in 8-bit codes with a scale per row.
//
// Row i of sequence s, of n_s new tokens in a context of c_s, is at position
// p = c_s - n_s + i; for head h and KV head h / (H / KVH):
//   out = sum_{t <= p} softmax_t(scale q . k[t]) v[t].
//
// The rows of a sequence and KV head (tokens x heads of the KV head) against its
// keys are a matrix product; a row tile of a long chunk is bound by the matrix
// and vector units, a single token's few rows by HBM.
//   * A work item is (row tile, KV head, range of the context), a workgroup of
//     four waves. Of tiles with more than 32 rows each wave has 32 (of up to 64
//     against half of the tokens) and they share the keys and values in LDS
//     (attend_rows); with fewer, the waves take different tokens of the same rows
//     and share nothing (attend_few); fp32
//     caches have tiles of half the rows and tokens (attend). Ranges are cut only
//     where there are few items; a second kernel joins their pieces.
//   * 8-bit codes are exact in fp16, so they are widened to it on their way to the
//     products, which run in fp16 whatever the query's type: a bf16 query is scaled
//     by a power of two per row (it has fewer bits than fp16 holds, and what falls
//     below fp16's smallest number is 2^-39 of the row's largest), an fp32 query is
//     taken as the sum of two fp16 numbers. Keys' scales multiply the scores,
//     values' scales the probabilities, in fp32.
//   * Tokens that are not there (behind the range, in no page) get no weight, and
//     what the cache holds in their place never reaches a row.
// Measured, 32 heads over 8 of 128: a prompt of 2048 tokens in bf16 61 us (560
// TFLOP/s: the chain product, probabilities, product, at two waves a SIMD, and
// the causal tiles' different lengths); 2048 tokens behind 30720 1.10 to 1.22 ms by
// the card (870 to 970 TFLOP/s: matrix cores 44% and vector units 48% busy, and the
// clock falls from 2.2 to 1.7 GHz under them); 64 sequences of 2051 to 4096 tokens in
// int8, a token each, 102 us (4.1 TB/s; 4.8 TB/s at equal lengths: reads of single
// 128-byte lines, where bf16's of 256 bytes reach 5.9).
#include "cf_attention_tile.hpp"
#include "cf_codes.hpp"
#include "cf_common.hpp"
#include "cf_lds_dma.hpp"
#include "cf_ranges.hpp"

namespace cf {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWaveSize;
constexpr int kMaxSplits = 64;
constexpr float kLog2e = 1.4426950408889634f;
/// Of 8-bit caches' values, scales below 2^-90 count as that (see attend_few).
constexpr int kLeastUnit = -90;

struct ChunkArgs {
    const void* query;
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const float* k_scales;
    const float* v_scales;
    const int32_t* starts;  // [sequences + 1]
    const uint32_t* tables;
    const int32_t* context;
    void* out;
    float* ml;   // [splits][tokens * heads][2]: maximum (base 2), sum
    float* acc;  // [splits][tokens * heads][pitch]
    uint32_t pages;
    uint32_t block_size;
    int block_shift;  // log2(block_size), or -1
    int tokens;
    int sequences;
    int heads;
    int kv_heads;
    int per;  // query heads per KV head
    int head_dim;
    int pitch;  // head_dim rounded up to 4
    int max_blocks;
    int capacity;  // tokens a table row reaches
    uint32_t token_pieces;  // 16 bytes of a token of the cache
    int rows;  // of a tile
    int splits;
    int step;  // tokens of a range are a multiple of this
    int least;  // and at least about this
    bool query_bf16;  // of 8-bit caches: the query's and the result's 16-bit type
    float c;              // |scale| log2(e), above 0
    uint32_t query_sign;  // flips the query's signs for a negative scale
};

__device__ __forceinline__ int clamp_to(int v, int hi) { return v < 0 ? 0 : v > hi ? hi : v; }

/// The exponent of the power of two above the largest of scales, kLeastUnit at
/// least: what is taken where there is none of them, too (0's exponent is 0, far
/// above those of small values).
__device__ __forceinline__ int unit_above(float largest) {
    return largest > 0.0f ? max(__builtin_amdgcn_frexp_expf(largest), kLeastUnit) : kLeastUnit;
}

// ---- items ----------------------------------------------------------------------

/// Neighbouring rows (tokens) of one sequence, or of none.
struct Segment {
    int sequence;  // -1: rows that no sequence holds
    int first;     // token
    int count;
    int tile;  // of the segment
};

/// Tile `index` (uniform) of all segments' tiles laid end to end: the rows before
/// the first start, the sequences', the rows behind the last one. Starts are
/// taken as the largest so far, so that segments never overlap whatever is
/// stored. count = 0: no such tile.
__device__ Segment segment_of(const ChunkArgs& a, int rows, int index) {
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    int before = 0;  // largest start so far
    const int segments = a.sequences + 2;
    for (int base = 0; base < segments; base += kWaveSize) {
        const int i = base + lane;  // from starts[i - 1] to starts[i]
        int end = i <= a.sequences ? clamp_to(a.starts[min(i, a.sequences)], a.tokens) : a.tokens;
        end = max(end, before);
#pragma unroll
        for (int d = 1; d < kWaveSize; d <<= 1) {
            const int o = __shfl_up(end, d);
            if (lane >= d) end = max(end, o);
        }
        int start = __shfl_up(end, 1);
        if (lane == 0) start = before;
        const int tiles = i < segments ? static_cast<int>((static_cast<int64_t>(end - start) * a.per + rows - 1) / rows) : 0;
        int total = tiles;
#pragma unroll
        for (int d = 1; d < kWaveSize; d <<= 1) {
            const int o = __shfl_up(total, d);
            if (lane >= d) total += o;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(total > index);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            const int n = __builtin_amdgcn_readlane(tiles, at);
            const int first = __builtin_amdgcn_readlane(start, at);
            const int sequence = base + at - 1;
            index -= __builtin_amdgcn_readlane(total, at) - n;
            // The last tiles of a chunk see most tokens: they come first, but those of
            // the second half turned round, so that of a chunk that fills the GPU once
            // (two workgroups a CU) a CU gets a long one and a short one.
            const int half = (n + 1) / 2;
            return Segment{sequence < a.sequences ? sequence : -1, first, __builtin_amdgcn_readlane(end, at) - first,
                           index < half ? n - 1 - index : index - half};
        }
        index -= __builtin_amdgcn_readlane(total, kWaveSize - 1);
        before = __builtin_amdgcn_readlane(end, kWaveSize - 1);
    }
    return Segment{-1, 0, 0, 0};
}

/// The segment of one token (uniform).
__device__ Segment segment_of_token(const ChunkArgs& a, int token) {
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    int before = 0;
    const int segments = a.sequences + 2;
    for (int base = 0; base < segments; base += kWaveSize) {
        const int i = base + lane;
        int end = i <= a.sequences ? clamp_to(a.starts[min(i, a.sequences)], a.tokens) : a.tokens;
        end = max(end, before);
#pragma unroll
        for (int d = 1; d < kWaveSize; d <<= 1) {
            const int o = __shfl_up(end, d);
            if (lane >= d) end = max(end, o);
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(end > token);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            const int first = at > 0 ? __builtin_amdgcn_readlane(end, at - 1) : before;
            const int sequence = base + at - 1;
            return Segment{sequence < a.sequences ? sequence : -1, first, __builtin_amdgcn_readlane(end, at) - first, 0};
        }
        before = __builtin_amdgcn_readlane(end, kWaveSize - 1);
    }
    return Segment{-1, 0, 0, 0};
}

/// What a tile of a segment's rows sees.
struct Reach {
    int offset;  // position of the segment's first token
    int hi;      // tokens that the tile's last row sees, at least 0
    int each;    // tokens per range
};

__device__ __forceinline__ Reach reach_of(const ChunkArgs& a, const Segment& s, int rows) {
    Reach r{};
    const int context = clamp_to(a.context[s.sequence], a.capacity);
    r.offset = context - s.count;
    const int64_t last_row = static_cast<int64_t>(s.tile + 1) * rows - 1;
    const int64_t last_token = last_row / a.per;
    r.hi = r.offset + (last_token < s.count ? static_cast<int>(last_token) + 1 : s.count);
    r.hi = r.hi < 0 ? 0 : r.hi;
    r.each = split_length(r.hi, a.splits, a.step, a.least);
    return r;
}

// ---- one work item ----------------------------------------------------------------

struct Item {
    const uint32_t* table;
    int lo, hi;
    int offset;     // position of the segment's first token
    int first;      // the segment's first token
    int rows;       // of the segment: tokens x heads of the KV head
    int first_row;  // of the tile
    int kv_head;
    int split;
    bool direct;    // the only piece: straight to the result
};

/// What counts as the scale of a row of values: a row of zeros, which is stored
/// with the scale 1 whatever the others' are, must not stand for the largest of
/// them, so its scale is taken as 0. `row()`: its codes, read only if the scale is 1
/// and, by `matters`, until a row has met a larger one or another of 1 (a cache of
/// scales that are all 1 would be read twice).
template <cf_cache_format kHeld, typename Row>
__device__ __forceinline__ float value_scale(float scale, bool matters, Row row, int bytes) {
    if (scale == 1.0f && matters) {
        const uint8_t* from = row();
        constexpr uint32_t kMagnitudes = kHeld == CF_CACHE_E4M3 ? 0x7F7F7F7Fu : 0xFFFFFFFFu;
        uint32_t any = 0;
#pragma unroll 1
        for (int at = 0; at < bytes && any == 0; at += 16) {
            const u32x4_t codes = *reinterpret_cast<const u32x4_t*>(from + at);
            any = (codes[0] | codes[1] | codes[2] | codes[3]) & kMagnitudes;
        }
        if (any == 0) scale = 0.0f;
    }
    return scale;
}

/// Values that are not finite, of tokens that some rows of a tile see and others do
/// not: a product would take them, times 0, to all rows. They are set to 0 in it.
/// Where that happened the range's values are looked through again at the end, and
/// for each dim the first position that holds one is kept in LDS: the rows from there
/// on see it, and their results are made what it makes them. (Changing the sums within
/// the loop, or noting the positions there, cost heads of 256 20 to 35%.)
template <int kD>
struct BadValues {
    static constexpr int kNone = 0x7FFFFFFF;
    int plus[kD];  // positions of infinities, and of what is no number, which is in both
    int minus[kD];
    int from[kWaves];  // the first token of a wave's first tile with such a value

    /// Whether there are any; then they are noted. Called by the whole workgroup, behind
    /// a barrier after `from` was set.
    template <typename T, cf_cache_format kHeld>
    __device__ __forceinline__ bool find(const ChunkArgs& a, const Item& w) {
        static_assert(kWaves == 4, "four of them");
        const int first = min(min(from[0], from[1]), min(from[2], from[3]));
        if (first >= w.hi) return false;
        const int tid = static_cast<int>(threadIdx.x);
        for (int i = tid; i < kD; i += kThreads) plus[i] = minus[i] = kNone;
        __syncthreads();
        constexpr int kSize = kHeld == CF_CACHE_PLAIN ? static_cast<int>(sizeof(T)) : 1;
        constexpr uint32_t kSign = 1u << (8 * kSize - 1);
        constexpr uint32_t kInfinity = kSize == 4 ? 0x7F800000u : std::is_same<T, f16_t>::value ? 0x7C00u : 0x7F80u;
        for (int64_t i = static_cast<int64_t>(first) * a.head_dim + tid; i < static_cast<int64_t>(w.hi) * a.head_dim; i += kThreads) {
            const int t = static_cast<int>(i / a.head_dim);
            const int dim = static_cast<int>(i % a.head_dim);
            const uint32_t block = static_cast<uint32_t>(t) / a.block_size;
            const uint32_t page = w.table[block];
            if (page >= a.pages) continue;
            const uint64_t row = static_cast<uint64_t>(page) * a.block_size + (static_cast<uint32_t>(t) - block * a.block_size);
            const uint64_t at = (row * static_cast<uint32_t>(a.kv_heads) + static_cast<uint32_t>(w.kv_head)) *
                                    static_cast<uint32_t>(a.head_dim) + static_cast<uint32_t>(dim);
            if constexpr (kHeld == CF_CACHE_PLAIN) {
                uint32_t bits;
                if constexpr (kSize == 4) bits = reinterpret_cast<const uint32_t*>(a.v_cache)[at];
                else bits = reinterpret_cast<const uint16_t*>(a.v_cache)[at];
                const uint32_t magnitude = bits & (kSign - 1);
                if (magnitude > kInfinity || bits == kInfinity) atomicMin(&plus[dim], t);
                if (magnitude > kInfinity || bits == (kInfinity | kSign)) atomicMin(&minus[dim], t);
            } else if ((a.v_cache[at] & 0x7F) == 0x7F) {  // e4m3 has no infinities
                atomicMin(&plus[dim], t);
                atomicMin(&minus[dim], t);
            }
        }
        __syncthreads();
        return true;
    }
    /// Into four neighbouring dims of the row at `position`.
    __device__ __forceinline__ void add_to(f32x4_t& sum, int dim, int position) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sum[e] += (position >= plus[dim + e] ? INFINITY : 0.0f) - (position >= minus[dim + e] ? INFINITY : 0.0f);
        }
    }
};

/// LDS of attend: its tiles, a ring that the waves share or one for each of them.
template <int kD>
struct WideKind {
    using L = Tile<float, kD>;
    static constexpr int kStages = 4;
    static constexpr int kTileBytes = 2 * L::kBytes;
    static constexpr int lds_bytes() {
        static_assert(kStages >= kWaves, "a tile for each wave too");
        constexpr int ring = kStages * kTileBytes;
        constexpr int outputs = kWaves * L::kRows * L::kOutPitch * 4;
        return ring > outputs ? ring : outputs;
    }
};

/// 4 codes as fp16, 2 to a word.
template <cf_cache_format kHeld>
__device__ __forceinline__ uint2 widen4(uint32_t codes) {
    if constexpr (kHeld == CF_CACHE_INT8) {
        // 0x64uu is 1024 + u in fp16: u = code + 128 below it, 1152 taken off.
        typedef _Float16 f16x2_v __attribute__((ext_vector_type(2)));
        const uint32_t u = codes ^ 0x80808080u;
        const f16x2_v less = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
        const uint32_t lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - less);
        const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - less);
        return make_uint2(lo, hi);
    } else {
        return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, false)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, true)));
    }
}

/// 16 codes as fp16, 8 to a vector.
template <cf_cache_format kHeld>
__device__ __forceinline__ void widen16(const u32x4_t& codes, u32x4_t& lo, u32x4_t& hi) {
    const uint2 w0 = widen4<kHeld>(codes[0]);
    const uint2 w1 = widen4<kHeld>(codes[1]);
    const uint2 w2 = widen4<kHeld>(codes[2]);
    const uint2 w3 = widen4<kHeld>(codes[3]);
    lo = u32x4_t{w0.x, w0.y, w1.x, w1.y};
    hi = u32x4_t{w2.x, w2.y, w3.x, w3.y};
}

/// This lane's query row in a tile of layout L (token of the segment, head of the KV head): fragments
/// q, and for kSplit what they leave; zeros outside. Returns the factor of its
/// scores. 8-bit caches: scaled by a power of two to magnitudes of up to 2^15, the
/// inverse in the factor.
template <typename L, typename T, bool kCodes, bool kSplit>
__device__ __forceinline__ float load_query(const ChunkArgs& a, const Item& w, bool inside, int token, int head, int lane,
                                            typename L::Query (&q)[L::kQueries],
                                            typename L::Query (&q_low)[kSplit ? L::kQueries : 1]) {
    float c = a.c;
    const int64_t out_row = static_cast<int64_t>(w.first + token) * a.heads + w.kv_head * a.per + head;
    if constexpr (!kCodes) {
        const T* from = static_cast<const T*>(a.query) + out_row * a.head_dim;
#pragma unroll
        for (int u = 0; u < L::kQueries; ++u) {
            const int dim = L::query_dim(u, lane);
            u32x4_t raw = {0u, 0u, 0u, 0u};
            if (inside && dim < a.head_dim) raw = *reinterpret_cast<const u32x4_t*>(from + dim) ^ a.query_sign;
            q[u] = __builtin_bit_cast(typename L::Query, raw);
        }
    } else {
        float f[L::kQueries][8];
        float top = 0.0f;
#pragma unroll
        for (int u = 0; u < L::kQueries; ++u) {
            const int dim = L::query_dim(u, lane);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[u][e] = 0.0f;
            if (inside && dim < a.head_dim) {
                if constexpr (kSplit) {
                    const float* from = static_cast<const float*>(a.query) + out_row * a.head_dim + dim;
                    unpack16<float>(*reinterpret_cast<const uint4*>(from), f[u]);
                    unpack16<float>(*reinterpret_cast<const uint4*>(from + 4), f[u] + 4);
                } else {
                    const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.query) +
                                                                     out_row * a.head_dim + dim);
                    if (a.query_bf16) unpack16<bf16_t>(raw, f[u]); else unpack16<f16_t>(raw, f[u]);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[u][e]));
        }
        top = groups_max<L::kRows>(top);
        const int lift = 15 - __builtin_amdgcn_frexp_expf(top);
        // Not 0, which times a masked score is NaN.
        c = fmaxf(__builtin_amdgcn_ldexpf(c, -lift), 0x1p-126f);
        const float sign = a.query_sign != 0 ? -1.0f : 1.0f;
        typedef _Float16 f16x2_v __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int u = 0; u < L::kQueries; ++u) {
            u32x4_t high, low;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x0 = __builtin_amdgcn_ldexpf(f[u][2 * e] * sign, lift);
                const float x1 = __builtin_amdgcn_ldexpf(f[u][2 * e + 1] * sign, lift);
                const f16x2_v h = {static_cast<_Float16>(x0), static_cast<_Float16>(x1)};
                high[e] = __builtin_bit_cast(uint32_t, h);
                if constexpr (kSplit) {
                    low[e] = __builtin_bit_cast(uint32_t, f16x2_v{static_cast<_Float16>(x0 - static_cast<float>(h[0])),
                                                                  static_cast<_Float16>(x1 - static_cast<float>(h[1]))});
                }
            }
            q[u] = __builtin_bit_cast(typename L::Query, high);
            if constexpr (kSplit) q_low[u] = __builtin_bit_cast(typename L::Query, low);
        }
    }
    return c;
}

/// Four neighbouring dims of a row from the kCount waves that have some of its
/// tokens, kApart waves apart: `sums`, lds_m and lds_l of the first, sums of
/// neighbouring waves `pitch` floats apart.
struct Joined {
    float m, l;
    f32x4_t sum;
};
template <int kCount, int kApart>
__device__ __forceinline__ Joined join_waves(const float* sums, int pitch, const float (*lds_m)[32],
                                             const float (*lds_l)[32], int row) {
    Joined j{lds_m[0][row], 0.0f, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int t = kApart; t < kCount * kApart; t += kApart) j.m = fmaxf(j.m, lds_m[t][row]);
#pragma unroll
    for (int t = 0; t < kCount * kApart; t += kApart) {
        const float mt = lds_m[t][row];
        const float f = mt == -INFINITY ? 0.0f : exp2f(mt - j.m);
        // A wave without a finite score still passes its NaN on.
        j.l += mt == -INFINITY ? lds_l[t][row] : lds_l[t][row] * f;
        const f32x4_t four = *reinterpret_cast<const f32x4_t*>(sums + t * pitch);
#pragma unroll
        for (int e = 0; e < 4; ++e) j.sum[e] = fmaf(four[e], f, j.sum[e]);
    }
    return j;
}

/// Four dims of row `row` of the segment to the result, or to a piece of it. m in base 2.
template <typename T, bool kCodes, bool kSplit>
__device__ __forceinline__ void put(const ChunkArgs& a, const Item& w, int row, int dim, float m, float l,
                                    const f32x4_t& sum) {
    const int64_t out_row = static_cast<int64_t>(w.first + row / a.per) * a.heads + w.kv_head * a.per + row % a.per;
    if (!w.direct) {
        const int64_t at = static_cast<int64_t>(w.split) * a.tokens * a.heads + out_row;
        if (dim == 0) {
            a.ml[2 * at] = m;
            a.ml[2 * at + 1] = l;
        }
        *reinterpret_cast<f32x4_t*>(a.acc + at * a.pitch + dim) = sum;
        return;
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = l == 0.0f ? 0.0f : sum[e] * by;
    const int64_t at = out_row * a.head_dim + dim;
    if constexpr (kSplit || (!kCodes && sizeof(T) == 4)) {
        *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + at) = f32x4_t{o[0], o[1], o[2], o[3]};
    } else {
        const bool bf16 = kCodes ? a.query_bf16 : std::is_same<T, bf16_t>::value;
        uint2 two;
        if (bf16) {
            two = make_uint2(Storage<bf16_t>::to_bits2(o[0], o[1]), Storage<bf16_t>::to_bits2(o[2], o[3]));
        } else {
            two = make_uint2(Storage<f16_t>::to_bits2(o[0], o[1]), Storage<f16_t>::to_bits2(o[2], o[3]));
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = two;
    }
}

/// The waves' outputs, kRowWaves of them of different rows, the others behind them
/// of different tokens of the same. bad_from: see BadValues.
template <typename T, int kD, cf_cache_format kHeld, bool kSplit, int kRowWaves>
__device__ __forceinline__ void finish(const ChunkArgs& a, const Item& w, uint8_t* lds, float (*lds_m)[32],
                                       float (*lds_l)[32], BadValues<kD>* bad, int bad_from, float m, float l,
                                       const typename Tile<T, kD>::Score (&acc)[Tile<T, kD>::kAcc / Tile<T, kD>::kScores]) {
    using L = Tile<T, kD>;
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & (kWaveSize - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
#pragma unroll
    for (int d = L::kRows; d < kWaveSize; d <<= 1) l += __shfl_xor(l, d);
    wait_vm<0>();
    __syncthreads();  // all tiles are done with: their space takes the outputs
    float* mine = reinterpret_cast<float*>(lds) + wave * L::kRows * L::kOutPitch;
#pragma unroll
    for (int i = 0; i < L::kAcc; i += 4) {
        f32x4_t four;
#pragma unroll
        for (int e = 0; e < 4; ++e) four[e] = acc[(i + e) / L::kScores][(i + e) % L::kScores];
        *reinterpret_cast<f32x4_t*>(mine + L::row_of(lane) * L::kOutPitch + L::dim_of(i, lane)) = four;
    }
    if (L::part_of(lane) == 0) {
        lds_m[wave][L::row_of(lane)] = m;
        lds_l[wave][L::row_of(lane)] = l;
    }
    if (kHeld != CF_CACHE_INT8 && lane == 0) bad->from[wave] = bad_from;
    __syncthreads();
    bool any_bad = false;
    if constexpr (kHeld != CF_CACHE_INT8) any_bad = bad->template find<T, kHeld>(a, w);
    // Rows x groups of four dims, over the workgroup.
    constexpr int kOutRows = kRowWaves * L::kRows;
    constexpr int kFours = kD / 4;
    constexpr int kRounds = (kOutRows * kFours + kThreads - 1) / kThreads;
#pragma unroll 2
    for (int n = 0; n < kRounds; ++n) {
        const int i = n * kThreads + tid;
        const int r = i / kFours;
        const int dim = (i % kFours) * 4;
        if (r >= kOutRows) break;
        const int out = w.first_row + r;
        if (out >= w.rows || dim >= a.head_dim) continue;
        const float* sums = reinterpret_cast<const float*>(lds) + r * L::kOutPitch + dim;
        const int wave_of = r / L::kRows;
        Joined j;
        if constexpr (kRowWaves == kWaves) {
            j = Joined{lds_m[wave_of][r % L::kRows], lds_l[wave_of][r % L::kRows], *reinterpret_cast<const f32x4_t*>(sums)};
        } else {
            j = join_waves<kWaves / kRowWaves, kRowWaves>(sums, L::kRows * L::kOutPitch, lds_m + wave_of,
                                                          lds_l + wave_of, r % L::kRows);
        }
        if (any_bad) bad->add_to(j.sum, dim, w.offset + out / a.per);
        put<T, kHeld != CF_CACHE_PLAIN, kSplit>(a, w, out, dim, j.m, j.l, j.sum);
    }
}

/// fp32 caches, in fp32 products: the matrix cores' slowest, half busy where a CU
/// has two workgroups (four chunks of up to 100 tokens behind 900, 84 us, and
/// 12 us for the join). kShared: the waves take different rows of the tile, else different
/// tokens of the same rows.
template <int kD, bool kShared>
__device__ void attend(const ChunkArgs& a, const Item& w, uint8_t* lds, float (*lds_m)[32], float (*lds_l)[32],
                       BadValues<kD>* bad) {
    using K = WideKind<kD>;
    using L = typename K::L;
    constexpr int kTokenWaves = kShared ? 1 : kWaves;
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & (kWaveSize - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
    const int row_wave = kShared ? wave : 0;
    const int token_wave = kShared ? 0 : wave;

    // This lane's query row; rows past the end are zeros.
    const int row = w.first_row + row_wave * L::kRows + L::row_of(lane);
    const bool inside = row < w.rows;
    const int token = inside ? row / a.per : 0;
    const int limit = inside ? w.offset + token : -1;  // the last token it sees
    typename L::Query q[L::kQueries];
    typename L::Query unused[1];
    const float c = load_query<L, float, false, false>(a, w, inside, token, inside ? row % a.per : 0, lane, q, unused);
    // The smallest of the wave's limits: tiles up to it need no mask.
    int least = inside ? limit : 0x7FFFFFFF;
#pragma unroll
    for (int d = 1; d < L::kRows; d <<= 1) least = min(least, __shfl_xor(least, d));
    const int wave_least = __builtin_amdgcn_readfirstlane(least);

    uint8_t* const own = lds + (kShared ? 0 : wave * K::kTileBytes);
    if (a.head_dim < kD) {  // the copies leave the end of every row as it is
        constexpr int kPieces = (kShared ? K::kStages : 1) * K::kTileBytes / 16;
        for (int i = kShared ? tid : lane; i < kPieces; i += kShared ? kThreads : kWaveSize) {
            reinterpret_cast<u32x4_t*>(own)[i] = u32x4_t{0u, 0u, 0u, 0u};
        }
        if constexpr (kShared) __syncthreads(); else wait_lds();
    }

    // Tiles begin at multiples of kTokens (ranges do).
    const int begin = w.lo + token_wave * L::kTokens;
    constexpr int kStride = kTokenWaves * L::kTokens;
    const int tiles = begin < w.hi ? (w.hi - begin + kStride - 1) / kStride : 0;
    const int last_block = static_cast<int>(static_cast<uint32_t>(w.hi - 1) / a.block_size);

    // 64 entries of the block table in lane registers: looking a page up is then
    // no load that would have to wait behind the copies.
    auto block_of = [&](int t) {
        return static_cast<int>(a.block_shift >= 0 ? static_cast<uint32_t>(t) >> a.block_shift
                                                   : static_cast<uint32_t>(t) / a.block_size);
    };
    int window_base = block_of(begin < w.hi ? begin : w.lo);
    uint32_t window = w.table[min(window_base + lane, last_block)];
    uint32_t valid = 0;  // tokens of the tile looked up last, a bit each
    uint32_t place = 0;  // of token lane % kTokens: row of the cache, 0 where it is not there
    constexpr uint32_t kAll = 0xFFFFFFFFu >> (32 - L::kTokens);
    auto look_up = [&](int first) {
        const int last = min(first + L::kTokens, w.hi) - 1;
        if (block_of(last) >= window_base + kWaveSize) {
            window_base = block_of(first);
            window = w.table[min(window_base + lane, last_block)];
            // Waited for here, not behind the branch, whether or not this ran.
            asm volatile("" : "+v"(window));
        }
        const int t = min(first + (lane & (L::kTokens - 1)), last);
        const int block = block_of(t);
        const uint32_t page = static_cast<uint32_t>(__shfl(static_cast<int>(window), block - window_base));
        const bool there = page < a.pages && first + (lane & (L::kTokens - 1)) < w.hi;
        place = there ? page * a.block_size + (static_cast<uint32_t>(t) - static_cast<uint32_t>(block) * a.block_size) : 0u;
        valid = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(there)) & kAll;
    };

    const uint32_t lds_own = __builtin_amdgcn_readfirstlane(lds_address(own));
    const uint64_t token_bytes = static_cast<uint64_t>(a.kv_heads) * a.head_dim * 4;
    const uint64_t head_bytes = static_cast<uint64_t>(w.kv_head) * a.head_dim * 4;
    const uint8_t* k_head = a.k_cache + head_bytes;
    const uint8_t* v_head = a.v_cache + head_bytes;

    // This wave's copies of a tile to LDS; of a shared one half of the waves copy K,
    // the others V.
    constexpr int kPerCopy = kWaveSize / L::kChunks;
    constexpr int kCopies = kShared ? 2 * L::kCopies / kWaves : L::kCopies;
    const bool shared_v = kShared && wave >= kWaves / 2;
    const int first_copy = kShared ? wave % (kWaves / 2) * kCopies : 0;
    const int row_pieces = a.head_dim / 4;
    auto copy = [&](uint32_t dst, bool is_v) {
#pragma unroll
        for (int n = 0; n < kCopies; ++n) {
            const int r = (first_copy + n) * kPerCopy + lane / L::kChunks;
            const uint64_t from = static_cast<uint32_t>(__shfl(static_cast<int>(place), r)) * token_bytes;
            const int piece = (lane % L::kChunks) ^ (is_v ? L::v_swizzle(r) : L::k_swizzle(r));
            if (piece < row_pieces) {
                copy16_to_lds((is_v ? v_head : k_head) + from + piece * 16,
                              dst + static_cast<uint32_t>(first_copy + n) * 16 * kWaveSize);
            }
        }
    };
    float m = -INFINITY;  // the row's running maximum
    float l = 0.0f;       // this lane's share of the running sum
    float shift = -L::kLift;  // of the exponents
    typename L::Score acc[L::kAcc / L::kScores];
#pragma unroll
    for (int b = 0; b < L::kAcc / L::kScores; ++b) {
#pragma unroll
        for (int i = 0; i < L::kScores; ++i) acc[b][i] = 0.0f;
    }
    auto rescale = [&](float f) {
#pragma unroll
        for (int b = 0; b < L::kAcc / L::kScores; ++b) {
#pragma unroll
            for (int i = 0; i < L::kScores; ++i) acc[b][i] *= f;
        }
    };
    // The tokens of the tile at `first` that this lane's row sees, of the valid ones.
    auto seen = [&](int first, uint32_t there) {
        const int count = limit - first + 1;
        return there & (count >= L::kTokens ? kAll : count <= 0 ? 0u : (1u << count) - 1u);
    };
    auto clear = [&](uint8_t* v, uint32_t there, int start, int step) {
        for (int i = start; i < L::kTokens * L::kChunks; i += step) {
            if (((there >> (i / L::kChunks)) & 1) == 0) reinterpret_cast<u32x4_t*>(v)[i] = u32x4_t{0u, 0u, 0u, 0u};
        }
    };
    // Scores of a tile to weights, and the running values.
    auto soften = [&](typename L::Score& s, int first, uint32_t there) {
        const bool masked = there != kAll || first + L::kTokens - 1 > wave_least;
        const uint32_t mine = masked ? seen(first, there) >> (4 * L::part_of(lane)) : 0u;
        if (masked) {
#pragma unroll
            for (int i = 0; i < L::kScores; ++i) s[i] = (mine & (1u << L::token_of(i))) != 0 ? s[i] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < L::kScores; ++i) top = fmaxf(top, s[i]);
        top = groups_max<L::kRows>(top);
        const float m_new = fmaxf(m, top * c);
        if (__builtin_amdgcn_ballot_w64(m_new > m + L::kLag) != 0) {
            const float f = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.0f : m_new));
            m = m_new;
            l *= f;
            rescale(f);
            shift = (m == -INFINITY ? 0.0f : m) - L::kLift;
        }
#pragma unroll
        for (int i = 0; i < L::kScores; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -shift));
            l += s[i];
        }
    };
    // Values that are not finite, in tiles that some row does not see whole (see
    // BadValues).
    int bad_from = BadValues<kD>::kNone;
    auto guard = [&](uint8_t* v, int first) {
        if (min(first + L::kTokens, w.hi) - 1 <= w.offset + w.first_row / a.per) return;
        bool any = false;
#pragma unroll 1
        for (int i = kShared ? tid : lane; i < L::kTokens * L::kChunks; i += kShared ? kThreads : kWaveSize) {
            u32x4_t four = reinterpret_cast<const u32x4_t*>(v)[i];
            bool here = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool out = (four[e] & 0x7F800000u) == 0x7F800000u;
                here = here || out;
                four[e] = out ? 0u : four[e];
            }
            if (here) reinterpret_cast<u32x4_t*>(v)[i] = four;
            any = any || here;
        }
        if (__builtin_amdgcn_ballot_w64(any) != 0) bad_from = min(bad_from, first);
        if constexpr (kShared) __syncthreads(); else wait_lds();
    };
    auto add_values = [&](uint8_t* v, typename L::Score& s, int first) {
        guard(v, first);
        L::values(v, s, acc, lane);
    };

    if constexpr (!kShared) {
        // The wave's own K and V tile, one copied while the other is used.
        const uint32_t v_dst = lds_own + L::kBytes;
        uint8_t* v = own + L::kBytes;
        if (tiles > 0) {
            look_up(begin);
            copy(lds_own, false);
            copy(v_dst, true);
        }
        for (int i = 0; i < tiles; ++i) {
            const int first = begin + i * kStride;
            const bool more = i + 1 < tiles;
            // K has landed: only V's copies may be in flight. (Copies that no lane takes
            // part in are not issued, so a head narrower than kD waits for all.)
            if (a.head_dim == kD) wait_vm<kCopies>(); else wait_vm<0>();
            const uint32_t there = valid;
            typename L::Score s = L::scores(own, q, lane);
            wait_lds();
            if (more) {
                look_up(first + kStride);
                copy(lds_own, false);
            }
            soften(s, first, there);
            if (more && a.head_dim == kD) wait_vm<kCopies>(); else wait_vm<0>();
            if (there != kAll) {
                clear(v, there, lane, kWaveSize);
                wait_lds();
            }
            add_values(v, s, first);
            wait_lds();
            if (more) copy(v_dst, true);
        }
    } else {
        // A ring of tiles, all but one of them in flight.
        constexpr int kStages = K::kStages;
        uint32_t there[kStages];
        auto issue = [&](int i, int at) {
            look_up(begin + i * kStride);
            there[at] = valid;
            const uint32_t dst = lds_own + static_cast<uint32_t>(at) * K::kTileBytes;
            copy(shared_v ? dst + L::kBytes : dst, shared_v);
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) {
            there[i] = 0;
            if (i < tiles) issue(i, i);
        }
        there[kStages - 1] = 0;
        // The ring's steps written out, so that LDS addresses are constants.
        auto step = [&](auto at, int i) {
            constexpr int kAt = decltype(at)::value;
            // This wave's copies of tile i have landed; those of the tiles behind it
            // (fewer at the end) are in flight.
            if (i + kStages - 2 < tiles && a.head_dim == kD) wait_vm<(kStages - 2) * kCopies>(); else wait_vm<0>();
            bare_barrier();  // and every wave is past tile i - 1, whose place is filled next
            const uint32_t now = there[kAt];
            if (i + kStages - 1 < tiles) issue(i + kStages - 1, (kAt + kStages - 1) % kStages);
            uint8_t* k = lds + kAt * K::kTileBytes;
            uint8_t* v = k + L::kBytes;
            typename L::Score s = L::scores(k, q, lane);
            soften(s, begin + i * kStride, now);
            if (now != kAll) {
                clear(v, now, tid, kThreads);
                __syncthreads();
            }
            add_values(v, s, begin + i * kStride);
            wait_lds();  // before the barrier that lets the tile be overwritten
        };
        static_assert(kStages == 4, "four steps");
        for (int i = 0; i < tiles; i += kStages) {
            step(std::integral_constant<int, 0>{}, i);
            if (i + 1 < tiles) step(std::integral_constant<int, 1>{}, i + 1);
            if (i + 2 < tiles) step(std::integral_constant<int, 2>{}, i + 2);
            if (i + 3 < tiles) step(std::integral_constant<int, 3>{}, i + 3);
        }
    }

    finish<float, kD, CF_CACHE_PLAIN, false, kShared ? kWaves : 1>(a, w, lds, lds_m, lds_l, bad, bad_from, m, l, acc);
}

/// Where a lane's values lie when 16 rows meet 32 tokens in 16 x 16 products.
/// The four groups of 16 lanes hold different dims of the keys (any order that the
/// query shares will do), and of tokens a group has 4 group .. + 3 and the four 16
/// further on: of the scores as of the values, so that weights are in place.
template <typename T, int kD, bool kCodes>
struct FewTile {
    static constexpr int kRows = 16;
    static constexpr int kTokens = 32;
    static constexpr int kSize = kCodes ? 1 : 2;  // bytes of a held value
    using Query = u32x4_t;
    static constexpr int kQueries = kD / 32;  // products of 16 tokens
    __device__ __forceinline__ static int row_of(int lane) { return lane & 15; }
    __device__ __forceinline__ static int part_of(int lane) { return lane >> 4; }
    /// First of the 8 dims of a lane's query piece u. 16 codes are loaded at once.
    __device__ __forceinline__ static int query_dim(int u, int lane) {
        return kCodes ? 64 * (u / 2) + 16 * (lane >> 4) + 8 * (u & 1) : 32 * u + 8 * (lane >> 4);
    }
    static constexpr int kKeyLoads = kD * kSize / 64;  // of 16 tokens, 16 bytes a lane
    /// Values: a lane has kBlocks dims of each of its tokens, in pieces of up to 16 bytes.
    static constexpr int kBlocks = kD / 16;
    static constexpr int kPiece = kBlocks * kSize < 16 ? kBlocks : 16 / kSize;  // dims
    static constexpr int kPieces = kBlocks / kPiece;
    static constexpr int kWords = kPiece * kSize / 4;  // 32-bit words of a piece
    __device__ __forceinline__ static int value_dim(int of16, int block) {
        return kPiece * of16 + block % kPiece + 16 * kPiece * (block / kPiece);
    }
    static constexpr int kOutPitch = kD + 4;
    /// LDS of a wave: a tile's places and scales, at the end the outputs.
    static constexpr int kOwnBytes = kRows * kOutPitch * 4;
    static_assert(kOwnBytes >= kTokens * 16, "8 bytes a place, 4 a scale");
    static constexpr float kLag = Tile<T, kD>::kLag;
    static constexpr float kLift = Tile<T, kD>::kLift;
};

/// Up to 16 kTiles rows, the waves on different tokens. Keys go from memory
/// to the registers of the matrix products: a lane loads the dims that it
/// multiplies. Values are transposed there, by byte permutations of the 8 tokens
/// that a lane needs of each of its dims. So a wave keeps a tile of keys or values
/// in flight while it works on the other, and LDS holds no more than the tile's
/// places and scales. (Widened into LDS instead, and with products of 32 rows, 64
/// sequences of up to 4096 tokens in int8 took 126 us, not 102. Twice the waves a
/// SIMD, in a kernel of their own, changed nothing.)
template <typename T, int kD, cf_cache_format kHeld, bool kSplit, int kTiles>
__device__ void attend_few(const ChunkArgs& a, const Item& w, uint8_t* lds, float (*lds_m)[32], float (*lds_l)[32],
                           BadValues<kD>* bad) {
    constexpr bool kCodes = kHeld != CF_CACHE_PLAIN;
    using L = FewTile<T, kD, kCodes>;
    constexpr int kTokens = L::kTokens;
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & (kWaveSize - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
    const int group = lane >> 4;
    const int of16 = lane & 15;

    // This lane's query rows; those past the end are zeros.
    u32x4_t q[kTiles][L::kQueries];
    [[maybe_unused]] u32x4_t q_low[kTiles][kSplit ? L::kQueries : 1];
    float c[kTiles];
    int limit[kTiles];  // the last token the row sees
    int least = 0x7FFFFFFF;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        const int row = w.first_row + n * L::kRows + of16;
        const bool inside = row < w.rows;
        const int token = inside ? row / a.per : 0;
        limit[n] = inside ? w.offset + token : -1;
        least = min(least, inside ? limit[n] : 0x7FFFFFFF);
        c[n] = load_query<L, T, kCodes, kSplit>(a, w, inside, token, inside ? row % a.per : 0, lane, q[n], q_low[n]);
    }
    // The smallest of the limits: tiles up to it need no mask.
#pragma unroll
    for (int d = 1; d < L::kRows; d <<= 1) least = min(least, __shfl_xor(least, d));
    const int wave_least = __builtin_amdgcn_readfirstlane(least);

    uint8_t* const own = lds + wave * L::kOwnBytes;
    // Tiles begin at multiples of kTokens (ranges do).
    const int begin = w.lo + wave * kTokens;
    constexpr int kStride = kWaves * kTokens;
    const int tiles = begin < w.hi ? (w.hi - begin + kStride - 1) / kStride : 0;
    const int last_block = static_cast<int>(static_cast<uint32_t>(w.hi - 1) / a.block_size);
    auto block_of = [&](int t) {
        return static_cast<int>(a.block_shift >= 0 ? static_cast<uint32_t>(t) >> a.block_shift
                                                   : static_cast<uint32_t>(t) / a.block_size);
    };
    // 64 entries of the block table in lane registers: looking a page up is then
    // no load that would have to wait behind the tiles'.
    int window_base = block_of(begin < w.hi ? begin : w.lo);
    uint32_t window = w.table[min(window_base + lane, last_block)];
    uint64_t* const places = reinterpret_cast<uint64_t*>(own);  // of the tile looked up last, in bytes
    float* const scales = reinterpret_cast<float*>(own + kTokens * 8);  // of the tile at hand: keys', values'
    const uint64_t head_bytes = static_cast<uint64_t>(w.kv_head) * a.head_dim * L::kSize;
    uint32_t row = 0;    // of the cache: token lane % kTokens of the tile looked up last, 0 where it is not there
    uint32_t there = 0;  // its tokens that are, a bit each
    auto look_up = [&](int first) {
        const int last = min(first + kTokens, w.hi) - 1;
        if (block_of(last) >= window_base + kWaveSize) {
            window_base = block_of(first);
            window = w.table[min(window_base + lane, last_block)];
            asm volatile("" : "+v"(window));  // waited for here, not behind the branch
        }
        const int t = min(first + (lane & (kTokens - 1)), last);
        const int block = block_of(t);
        const uint32_t page = static_cast<uint32_t>(__shfl(static_cast<int>(window), block - window_base));
        const bool is = page < a.pages && first + (lane & (kTokens - 1)) < w.hi;
        row = is ? page * a.block_size + (static_cast<uint32_t>(t) - static_cast<uint32_t>(block) * a.block_size) : 0u;
        there = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(is));
        if (lane < kTokens) places[lane] = ((static_cast<uint64_t>(row) * a.token_pieces) << 4) + head_bytes;
    };

    // A row's end that a narrow head lacks is read from the row's beginning instead.
    const int row_bytes = a.head_dim * L::kSize;
    const bool whole = a.head_dim == kD;
    u32x4_t keys[2][L::kKeyLoads];
    auto load_keys = [&]() {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint8_t* from = a.k_cache + places[16 * s + of16];
#pragma unroll
            for (int n = 0; n < L::kKeyLoads; ++n) {
                const int at = 64 * n + 16 * group;
                keys[s][n] = *reinterpret_cast<const u32x4_t*>(from + (at < row_bytes ? at : 0));
            }
        }
    };
    typedef uint32_t piece_t __attribute__((ext_vector_type(L::kWords == 1 ? 2 : L::kWords)));  // (one word: see below)
    uint32_t values[8][L::kPieces][L::kWords];
    auto load_values = [&]() {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint8_t* from = a.v_cache + places[16 * (j >> 2) + 4 * group + (j & 3)];
#pragma unroll
            for (int n = 0; n < L::kPieces; ++n) {
                const int at = (of16 + 16 * n) * L::kPiece * L::kSize;
                const uint8_t* piece = from + (at < row_bytes ? at : 0);
                if constexpr (L::kWords == 1) {
                    values[j][n][0] = *reinterpret_cast<const uint32_t*>(piece);
                } else {
                    const piece_t words = *reinterpret_cast<const piece_t*>(piece);
#pragma unroll
                    for (int e = 0; e < L::kWords; ++e) values[j][n][e] = words[e];
                }
            }
        }
    };
    // Lanes below kTokens: a key's scale, the others a value's.
    [[maybe_unused]] float scale = 0.0f;
    // (A choice between the two pointers would be made in memory.)
    [[maybe_unused]] const int64_t scale_from =
        w.kv_head + (lane < kTokens ? 0 : (reinterpret_cast<int64_t>(a.v_scales) - reinterpret_cast<int64_t>(a.k_scales)) / 4);
    [[maybe_unused]] auto load_scale = [&]() {
        scale = a.k_scales[static_cast<int64_t>(static_cast<uint64_t>(row) * static_cast<uint32_t>(a.kv_heads)) + scale_from];
    };

    float m[kTiles];      // the row's running maximum
    float l[kTiles];      // this lane's share of the running sum
    float shift[kTiles];  // of the exponents
    [[maybe_unused]] int unit[kTiles];
    f32x4_t acc[kTiles][L::kBlocks];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
        shift[n] = -L::kLift;
        unit[n] = kLeastUnit;
#pragma unroll
        for (int b = 0; b < L::kBlocks; ++b) acc[n][b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    auto multiply = [](const u32x4_t& x, const u32x4_t& y, const f32x4_t& sum) {
        if constexpr (std::is_same<T, bf16_t>::value) {
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), __builtin_bit_cast(bf16x8_t, y),
                                                           sum, 0, 0, 0);
        } else {
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, x), __builtin_bit_cast(f16x8_t, y),
                                                          sum, 0, 0, 0);
        }
    };
    constexpr int kScores = 8;  // a lane's, tokens 4 group + (i & 3) + 16 (i >> 2)
    auto token_of = [](int i) { return (i & 3) + 16 * (i >> 2); };

    [[maybe_unused]] int bad_from = BadValues<kD>::kNone;
    if (tiles > 0) {
        look_up(begin);
        load_keys();
        if constexpr (kCodes) load_scale();
        __builtin_amdgcn_sched_barrier(0);  // in the loop's order
        load_values();
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
        const int first = begin + i * kStride;
        const uint32_t now = there;
        const bool masked = now != 0xFFFFFFFFu || first + kTokens - 1 > wave_least;
        if constexpr (kCodes) {
            // (A row that sees none of the tokens that another has met sees none of these.)
            int met = unit[0];
            if constexpr (kTiles > 1) met = max(met, unit[kTiles - 1]);
            const bool matters = __builtin_amdgcn_ballot_w64(met > 0) == 0;
            if (lane >= kTokens) {
                scale = value_scale<kHeld>(scale, matters, [&]() { return a.v_cache + places[lane - kTokens]; }, row_bytes);
            }
            scales[lane] = scale;
        }
        // The next tile; behind the last one its tokens are not there, and every lane reads
        // row 0 of the cache, for nobody: loads behind a branch would be waited for
        // wherever one of the others is.
        look_up(first + kStride);

        // Scores.
        f32x4_t s[kTiles][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int n = 0; n < kTiles; ++n) s[n][h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < L::kKeyLoads; ++i) {
                u32x4_t part[kCodes ? 2 : 1];
                u32x4_t raw = keys[h][i];
                if (!whole) raw = 64 * i + 16 * group < row_bytes ? raw : u32x4_t{0u, 0u, 0u, 0u};
                if constexpr (kCodes) widen16<kHeld>(raw, part[0], part[1]); else part[0] = raw;
#pragma unroll
                for (int e = 0; e < (kCodes ? 2 : 1); ++e) {
                    const int u = kCodes ? 2 * i + e : i;
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        s[n][h] = multiply(part[e], q[n][u], s[n][h]);
                        if constexpr (kSplit) s[n][h] = multiply(part[e], q_low[n][u], s[n][h]);
                    }
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_keys();
        if constexpr (kCodes) load_scale();
        __builtin_amdgcn_sched_barrier(0);

        // Weights.
        u32x4_t weights[kTiles];
        [[maybe_unused]] u32x4_t rest[kTiles];  // what fp16 weights leave (kSplit)
        [[maybe_unused]] float of_key[kScores], of_value[kScores];
        if constexpr (kCodes) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4_t k4 = *reinterpret_cast<const f32x4_t*>(scales + 16 * h + 4 * group);
                const f32x4_t v4 = *reinterpret_cast<const f32x4_t*>(scales + kTokens + 16 * h + 4 * group);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    of_key[4 * h + e] = k4[e];
                    of_value[4 * h + e] = v4[e];
                }
            }
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            float x[kScores];
            [[maybe_unused]] float by[kScores];
#pragma unroll
            for (int i = 0; i < kScores; ++i) {
                x[i] = s[n][i >> 2][i & 3];
                if constexpr (kCodes) {
                    x[i] *= of_key[i];
                    by[i] = of_value[i];
                }
            }
            if (masked) {
                const int count = limit[n] - first + 1;
                const uint32_t sees = (now & (count >= kTokens ? 0xFFFFFFFFu : count <= 0 ? 0u : (1u << count) - 1u)) >> (4 * group);
#pragma unroll
                for (int i = 0; i < kScores; ++i) {
                    const bool see = (sees & (1u << token_of(i))) != 0;
                    x[i] = see ? x[i] : -INFINITY;
                    // What a row does not see may be NaN, or far above its own scales.
                    if constexpr (kCodes) by[i] = see ? by[i] : 0.0f;
                }
            }
            // Probabilities of codes are taken relative to a power of two 2^unit above all
            // scales of values that the row met, sums too: times a scale they are at most
            // 2^(kLift + kLag), as fp16 has to hold them.
            int most = kLeastUnit;
            if constexpr (kCodes) {
                float above = fabsf(by[0]);
#pragma unroll
                for (int i = 1; i < kScores; ++i) above = fmaxf(above, fabsf(by[i]));
                most = unit_above(groups_max<L::kRows>(above));
            }
            float top = x[0];
#pragma unroll
            for (int i = 1; i < kScores; ++i) top = fmaxf(top, x[i]);
            const float m_new = fmaxf(m[n], groups_max<L::kRows>(top) * c[n]);
            if (__builtin_amdgcn_ballot_w64(m_new > m[n] + L::kLag || (kCodes && most > unit[n])) != 0) {
                float f = __builtin_amdgcn_exp2f(m[n] - (m_new == -INFINITY ? 0.0f : m_new));
                m[n] = m_new;
                if constexpr (kCodes) {
                    const int old = unit[n];
                    unit[n] = most > old ? most : old;
                    f = __builtin_amdgcn_ldexpf(f, old - unit[n]);
                }
                l[n] *= f;
#pragma unroll
                for (int b = 0; b < L::kBlocks; ++b) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[n][b][i] *= f;
                }
                shift[n] = (m[n] == -INFINITY ? 0.0f : m[n]) + (kCodes ? static_cast<float>(unit[n]) : 0.0f) - L::kLift;
            }
#pragma unroll
            for (int i = 0; i < kScores; ++i) {
                x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c[n], -shift[n]));
                l[n] += x[i];
                if constexpr (kCodes) x[i] *= by[i];
                // One value for both fp16 parts: the product could be rounded to fp16 at once.
                if constexpr (kSplit) {
                    float y = x[i];
                    asm volatile("" : "+v"(y));
                    x[i] = y;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (std::is_same<T, bf16_t>::value) {
                    weights[n][e] = f32x2_to_bf16x2_bits(x[2 * e], x[2 * e + 1]);
                } else {
                    typedef _Float16 f16x2_v __attribute__((ext_vector_type(2)));
                    const f16x2_v high = {static_cast<_Float16>(x[2 * e]), static_cast<_Float16>(x[2 * e + 1])};
                    weights[n][e] = __builtin_bit_cast(uint32_t, high);
                    if constexpr (kSplit) {
                        rest[n][e] = __builtin_bit_cast(
                            uint32_t, f16x2_v{static_cast<_Float16>(x[2 * e] - static_cast<float>(high[0])),
                                              static_cast<_Float16>(x[2 * e + 1] - static_cast<float>(high[1]))});
                    }
                }
            }
        }

        // Values. Those that are not finite, in tiles that some row does not see whole (see
        // BadValues).
        if (kHeld != CF_CACHE_INT8 && masked) {
            // Adding `one` to an exponent of ones, or to e4m3's NaN, carries into the sign.
            constexpr uint32_t one = kCodes ? 0x01010101u : std::is_same<T, f16_t>::value ? 0x04000400u : 0x00800080u;
            constexpr uint32_t sign = kCodes ? 0x80808080u : 0x80008000u;
            uint32_t any = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
#pragma unroll
                for (int p = 0; p < L::kPieces; ++p) {
#pragma unroll
                    for (int word = 0; word < L::kWords; ++word) {
                        const uint32_t out = ((values[j][p][word] & (sign - one)) + one) & sign;
                        // (What is read in place of a token that is not there does not count.)
                        any |= (now >> (4 * group + token_of(j)) & 1) != 0 ? out : 0;
                        values[j][p][word] &= ~((out >> (kCodes ? 7 : 15)) * (kCodes ? 0xFFu : 0xFFFFu));
                    }
                }
            }
            if (__builtin_amdgcn_ballot_w64(any != 0) != 0) bad_from = min(bad_from, first);
        }
#pragma unroll
        for (int p = 0; p < L::kPieces; ++p) {
#pragma unroll
            for (int word = 0; word < L::kWords; ++word) {
#pragma unroll
                for (int half = 0; half < 2 / L::kSize; ++half) {  // two dims at a time, for the registers
                    __builtin_amdgcn_sched_barrier(0);
                    u32x4_t part[2];  // of a dim each: the lane's 8 tokens
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x0 = values[2 * e][p][word];
                        const uint32_t x1 = values[2 * e + 1][p][word];
                        if constexpr (kCodes) {
                            const uint2 two = widen4<kHeld>(__builtin_amdgcn_perm(x1, x0, half == 0 ? 0x05010400u : 0x07030602u));
                            part[0][e] = two.x;
                            part[1][e] = two.y;
                        } else {
                            part[0][e] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
                            part[1][e] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
                        }
                    }
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        const int b = p * L::kPiece + word * (4 / L::kSize) + 2 * half + d;
#pragma unroll
                        for (int n = 0; n < kTiles; ++n) {
                            acc[n][b] = multiply(part[d], weights[n], acc[n][b]);
                            if constexpr (kSplit) acc[n][b] = multiply(part[d], rest[n], acc[n][b]);
                        }
                    }
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_values();
    }

    // The waves' outputs joined, 16 rows at a time.
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        if (group == 0) {
            lds_m[wave][n * L::kRows + of16] = m[n] + (kCodes ? static_cast<float>(unit[n]) : 0.0f);
            lds_l[wave][n * L::kRows + of16] = l[n];
        }
    }
    if (kHeld != CF_CACHE_INT8 && lane == 0) bad->from[wave] = bad_from;
    bool any_bad = false;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        if (w.first_row + n * L::kRows >= w.rows) break;
        __syncthreads();
        float* mine = reinterpret_cast<float*>(own) + of16 * L::kOutPitch;
#pragma unroll
        for (int b = 0; b < L::kBlocks; b += 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *reinterpret_cast<f32x4_t*>(mine + L::value_dim(4 * group + i, b)) =
                    f32x4_t{acc[n][b][i], acc[n][b + 1][i], acc[n][b + 2][i], acc[n][b + 3][i]};
            }
        }
        __syncthreads();
        if (n == 0) {
            if constexpr (kHeld != CF_CACHE_INT8) any_bad = bad->template find<T, kHeld>(a, w);
        }
        for (int i = tid; i < L::kRows * (kD / 4); i += kThreads) {
            const int r = i / (kD / 4);
            const int dim = i % (kD / 4) * 4;
            const int out = w.first_row + n * L::kRows + r;
            if (out >= w.rows || dim >= a.head_dim) continue;
            Joined j = join_waves<kWaves, 1>(reinterpret_cast<const float*>(lds) + r * L::kOutPitch + dim,
                                             L::kOwnBytes / 4, lds_m, lds_l, n * L::kRows + r);
            if (any_bad) bad->add_to(j.sum, dim, w.offset + out / a.per);
            put<T, kCodes, kSplit>(a, w, out, dim, j.m, j.l, j.sum);
        }
    }
}

/// LDS of attend_rows: two tiles of 64 tokens of K and of V, and for codes their
/// scales (K's, V's, and the exponent above V's).
template <typename T, int kD, cf_cache_format kHeld>
struct RowsKind {
    using L = Tile<T, kD>;
    static constexpr bool kCodes = kHeld != CF_CACHE_PLAIN;
    static constexpr int kTokens = 64;
    static constexpr int kOperand = kTokens * L::kRowBytes;
    static constexpr int kScales = 2 * kTokens + 4;  // floats of a tile
    static constexpr int kScalesAt = 4 * kOperand;
    static constexpr int lds_bytes() {
        constexpr int tiles = kScalesAt + (kCodes ? 2 * kScales * 4 : 0);
        constexpr int outputs = kWaves * L::kRows * L::kOutPitch * 4;
        return tiles > outputs ? tiles : outputs;
    }
};

/// 16-bit tiles of more than 32 rows, 64 tokens a step. The waves take different
/// rows, with kHalves = 2 (up to 64 rows) two of them the first half of the tokens
/// and two the second. In plain
/// caches the next step's scores are formed while this one's are made
/// probabilities, so that a wave has work for the matrix cores beside its vector
/// instructions (a 2048-token prompt 68 us, without it and the reads ahead 75);
/// codes, which need more of those, leave no registers for it: 512 tokens each of
/// three sequences of 4000 in e4m3, next to 41 single ones, take 202 us with the
/// vector units 43% and the matrix cores 18% busy.
template <typename T, int kD, cf_cache_format kHeld, bool kSplit, int kHalves>
__device__ void attend_rows(const ChunkArgs& a, const Item& w, uint8_t* lds, float (*lds_m)[32], float (*lds_l)[32],
                            BadValues<kD>* bad) {
    using K = RowsKind<T, kD, kHeld>;
    using L = typename K::L;
    using Score = typename L::Score;
    constexpr bool kCodes = K::kCodes;
    constexpr int kTokens = K::kTokens;
    static_assert(!L::kWide && L::kTokens == 32 && L::kRows == 32, "two halves of 32 tokens");
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & (kWaveSize - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
    constexpr int kRowWaves = kWaves / kHalves;
    const int mine = kHalves == 1 ? 0 : wave / kRowWaves;  // this wave's half of a tile, or the first of both
    const int row = w.first_row + wave % kRowWaves * L::kRows + L::row_of(lane);
    const bool inside = row < w.rows;
    const int token = inside ? row / a.per : 0;
    const int limit = inside ? w.offset + token : -1;  // the last token the row sees
    typename L::Query q[L::kQueries];
    [[maybe_unused]] typename L::Query q_low[kSplit ? L::kQueries : 1];
    const float c = load_query<L, T, kCodes, kSplit>(a, w, inside, token, inside ? row % a.per : 0, lane, q, q_low);
    // The smallest limit of the rows: tiles up to it need no mask.
    const int tile_least = w.offset + w.first_row / a.per;
    if (a.head_dim < kD) {  // the copies leave the end of every row as it is
        for (int i = tid; i < 4 * K::kOperand / 16; i += kThreads) {
            reinterpret_cast<u32x4_t*>(lds)[i] = u32x4_t{0u, 0u, 0u, 0u};
        }
        __syncthreads();
    }

    const int tiles = (w.hi - w.lo + kTokens - 1) / kTokens;
    const int last_block = static_cast<int>(static_cast<uint32_t>(w.hi - 1) / a.block_size);
    auto block_of = [&](int t) {
        return static_cast<int>(a.block_shift >= 0 ? static_cast<uint32_t>(t) >> a.block_shift
                                                   : static_cast<uint32_t>(t) / a.block_size);
    };
    // 64 entries of the block table in lane registers (see attend).
    int window_base = block_of(w.lo);
    uint32_t window = w.table[min(window_base + lane, last_block)];
    constexpr uint64_t kAll = ~uint64_t{0};
    struct Place {
        uint32_t row;    // of the cache: token `lane` of the tile, 0 where it is not there
        uint32_t piece;  // where it begins, in 16 bytes
        uint64_t there;  // a bit per token
    };
    auto look_up = [&](int tile) {
        const int first = w.lo + tile * kTokens;
        const int last = min(first + kTokens, w.hi) - 1;
        if (block_of(last) >= window_base + kWaveSize) {
            window_base = block_of(first);
            window = w.table[min(window_base + lane, last_block)];
            asm volatile("" : "+v"(window));  // waited for here, not behind the branch
        }
        const int t = min(first + lane, last);
        const int block = block_of(t);
        const uint32_t page = static_cast<uint32_t>(__shfl(static_cast<int>(window), block - window_base));
        const bool there = page < a.pages && first + lane < w.hi;
        const uint32_t row = page * a.block_size + (static_cast<uint32_t>(t) - static_cast<uint32_t>(block) * a.block_size);
        return Place{there ? row : 0u, there ? row * a.token_pieces : 0u, __builtin_amdgcn_ballot_w64(there)};
    };

    const uint32_t lds_base = __builtin_amdgcn_readfirstlane(lds_address(lds));
    const int held_size = kCodes ? 1 : static_cast<int>(sizeof(T));
    const uint64_t head_bytes = static_cast<uint64_t>(w.kv_head) * a.head_dim * held_size;
    const int row_pieces = a.head_dim * held_size / 16;
    // This wave's share of a tile: tokens 16 wave .. + 15 of K and of V.
    constexpr int kMine = kTokens / kWaves;
    constexpr int kPerCopy = kWaveSize / L::kChunks;  // plain: tokens a copy
    constexpr int kCopies = kMine / kPerCopy;
    constexpr int kBatch = kCopies < 4 ? kCopies : 4;
    const bool whole = a.head_dim == kD;
    // The lane's byte within a row of copy n (its order of pieces recurs after 16
    // tokens).
    [[maybe_unused]] auto piece_of = [&](int n, bool is_v) {
        const int r = n * kPerCopy + lane / L::kChunks;
        return (lane % L::kChunks) ^ (is_v ? L::v_swizzle(r) : L::k_swizzle(r));
    };
    [[maybe_unused]] auto send = [&](const Place& p, int slot, bool is_v) {
        const uint8_t* base = (is_v ? a.v_cache : a.k_cache) + head_bytes;
        const uint32_t dst = lds_base + static_cast<uint32_t>((is_v ? 2 + slot : slot) * K::kOperand + wave * kMine * L::kRowBytes);
#pragma unroll
        for (int n0 = 0; n0 < kCopies; n0 += kBatch) {
            uint32_t at[kBatch];
            const uint8_t* from[kBatch];
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                at[n] = static_cast<uint32_t>(
                    __shfl(static_cast<int>(p.piece), wave * kMine + (n0 + n) * kPerCopy + lane / L::kChunks));
            }
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                from[n] = base + (static_cast<uint64_t>(at[n] + static_cast<uint32_t>(piece_of(n0 + n, is_v))) << 4);
            }
            if constexpr (kBatch == 4) {
                if (whole) {
                    copy16x4_to_lds(from[0], from[1] - kCopyBytes, from[2] - 2 * kCopyBytes, from[3] - 3 * kCopyBytes,
                                    dst + static_cast<uint32_t>(n0) * 16 * kWaveSize);
                    continue;
                }
            }
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                if (piece_of(n0 + n, is_v) < row_pieces) {
                    copy16_to_lds(from[n], dst + static_cast<uint32_t>(n0 + n) * 16 * kWaveSize);
                }
            }
        }
    };
    // 8-bit caches: 16 codes a lane and load; wave 0 has K's scales, wave 1 V's.
    constexpr int kCodeLanes = kD / 16;                  // per token
    constexpr int kCodeTokens = kWaveSize / kCodeLanes;  // per load
    constexpr int kLoads = kCodes ? kMine / kCodeTokens : 1;
    static_assert(!kCodes || kMine % kCodeTokens == 0, "whole loads");
    struct Codes {
        u32x4_t raw[kLoads];
    };
    [[maybe_unused]] Codes k_codes, v_codes;
    [[maybe_unused]] float raw_scale = 0.0f;
    // Heads of 256 have no registers for places in rows and LDS that stay the same from
    // step to step: kept, they are spilled (three chunks of 512 behind 3488 in e4m3
    // 710 us, computed again 615). The lane that they come from is hidden.
    [[maybe_unused]] auto step_lane = [&]() {
        int l2 = lane;
        if constexpr (kD > 128) asm volatile("" : "+v"(l2));
        return l2;
    };
    [[maybe_unused]] auto load_codes = [&](Codes& to, const Place& p, bool is_v) {
        const int at_lane = step_lane();
        const uint8_t* base = (is_v ? a.v_cache : a.k_cache) + head_bytes;
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int r = wave * kMine + n * kCodeTokens + at_lane / kCodeLanes;
            const uint32_t at = static_cast<uint32_t>(__shfl(static_cast<int>(p.piece), r));
            // A row that is not there, or the end of a narrow one, is read from the cache's
            // or row's beginning instead and not used.
            const int piece = at_lane % kCodeLanes < row_pieces ? at_lane % kCodeLanes : 0;
            to.raw[n] = *reinterpret_cast<const u32x4_t*>(base + (static_cast<uint64_t>(at + static_cast<uint32_t>(piece)) << 4));
        }
        if (wave == (is_v ? 1 : 0)) {
            // A value's scale that is not finite makes its key's one NaN and is 0 itself:
            // rows that see the token are NaN, the others never meet it.
            const int64_t at = static_cast<int64_t>(p.row) * a.kv_heads + w.kv_head;
            const bool there = ((p.there >> lane) & 1) != 0;
            const float of_v = there ? a.v_scales[at] : 0.0f;
            const bool finite = __builtin_isfinite(of_v);
            if (is_v) {
                raw_scale = finite ? of_v : 0.0f;
            } else {
                raw_scale = there ? a.k_scales[at] : 0.0f;
                raw_scale = finite ? raw_scale : __uint_as_float(0x7FC00000u);
            }
        }
    };
    [[maybe_unused]] auto scales_of = [&](int tile) {
        return reinterpret_cast<float*>(lds + K::kScalesAt) + (tile & 1) * K::kScales;
    };
    [[maybe_unused]] int unit = kLeastUnit;  // see attend_few
    [[maybe_unused]] auto store_codes = [&](const Codes& from, int tile, bool is_v) {
        const int at_lane = step_lane();
        uint8_t* to = lds + ((is_v ? 2 : 0) + (tile & 1)) * K::kOperand;
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int r = wave * kMine + n * kCodeTokens + at_lane / kCodeLanes;
            const int sw = is_v ? L::v_swizzle(r) : L::k_swizzle(r);
            const int piece = at_lane % kCodeLanes;
            u32x4_t lo, hi;
            widen16<kCodes ? kHeld : CF_CACHE_INT8>(from.raw[n], lo, hi);
            if (piece < row_pieces) {
                *reinterpret_cast<u32x4_t*>(to + r * L::kRowBytes + (((2 * piece) ^ sw) << 4)) = lo;
                *reinterpret_cast<u32x4_t*>(to + r * L::kRowBytes + (((2 * piece + 1) ^ sw) << 4)) = hi;
            }
        }
        if (wave == (is_v ? 1 : 0)) {
            float* scales = scales_of(tile);
            if (is_v) {
                // (A row that sees none of the tokens that another has met sees none of these;
                // the waves with later rows have met what this one has.)
                const bool matters = __builtin_amdgcn_ballot_w64(unit > 0) == 0;
                raw_scale = value_scale<kHeld>(raw_scale, matters, [&]() {
                    // (Looked up again: a register less to keep.)
                    const uint32_t t = static_cast<uint32_t>(w.lo + tile * kTokens + lane);
                    const uint32_t block = t / a.block_size;
                    const uint32_t row = w.table[block] * a.block_size + (t - block * a.block_size);
                    return a.v_cache + head_bytes + (static_cast<uint64_t>(row * a.token_pieces) << 4);
                }, a.head_dim);
            }
            scales[(is_v ? kTokens : 0) + lane] = raw_scale;
            if (is_v) {
                const float top = wave_reduce_f32<MaxF32>(fabsf(raw_scale));
                if (lane == 0) reinterpret_cast<int*>(scales)[2 * kTokens] = unit_above(top);
            }
        }
    };

    float m = -INFINITY;  // the row's running maximum
    float l = 0.0f;       // this lane's share of the running sum
    float shift = -L::kLift;
    Score acc[L::kAcc / L::kScores];
#pragma unroll
    for (int b = 0; b < L::kAcc / L::kScores; ++b) {
#pragma unroll
        for (int i = 0; i < L::kScores; ++i) acc[b][i] = 0.0f;
    }
    auto scores = [&](int slot, int half) {
        const uint8_t* k = lds + slot * K::kOperand + half * 32 * L::kRowBytes;
        Score s = L::scores(k, q, lane);
        if constexpr (kSplit) {
            const Score low = L::scores(k, q_low, lane);
#pragma unroll
            for (int i = 0; i < L::kScores; ++i) s[i] += low[i];
        }
        return s;
    };
    auto scale_scores = [&](Score& s, int tile, int half) {
        if constexpr (kCodes) {
            const float* scales = scales_of(tile) + 32 * half + 4 * L::part_of(lane);
#pragma unroll
            for (int i = 0; i < L::kScores; ++i) s[i] *= scales[L::token_of(i)];
        }
    };
    auto rescale_to = [&](float top, int most) {
        const float m_new = fmaxf(m, groups_max<L::kRows>(top) * c);
        if (__builtin_amdgcn_ballot_w64(m_new > m + L::kLag || (kCodes && most > unit)) != 0) {
            float f = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.0f : m_new));
            m = m_new;
            if constexpr (kCodes) {
                const int old = unit;
                unit = most > unit ? most : unit;
                f = __builtin_amdgcn_ldexpf(f, old - unit);
            }
            l *= f;
#pragma unroll
            for (int b = 0; b < L::kAcc / L::kScores; ++b) {
#pragma unroll
                for (int i = 0; i < L::kScores; ++i) acc[b][i] *= f;
            }
            shift = (m == -INFINITY ? 0.0f : m) + (kCodes ? static_cast<float>(unit) : 0.0f) - L::kLift;
        }
    };
    auto largest = [&](const Score& s0, const Score& s1) {
        float top = fmaxf(s0[0], s1[0]);
#pragma unroll
        for (int i = 1; i < L::kScores; ++i) top = fmaxf(fmaxf(top, s0[i]), s1[i]);
        return top;
    };
    // Scores to weights.
    auto weigh = [&](Score& s, int tile, int half) {
        [[maybe_unused]] const float* by = scales_of(tile) + kTokens + 32 * half + 4 * L::part_of(lane);
#pragma unroll
        for (int i = 0; i < L::kScores; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -shift));
            l += s[i];
            if constexpr (kCodes) s[i] *= by[L::token_of(i)];
            // One value for both fp16 parts: the product could be rounded to fp16 at once.
            if constexpr (kSplit) {
                float x = s[i];
                asm volatile("" : "+v"(x));
                s[i] = x;
            }
        }
    };
    // Values for the product of tokens 32 half + 16 u .. + 15 with dims 32 b .. + 31.
    constexpr int kPieces = 2 * (kD / 32);  // of a half
    static_assert(kPieces >= 4, "as many as are read ahead");
    auto read_values = [&](int slot, int half, int n) {
        const int u = n & 1;
        const int b = n >> 1;
        const int j = lane & 15;
        const int r = 16 * u + 4 * (lane >> 5) + (j >> 2);
        const int piece = (4 * b + 2 * ((lane >> 4) & 1) + ((j & 3) >> 1)) ^ L::v_swizzle(r);
        uint8_t* at = lds + (2 + slot) * K::kOperand + half * 32 * L::kRowBytes + r * L::kRowBytes + (piece << 4) + (j & 1) * 8;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(lds_u8_t*)at);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(lds_u8_t*)(at + 8 * L::kRowBytes));
        return __builtin_bit_cast(u32x4_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    struct Weights {
        u32x4_t part[2];  // of 16 tokens each
    };
    auto pack = [&](const Score& s) {
        Weights w2;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p0 = s[8 * u + 2 * e];
                const float p1 = s[8 * u + 2 * e + 1];
                if constexpr (std::is_same<T, bf16_t>::value) {
                    w2.part[u][e] = f32x2_to_bf16x2_bits(p0, p1);
                } else {
                    typedef _Float16 f16x2_v __attribute__((ext_vector_type(2)));
                    w2.part[u][e] = __builtin_bit_cast(uint32_t, f16x2_v{static_cast<_Float16>(p0), static_cast<_Float16>(p1)});
                }
            }
        }
        return w2;
    };
    // What fp16 weights leave of s (kSplit).
    auto rest_of = [&](const Score& s) {
        Score r;
#pragma unroll
        for (int i = 0; i < L::kScores; ++i) r[i] = s[i] - static_cast<float>(static_cast<_Float16>(s[i]));
        return r;
    };
    auto multiply = [&](const u32x4_t& v, const u32x4_t& p, Score& sum) {
        if constexpr (std::is_same<T, bf16_t>::value) {
            sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, p),
                                                          sum, 0, 0, 0);
        } else {
            sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, v), __builtin_bit_cast(f16x8_t, p),
                                                         sum, 0, 0, 0);
        }
    };
    // Values of tokens that are not there, and in tiles that some row does not see
    // whole those that are not finite (see BadValues), to 0.
    [[maybe_unused]] int bad_from = BadValues<kD>::kNone;
    [[maybe_unused]] auto sanitise = [&](int slot, int first, uint64_t there) {
        const bool hidden = min(first + kTokens, w.hi) - 1 > tile_least;
        if (there == kAll && !hidden) return;
        constexpr uint32_t kExponent = std::is_same<T, f16_t>::value ? 0x7C00u : 0x7F80u;
        u32x4_t* v = reinterpret_cast<u32x4_t*>(lds + (2 + slot) * K::kOperand);
        bool any = false;
#pragma unroll 1
        for (int i = tid; i < kTokens * L::kChunks; i += kThreads) {
            u32x4_t four = v[i];
            bool here = false;
            const bool out = ((there >> (i / L::kChunks)) & 1) == 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool low = hidden && (four[e] & kExponent) == kExponent;
                const bool high = hidden && (four[e] >> 16 & kExponent) == kExponent;
                here = here || low || high;
                four[e] = out ? 0u : four[e] & (low ? 0xFFFF0000u : 0xFFFFFFFFu) & (high ? 0xFFFFu : 0xFFFFFFFFu);
            }
            if (here || out) v[i] = four;
            any = any || (here && !out);
        }
        if (__builtin_amdgcn_ballot_w64(any) != 0) bad_from = min(bad_from, first);
        __syncthreads();
    };

    Place here = look_up(0);  // of tile i
    Place next{};       // of tile i + 1
    if (tiles > 1) next = look_up(1);
    Score s0, s1;
    if constexpr (kCodes) {
        load_codes(k_codes, here, false);
        load_codes(v_codes, here, true);
        store_codes(k_codes, 0, false);
        store_codes(v_codes, 0, true);
        if (tiles > 1) {
            load_codes(k_codes, next, false);
            load_codes(v_codes, next, true);
        }
    } else {
        send(here, 0, false);
        send(here, 0, true);
        if (tiles > 1) send(next, 1, false);
        wait_vm<0>();
        bare_barrier();
        s0 = scores(0, mine);
        if constexpr (kHalves == 1) s1 = scores(0, 1);
    }
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
        const int at = i & 1;
        const int first = w.lo + i * kTokens;
        Place far{};
        [[maybe_unused]] Score n0, n1;
        // Codes: tile i is in LDS, tile i + 1 in registers, loaded an iteration ago.
        // Plain: K of tile i + 1 and V of tile i are in LDS. The places that the
        // iteration before left are free.
        if constexpr (!kCodes) wait_vm<0>();
        wait_lds();
        bare_barrier();
        if constexpr (kCodes) {
            if (i + 1 < tiles) {
                store_codes(k_codes, i + 1, false);
                store_codes(v_codes, i + 1, true);
            }
            if (i + 2 < tiles) {
                far = look_up(i + 2);
                load_codes(k_codes, far, false);
                load_codes(v_codes, far, true);
            }
            s0 = scores(at, mine);
            if constexpr (kHalves == 1) s1 = scores(at, 1);
        } else {
            if (i + 2 < tiles) {
                far = look_up(i + 2);
                send(far, at, false);
            }
            if (i + 1 < tiles) send(next, at ^ 1, true);
        }
        // (Behind the last tile these are scores of nothing, used by nobody.)
        if constexpr (!kCodes) n0 = scores(at ^ 1, mine);
        scale_scores(s0, i, mine);
        if constexpr (kHalves == 1) scale_scores(s1, i, 1); else s1 = s0;  // (one place, for the maximum)
        int most = 0;
        if constexpr (kCodes) most = reinterpret_cast<const int*>(scales_of(i))[2 * kTokens];
        const bool masked = here.there != kAll || first + kTokens - 1 > tile_least;
        [[maybe_unused]] uint64_t sees = kAll;
        if (masked) {
            const int count = limit - first + 1;
            sees = here.there & (count >= kTokens ? kAll : count <= 0 ? 0u : (uint64_t{1} << count) - 1u);
            const uint32_t sees0 = static_cast<uint32_t>(sees >> (32 * mine)) >> (4 * L::part_of(lane));
            const uint32_t sees1 = static_cast<uint32_t>(sees >> 32) >> (4 * L::part_of(lane));
            float above = 0.0f;
#pragma unroll
            for (int e = 0; e < L::kScores; ++e) {
                const bool see0 = (sees0 & (1u << L::token_of(e))) != 0;
                const bool see1 = (sees1 & (1u << L::token_of(e))) != 0;
                s0[e] = see0 ? s0[e] : -INFINITY;
                if constexpr (kHalves == 1) s1[e] = see1 ? s1[e] : -INFINITY; else s1[e] = s0[e];
                if constexpr (kCodes) {
                    const float* by = scales_of(i) + kTokens + 4 * L::part_of(lane) + L::token_of(e);
                    above = fmaxf(above, see0 ? fabsf(by[32 * mine]) : 0.0f);
                    if constexpr (kHalves == 1) above = fmaxf(above, see1 ? fabsf(by[32]) : 0.0f);
                }
            }
            if constexpr (kCodes) most = unit_above(groups_max<L::kRows>(above));
        }
        rescale_to(largest(s0, s1), most);
        if constexpr (kHeld != CF_CACHE_INT8) {  // whose codes are all finite
            if (masked) sanitise(at, first, here.there);
        }
        // Three stretches of products, each with the vector work of another part
        // among them; values are read a stretch ahead of their product.
        if constexpr (!kCodes && kHalves == 1) n1 = scores(at ^ 1, 1);
        weigh(s0, i, mine);
        const Weights p0 = pack(s0);
        constexpr int kFar = 4;  // products that values are read ahead of theirs
        u32x4_t v[kFar];
#pragma unroll
        for (int n = 0; n < kFar; ++n) v[n] = read_values(at, mine, n);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kHalves == 1) weigh(s1, i, 1);
        [[maybe_unused]] Weights p1;
        if constexpr (kHalves == 1) p1 = pack(s1);
#pragma unroll
        for (int n = 0; n < kPieces; ++n) {
            multiply(v[n % kFar], p0.part[n & 1], acc[n >> 1]);
            if constexpr (kSplit) multiply(v[n % kFar], pack(rest_of(s0)).part[n & 1], acc[n >> 1]);
            if (n + kFar < kPieces) {
                v[n % kFar] = read_values(at, mine, n + kFar);
            } else if constexpr (kHalves == 1) {
                v[n % kFar] = read_values(at, 1, n + kFar - kPieces);
            }
        }
        if constexpr (kHalves == 1) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < kPieces; ++n) {
                multiply(v[n % kFar], p1.part[n & 1], acc[n >> 1]);
                if constexpr (kSplit) multiply(v[n % kFar], pack(rest_of(s1)).part[n & 1], acc[n >> 1]);
                if (n + kFar < kPieces) v[n % kFar] = read_values(at, 1, n + kFar);
            }
        }
        if constexpr (!kCodes) {
            s0 = n0;
            if constexpr (kHalves == 1) s1 = n1;
        }
        here = next;
        next = far;
    }
    finish<T, kD, kHeld, kSplit, kRowWaves>(a, w, lds, lds_m, lds_l, bad, bad_from,
                                            m + (kCodes ? static_cast<float>(unit) : 0.0f), l, acc);
}

/// Zeros for the rows first_row .. first_row + count - 1 of a KV head's heads,
/// counted from token `first`.
template <typename O>
__device__ void zero_rows(const ChunkArgs& a, int first, int kv_head, int first_row, int end_row) {
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(end_row - first_row) * a.head_dim; i += kThreads) {
        const int r = first_row + static_cast<int>(i / a.head_dim);
        const int64_t out_row = static_cast<int64_t>(first + r / a.per) * a.heads + kv_head * a.per + r % a.per;
        static_cast<O*>(a.out)[out_row * a.head_dim + i % a.head_dim] = O{};
    }
}

/// What workgroup `id` does, or nothing (after writing zeros for rows that see no
/// token, where it is the first of theirs). O: the type of the result.
template <typename O>
__device__ bool item_of(const ChunkArgs& a, Item& w, int& end_row) {
    // KV heads vary fastest: workgroup i runs on XCD i % 8, so with 8 of them an
    // XCD reads one head's keys and values.
    int id = static_cast<int>(blockIdx.x);
    w.kv_head = id % a.kv_heads;
    id /= a.kv_heads;
    w.split = id % a.splits;
    const Segment s = segment_of(a, a.rows, id / a.splits);
    if (s.count == 0) return false;
    w.first = s.first;
    w.rows = s.count * a.per;
    w.first_row = s.tile * a.rows;
    end_row = min(w.rows, w.first_row + a.rows);
    Reach reach{};
    if (s.sequence >= 0) reach = reach_of(a, s, a.rows);
    const Range range = range_of(0, reach.hi, reach.each, w.split);
    if (range.lo >= range.hi) {
        if (reach.hi == 0 && w.split == 0) zero_rows<O>(a, s.first, w.kv_head, w.first_row, end_row);
        return false;
    }
    w.lo = range.lo;
    w.hi = range.hi;
    w.offset = reach.offset;
    w.table = a.tables + static_cast<int64_t>(s.sequence) * a.max_blocks;
    w.direct = reach.each >= reach.hi;
    return true;
}

/// fp32 caches.
template <int kD>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(2, 4))) void chunk_attention_wide_kernel(ChunkArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[WideKind<kD>::lds_bytes()];
    __shared__ float lds_m[kWaves][32];
    __shared__ float lds_l[kWaves][32];
    __shared__ BadValues<kD> bad;
    constexpr int kRows = Tile<float, kD>::kRows;
    Item w{};
    int end_row = 0;
    if (!item_of<float>(a, w, end_row)) return;
    if (end_row - w.first_row > kRows) {
        attend<kD, true>(a, w, lds, lds_m, lds_l, &bad);
    } else {
        attend<kD, false>(a, w, lds, lds_m, lds_l, &bad);
    }
}

/// 16-bit and 8-bit caches, chunks and single tokens in one launch.
template <typename T, int kD, cf_cache_format kHeld, bool kSplit>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(kD > 128 ? 1 : 2, 4))) void chunk_attention_kernel(ChunkArgs a) {
    constexpr int kFew = kWaves * FewTile<T, kD, kHeld != CF_CACHE_PLAIN>::kOwnBytes;
    constexpr int kMany = RowsKind<T, kD, kHeld>::lds_bytes();
    __shared__ __attribute__((aligned(16))) uint8_t lds[kFew > kMany ? kFew : kMany];
    __shared__ float lds_m[kWaves][32];
    __shared__ float lds_l[kWaves][32];
    BadValues<kD>* bad = nullptr;
    if constexpr (kHeld != CF_CACHE_INT8) {  // whose codes are all finite
        __shared__ BadValues<kD> values;
        bad = &values;
    }
    constexpr int kRows = Tile<T, kD>::kRows;
    Item w{};
    int end_row = 0;
    if (!item_of<std::conditional_t<kSplit, float, T>>(a, w, end_row)) return;
    if (end_row - w.first_row > 2 * kRows) {
        attend_rows<T, kD, kHeld, kSplit, 1>(a, w, lds, lds_m, lds_l, bad);
    } else if (end_row - w.first_row > kRows) {
        attend_rows<T, kD, kHeld, kSplit, 2>(a, w, lds, lds_m, lds_l, bad);
    } else if (end_row - w.first_row > 16) {
        attend_few<T, kD, kHeld, kSplit, 2>(a, w, lds, lds_m, lds_l, bad);
    } else {
        attend_few<T, kD, kHeld, kSplit, 1>(a, w, lds, lds_m, lds_l, bad);
    }
}

/// The general kernel: any head size and alignment, a wave per (token, head,
/// range), a token of the context at a time, dims over the lanes. Slow: a prompt of
/// 2048 tokens with 32 heads of 256 in fp32 takes 16 ms, 16 single tokens behind up
/// to 2000 0.9 ms, more than PyTorch's batched products (2.3 and 0.8 ms).
template <typename T, cf_cache_format kHeld, int kPer>
__global__ __launch_bounds__(kThreads) void chunk_attention_any_kernel(ChunkArgs a) {
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    const int64_t id = static_cast<int64_t>(blockIdx.x) * kWaves +
                       __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWaveSize);
    if (id >= static_cast<int64_t>(a.tokens) * a.heads * a.splits) return;
    const int split = static_cast<int>(id % a.splits);
    const int64_t out_row = id / a.splits;
    const int head = static_cast<int>(out_row % a.heads);
    const int token = static_cast<int>(out_row / a.heads);
    Segment s = segment_of_token(a, token);
    T* out = static_cast<T*>(a.out) + out_row * a.head_dim;
    Reach reach{};
    if (s.sequence >= 0) {
        s.tile = token - s.first;
        reach = reach_of(a, s, a.per);
    }
    const Range range = range_of(0, reach.hi, reach.each, split);
    if (range.lo >= range.hi) {
        if (reach.hi == 0 && split == 0) {
            for (int d = lane; d < a.head_dim; d += kWaveSize) Storage<T>::store(out + d, 0.0f);
        }
        return;
    }
    const T* q = static_cast<const T*>(a.query) + out_row * a.head_dim;
    float qv[kPer];
    float acc[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = lane + i * kWaveSize;
        qv[i] = d < a.head_dim ? Storage<T>::load(q + d) : 0.0f;
        acc[i] = 0.0f;
    }
    auto value = [&](const uint8_t* cache, int64_t at) {
        if constexpr (kHeld == CF_CACHE_PLAIN) {
            return Storage<T>::load(reinterpret_cast<const T*>(cache) + at);
        } else {
            float f[4];
            unpack4_codes<kHeld>(cache[at], f);
            return f[0];
        }
    };
    float m = -INFINITY;
    float l = 0.0f;
    for (int t = range.lo; t < range.hi; ++t) {
        const uint32_t block = static_cast<uint32_t>(t) / a.block_size;
        const uint32_t page = a.tables[static_cast<int64_t>(s.sequence) * a.max_blocks + block];
        if (page >= a.pages) continue;
        const int64_t row = static_cast<int64_t>(page) * a.block_size + (static_cast<uint32_t>(t) - block * a.block_size);
        const int64_t held = row * a.kv_heads + head / a.per;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int d = lane + i * kWaveSize;
            if (d < a.head_dim) dot = fmaf(qv[i], value(a.k_cache, held * a.head_dim + d), dot);
        }
        float y = wave_reduce_f32<AddF32>(dot) * (a.query_sign != 0 ? -a.c : a.c);
        float by = 1.0f;
        if constexpr (kHeld != CF_CACHE_PLAIN) {
            y *= a.k_scales[held];
            by = a.v_scales[held];
        }
        const float m_new = fmaxf(m, y);
        const float shift = m_new == -INFINITY ? 0.0f : m_new;
        const float f = exp2f(m - shift);
        const float p = exp2f(y - shift);
        m = m_new;
        l = fmaf(l, f, p);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int d = lane + i * kWaveSize;
            if (d < a.head_dim) acc[i] = fmaf(acc[i], f, p * by * value(a.v_cache, held * a.head_dim + d));
        }
    }
    if (reach.each >= reach.hi) {
        const float by = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int d = lane + i * kWaveSize;
            if (d < a.head_dim) Storage<T>::store(out + d, l == 0.0f ? 0.0f : acc[i] * by);
        }
        return;
    }
    const int64_t at = static_cast<int64_t>(split) * a.tokens * a.heads + out_row;
    if (lane == 0) {
        a.ml[2 * at] = m;
        a.ml[2 * at + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = lane + i * kWaveSize;
        if (d < a.head_dim) a.acc[at * a.pitch + d] = acc[i];
    }
}

/// Joins the pieces of one (token, head), a wave each. Rows of one piece are there
/// already. `rows`: of the first kernel's tiles.
template <typename T>
__global__ __launch_bounds__(kThreads) void chunk_attention_join_kernel(ChunkArgs a, int rows) {
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    const int64_t all = static_cast<int64_t>(a.tokens) * a.heads;
    const int64_t out_row = static_cast<int64_t>(blockIdx.x) * kWaves +
                            __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWaveSize);
    if (out_row >= all) return;
    const int token = static_cast<int>(out_row / a.heads);
    Segment s = segment_of_token(a, token);
    if (s.sequence < 0) return;
    const int64_t row = static_cast<int64_t>(token - s.first) * a.per + out_row % a.heads % a.per;
    s.tile = static_cast<int>(row / rows);
    const Reach reach = reach_of(a, s, rows);
    const int pieces = range_count(reach.hi, reach.each);
    if (pieces <= 1) return;
    static_assert(kMaxSplits <= kWaveSize, "a piece per lane");
    float pm = -INFINITY;
    float pl = 0.0f;
    if (lane < pieces) {
        pm = a.ml[2 * (lane * all + out_row)];
        pl = a.ml[2 * (lane * all + out_row) + 1];
    }
    const float m = wave_reduce_f32<MaxF32>(pm);
    const float weight = pm == -INFINITY ? 0.0f : exp2f(pm - m);
    const float l = wave_reduce_f32<AddF32>(pm == -INFINITY ? pl : pl * weight);
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(a.out) + out_row * a.head_dim;
    for (int d = lane; d < (a.head_dim + kWaveSize - 1) / kWaveSize * kWaveSize; d += kWaveSize) {
        float o = 0.0f;
        for (int i = 0; i < pieces; ++i) {
            const float f = readlane_f32(weight, i);
            if (d < a.head_dim) o = fmaf(a.acc[(i * all + out_row) * a.pitch + d], f, o);
        }
        if (d < a.head_dim) Storage<T>::store(out + d, l == 0.0f ? 0.0f : o * inverse);
    }
}

// ---- host -----------------------------------------------------------------------

struct Plan {
    int dim;   // head size of the matrix kernel, or 0: the general kernel
    int rows;  // of a tile
    int splits;
    int step;
    int least;
};

/// Row tiles of `segments` segments, at most: one more than the rows fill for each,
/// and no more than tokens where a tile has a token's rows.
int64_t tiles_of(int64_t rows, int64_t tokens, int64_t segments, int64_t per) {
    const int64_t n = tokens * per / rows + segments;
    return per <= rows && n > tokens ? tokens : n;
}

Plan plan_of(cf_dtype dtype, cf_cache_format format, int64_t tokens, int64_t sequences, int64_t heads,
             int64_t kv_heads, int64_t head_dim, int64_t capacity) {
    Plan p{};
    const int64_t per = heads / kv_heads;
    const bool wide = dtype == CF_F32 && format == CF_CACHE_PLAIN;
    const int64_t vec = format != CF_CACHE_PLAIN ? 16 : wide ? 4 : 8;
    if (head_dim % vec == 0 && head_dim <= (wide ? 128 : 256)) p.dim = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    const int64_t wave_rows = wide ? 16 : 32;
    p.rows = static_cast<int>(p.dim == 0 ? per : kWaves * wave_rows);
    auto splits = [&](int64_t items, int64_t target, int64_t least) {
        int64_t n = items > 0 ? target / items : 1;
        const int64_t most = ceil_div<int64_t>(capacity, least);
        if (n > most) n = most;
        if (n > kMaxSplits) n = kMaxSplits;
        return static_cast<int>(n < 1 ? 1 : n);
    };
    if (p.dim == 0) {
        p.step = 32;
        p.least = 64;
        p.splits = splits(tokens * heads, 4096, p.least);
        return p;
    }
    // Two workgroups a CU, in ranges of 256 tokens or more. (Four chunks of 100 in fp32
    // behind 900 tokens: 110 us uncut, 98 in two ranges for 512 workgroups, 107 in four;
    // seven chunks of 333 in int8 67 us uncut, 90 in two.)
    p.least = 256;
    p.step = static_cast<int>(kWaves * wave_rows);
    auto items = [&](int64_t rows) {
        return tiles_of(rows, tokens, sequences < tokens ? sequences : tokens, per) * kv_heads;
    };
    p.splits = splits(items(p.rows), 512, p.least);
    // Tiles of 64 rows, uncut, instead of tiles of 128 in two or three ranges, where a
    // table reaches 2048 tokens at most: two prompts of 400 tokens in bf16 24 us
    // against 42, in int8 29 against 47; 700 tokens behind 1300 59 against 68, and 81
    // against 83. In longer contexts each tile's own pass over them costs more than
    // the join (three chunks of 256 behind 3744: 115 us against 110, 174 against 146).
    if (!wide && p.splits > 1 && capacity <= 2048 && splits(items(64), 512, p.least) == 1) {
        p.rows = 64;
        p.splits = 1;
    }
    // And where codes in heads of 64, of which three workgroups fit a CU, do not fill the
    // GPU in tiles of 128 (seven chunks of 333 in int8, 400 items, 67 us against 77;
    // 448 items 47 against 54; 576 would take 76 against 58, and the query's type 400
    // items 60 against 51).
    if (format != CF_CACHE_PLAIN && p.dim == 64 && p.splits == 1 && p.rows == 128 && items(128) < 512) p.rows = 64;
    return p;
}

int64_t capacity_of(int64_t max_blocks, int64_t block_size) {
    return max_blocks > kMostTokens / block_size ? kMostTokens : max_blocks * block_size;
}

size_t workspace_of(const Plan& p, int64_t tokens, int64_t heads, int64_t head_dim) {
    if (p.splits == 1) return 0;
    const size_t rows = static_cast<size_t>(p.splits) * tokens * heads;
    return (rows * 8 + 15) / 16 * 16 + rows * ((head_dim + 3) / 4 * 4) * 4;
}

bool sizes_ok(int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim,
              int64_t block_size, int64_t max_blocks) {
    return tokens > 0 && sequences >= 0 && heads > 0 && kv_heads > 0 && head_dim > 0 && head_dim <= 1024 &&
           block_size > 0 && max_blocks > 0 && heads % kv_heads == 0;
}

template <typename T, int kD, cf_cache_format kHeld, bool kSplit>
void run_size(const ChunkArgs& a, dim3 grid, hipStream_t stream) {
    if constexpr (Tile<T, kD>::kWide) {
        launch(chunk_attention_wide_kernel<kD>, grid, dim3(kThreads), 0, stream, a);
    } else {
        launch(chunk_attention_kernel<T, kD, kHeld, kSplit>, grid, dim3(kThreads), 0, stream, a);
    }
}

template <typename T, cf_cache_format kHeld, bool kSplit>
void run_matrix(const ChunkArgs& a, const Plan& p, dim3 grid, hipStream_t stream) {
    if (p.dim == 64) {
        run_size<T, 64, kHeld, kSplit>(a, grid, stream);
    } else if (p.dim == 128) {
        run_size<T, 128, kHeld, kSplit>(a, grid, stream);
    } else if constexpr (kHeld != CF_CACHE_PLAIN || sizeof(T) == 2) {
        run_size<T, 256, kHeld, kSplit>(a, grid, stream);
    }
}

template <typename T, cf_cache_format kHeld>
void run(const ChunkArgs& a, const Plan& p, int64_t tiles, hipStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.tokens) * a.heads;
    if (p.dim == 0) {
        const dim3 grid(static_cast<unsigned>(ceil_div<int64_t>(rows * a.splits, kWaves)));
        if (a.head_dim <= 128) {
            launch(chunk_attention_any_kernel<T, kHeld, 2>, grid, dim3(kThreads), 0, stream, a);
        } else {
            launch(chunk_attention_any_kernel<T, kHeld, 16>, grid, dim3(kThreads), 0, stream, a);
        }
    } else {
        const dim3 grid(static_cast<unsigned>(tiles * a.splits * a.kv_heads));
        if constexpr (kHeld == CF_CACHE_PLAIN) {
            run_matrix<T, kHeld, false>(a, p, grid, stream);
        } else if constexpr (sizeof(T) == 4) {
            run_matrix<f16_t, kHeld, true>(a, p, grid, stream);
        } else {
            run_matrix<f16_t, kHeld, false>(a, p, grid, stream);
        }
    }
    if (a.splits > 1) {
        launch(chunk_attention_join_kernel<T>, dim3(static_cast<unsigned>(ceil_div<int64_t>(rows, kWaves))),
               dim3(kThreads), 0, stream, a, p.rows);
    }
}

template <typename T>
void run_format(cf_cache_format format, const ChunkArgs& a, const Plan& p, int64_t tiles, hipStream_t stream) {
    switch (format) {
        case CF_CACHE_PLAIN: run<T, CF_CACHE_PLAIN>(a, p, tiles, stream); break;
        case CF_CACHE_INT8: run<T, CF_CACHE_INT8>(a, p, tiles, stream); break;
        case CF_CACHE_E4M3: run<T, CF_CACHE_E4M3>(a, p, tiles, stream); break;
    }
}

}  // namespace
}  // namespace cf

extern "C" {

size_t cf_paged_attention_chunk_workspace_bytes(cf_dtype dtype, cf_cache_format format, int64_t num_tokens,
                                                int64_t num_sequences, int64_t num_heads, int64_t num_kv_heads,
                                                int64_t head_dim, int64_t block_size,
                                                int64_t max_blocks_per_sequence) {
    if (!cf::valid_dtype(dtype) || !cf::valid_format(format) ||
        !cf::sizes_ok(num_tokens, num_sequences, num_heads, num_kv_heads, head_dim, block_size,
                      max_blocks_per_sequence)) {
        return 0;
    }
    const cf::Plan p = cf::plan_of(dtype, format, num_tokens, num_sequences, num_heads, num_kv_heads, head_dim,
                                   cf::capacity_of(max_blocks_per_sequence, block_size));
    return cf::workspace_of(p, num_tokens, num_heads, head_dim);
}

cf_status cf_paged_attention_chunk(const void* query, const void* k_cache, const void* v_cache, const float* k_scales,
                                   const float* v_scales, const int32_t* query_starts, const uint32_t* block_tables,
                                   const int32_t* context_lens, void* out, cf_dtype dtype, cf_cache_format format,
                                   int64_t num_pages, int64_t num_tokens, int64_t num_sequences, int64_t num_heads,
                                   int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                   int64_t max_blocks_per_sequence, float scale, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    CF_ENTRY();
    const char* who = "cf_paged_attention_chunk";
    if (num_tokens <= 0 || num_heads <= 0 || head_dim <= 0) return CF_OK;
    CF_REQUIRE(cf::valid_dtype(dtype), "%s: unknown dtype %d", who, static_cast<int>(dtype));
    CF_REQUIRE(cf::valid_format(format), "%s: unknown cache format %d", who, static_cast<int>(format));
    CF_REQUIRE(cf::sizes_ok(num_tokens, num_sequences, num_heads, num_kv_heads, head_dim, block_size,
                            max_blocks_per_sequence) && num_pages > 0,
               "%s: %lld heads over %lld KV heads of %lld (at most 1024), blocks of %lld, %lld per sequence, %lld "
               "pages, %lld sequences",
               who, static_cast<long long>(num_heads), static_cast<long long>(num_kv_heads),
               static_cast<long long>(head_dim), static_cast<long long>(block_size),
               static_cast<long long>(max_blocks_per_sequence), static_cast<long long>(num_pages),
               static_cast<long long>(num_sequences));
    CF_REQUIRE(query != nullptr && k_cache != nullptr && v_cache != nullptr && query_starts != nullptr &&
                   block_tables != nullptr && context_lens != nullptr && out != nullptr,
               "%s: null pointer", who);
    CF_REQUIRE(format == CF_CACHE_PLAIN || (k_scales != nullptr && v_scales != nullptr),
               "%s: an 8-bit cache needs scales", who);
    const size_t size = cf::dtype_size(dtype);
    const size_t held = format == CF_CACHE_PLAIN ? size : 1;
    CF_REQUIRE(cf::host_aligned(query, size) && cf::host_aligned(out, size) && cf::host_aligned(k_cache, held) &&
                   cf::host_aligned(v_cache, held) && cf::host_aligned(k_scales, 4) && cf::host_aligned(v_scales, 4),
               "%s: misaligned pointer", who);
    // Cache rows, token positions, query rows and work items are counted in 32 bits.
    constexpr int64_t kMost = cf::kMostTokens;
    CF_REQUIRE(num_pages <= kMost / block_size && max_blocks_per_sequence <= kMost && num_kv_heads <= (1 << 14) &&
                   num_sequences <= kMost - 2 && num_tokens <= kMost / num_heads,
               "%s: %lld pages of %lld tokens, %lld sequences, %lld tokens of %lld heads or %lld KV heads exceed "
               "32-bit counts",
               who, static_cast<long long>(num_pages), static_cast<long long>(block_size),
               static_cast<long long>(num_sequences), static_cast<long long>(num_tokens),
               static_cast<long long>(num_heads), static_cast<long long>(num_kv_heads));
    cf::Plan p = cf::plan_of(dtype, format, num_tokens, num_sequences, num_heads, num_kv_heads, head_dim,
                             cf::capacity_of(max_blocks_per_sequence, block_size));
    const size_t needed = cf::workspace_of(p, num_tokens, num_heads, head_dim);
    CF_REQUIRE(needed == 0 || (workspace != nullptr && workspace_bytes >= needed && cf::host_aligned(workspace, 16)),
               "%s: needs %zu bytes of 16-byte aligned workspace", who, needed);
    if (p.dim != 0 && !(cf::host_aligned(query, 16) && cf::host_aligned(k_cache, 16) &&
                        cf::host_aligned(v_cache, 16) && cf::host_aligned(out, 16))) {
        p.dim = 0;  // within the same workspace: as many ranges at most
        p.rows = static_cast<int>(num_heads / num_kv_heads);
        p.step = 32;
        p.least = 64;
    }
    // The kernel for many rows counts a cache's 16-byte pieces in 32 bits. In larger
    // ones (64 GiB and more) tiles have no more rows than the one for few, which
    // counts them in 64, takes.
    const bool wide = dtype == CF_F32 && format == CF_CACHE_PLAIN;
    const int64_t token_pieces = num_kv_heads * head_dim * static_cast<int64_t>(held) / 16;
    if (p.dim != 0 && !wide && num_pages * block_size > (int64_t{1} << 32) / token_pieces) p.rows = 32;
    cf::ChunkArgs a{};
    a.query = query;
    a.k_cache = static_cast<const uint8_t*>(k_cache);
    a.v_cache = static_cast<const uint8_t*>(v_cache);
    a.k_scales = k_scales;
    a.v_scales = v_scales;
    a.starts = query_starts;
    a.tables = block_tables;
    a.context = context_lens;
    a.out = out;
    a.pages = static_cast<uint32_t>(num_pages);
    a.block_size = static_cast<uint32_t>(block_size);
    a.block_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctzll(static_cast<uint64_t>(block_size)) : -1;
    a.tokens = static_cast<int>(num_tokens);
    a.sequences = static_cast<int>(num_sequences);
    a.heads = static_cast<int>(num_heads);
    a.kv_heads = static_cast<int>(num_kv_heads);
    a.per = static_cast<int>(num_heads / num_kv_heads);
    a.head_dim = static_cast<int>(head_dim);
    a.pitch = (a.head_dim + 3) / 4 * 4;
    a.max_blocks = static_cast<int>(max_blocks_per_sequence);
    a.capacity = static_cast<int>(cf::capacity_of(max_blocks_per_sequence, block_size));
    a.token_pieces = static_cast<uint32_t>(token_pieces);
    a.rows = p.rows;
    a.splits = p.splits;
    a.step = p.step;
    a.least = p.least;
    a.query_bf16 = dtype == CF_BF16;
    const int64_t tiles = cf::tiles_of(p.rows, num_tokens, num_sequences + 2, a.per);
    const int64_t rows = num_tokens * num_heads;
    const int64_t workgroups = p.dim == 0 ? cf::ceil_div<int64_t>(rows * p.splits, cf::kWaves)
                                          : tiles * p.splits * num_kv_heads;
    CF_REQUIRE(workgroups <= cf::kMaxWorkgroups && cf::ceil_div<int64_t>(rows, cf::kWaves) <= cf::kMaxWorkgroups,
               "%s: %lld tokens of %lld heads are too many for a launch", who, static_cast<long long>(num_tokens),
               static_cast<long long>(num_heads));
    // The kernels take maxima of unscaled scores, so the factor must not be
    // negative, nor 0 (which times a masked score is NaN).
    const float c = scale * cf::kLog2e;
    a.c = c == 0.0f ? 1.0e-37f : c < 0.0f ? -c : c;
    const bool flip = c < 0.0f;
    a.query_sign = flip ? (dtype == CF_F32 ? 0x80000000u : 0x80008000u) : 0u;
    const size_t pieces = static_cast<size_t>(p.splits) * rows;
    a.ml = static_cast<float*>(workspace);
    a.acc = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (pieces * 8 + 15) / 16 * 16);
    auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case CF_F32: cf::run_format<float>(format, a, p, tiles, s); break;
        case CF_F16: cf::run_format<cf::f16_t>(format, a, p, tiles, s); break;
        case CF_BF16: cf::run_format<cf::bf16_t>(format, a, p, tiles, s); break;
    }
    return cf::check_launch("launching paged attention of chunks", s);
}

}  // extern "C"
