// Attention for one decode step over a paged cache whose sequences share
// prompts: what cf_paged_attention computes, with the keys and values of a
// shared prompt read once for all the sequences behind it.
//
// For sequence s, head h, KV head h / (H / KVH) and context c:
//   out[s, h] = sum_{t < c} softmax_t(scale q[s, h] . k[t]) v[t].
// Sequences group_starts[g] .. group_starts[g + 1] - 1 hold the same K and V
// in their first prefix_lens[g] tokens. A sequence's context is cut in two:
// its group's prefix, which it attends to together with the other sequences
// of the group, and the rest, alone; the parts are joined by the rescaling
// rule of a softmax (running maximum, sum, weighted values). A sequence whose
// context is shorter than its group's prefix goes alone from its first token.
//
// Reading each prefix once makes it a matrix product: the query rows of a
// group (sequences x heads of a KV head) against the prefix, on the matrix
// cores. The rests stay bound by HBM.
//   * A work item is (row tile, KV head, token range) of a prefix or (sequence,
//     KV head, token range) of a rest, a workgroup of four waves each (a wave,
//     where there are many rests), both kinds in one launch, the items of all
//     groups laid end to end. Long ranges are split from the lengths found on
//     the device; a second kernel joins the pieces.
//   * Scores are formed transposed, S^T = K Q^T: a lane then holds one query
//     row and several tokens, so a row's maximum and sum are lane-local but for
//     one exchange, and the probabilities are in place as the B operand of
//     O^T += V^T P^T without moving between lanes.
//   * K and V tiles go from the cache straight to LDS (no registers), in 16-byte
//     pieces whose order inside a row is changed so that the fragment reads hit
//     all banks. Tiles with many query rows are shared by four waves of
//     different rows through a ring of stages; tiles with few rows belong to
//     one wave, the four waves taking different tokens.
//   * 16-bit caches run 32 x 32 x 16 MFMA over 32 rows and 32 tokens, fp32
//     caches 16 x 16 x 4 fp32 MFMA over 16 rows and 16 tokens (fp32 products).
//     Probabilities are rounded to the cache's type for the second product
//     (relative error half an ulp each, of either sign; for fp16's smallest
//     numbers see kLift); sums stay in fp32.
//   * Measured, 32 query and 8 KV heads of 128 in bf16, with the join: 128
//     sequences behind 32768 tokens 100 + 9.9 us, 690 TFLOP/s: neither the matrix
//     cores (31% busy) nor the vector units (34%), but the chain from one product
//     through the probabilities to the next at two waves per SIMD. 64 sequences
//     behind 4099 tokens 26 + 6.7 us, 3.2 TB/s: one round of work, the CUs busy
//     for 57% of it. 8 behind 1000 tokens 9 + 3.5 us: the launches' chains. 16 in
//     two groups behind 2048 tokens in fp32 27 + 4.7 us: 680 workgroups on 512
//     places, matrix cores 12% busy.
// Tokens behind a range's end, and tokens whose page is not in the cache, get
// no weight: their scores are replaced and their V rows are cleared in LDS, so
// that whatever lies there (NaN, infinities) stays out.
#include "cf_attention_tile.hpp"
#include "cf_common.hpp"
#include "cf_lds_dma.hpp"
#include "cf_ranges.hpp"

namespace cf {
namespace {

constexpr int kWaves = 4;  // per workgroup where nothing else is said
constexpr int kThreads = kWaves * kWaveSize;
constexpr int kMaxSplits = 64;
constexpr float kLog2e = 1.4426950408889634f;

struct SharedArgs {
    const void* query;
    const void* k_cache;
    const void* v_cache;
    const int32_t* starts;  // [groups + 1]
    const int32_t* prefix;  // [groups]
    const uint32_t* tables;
    const int32_t* context;
    void* out;
    float* ml;   // [slots][sequences * heads][2]: maximum (base 2), sum
    float* acc;  // [slots][sequences * heads][pitch]
    uint32_t pages;
    uint32_t block_size;
    int block_shift;      // log2(block_size), or -1
    uint32_t page_bytes;  // 0: 2^32 or more
    int sequences;
    int heads;
    int kv_heads;
    int per;          // query heads per KV head
    int head_dim;
    int pitch;        // head_dim rounded up to 4
    int groups;
    int max_blocks;
    int capacity;     // tokens a table row reaches
    int prefix_splits;
    int rest_splits;
    int prefix_tiles;  // row tiles over all groups, at most
    int rest_tiles;    // row tiles per sequence and KV head
    int prefix_step;   // tokens of a prefix's range are a multiple of this; 0: nothing is shared
    int prefix_least;  // and at least about this
    int rest_step;     // the same for rests
    int rest_least;
    bool rest_solo;    // a wave per rest item
    int prefix_items;  // workgroups of the first kind
    float c;           // |scale| log2(e), above 0
    uint32_t query_sign;  // flips the query's signs for a negative scale
};

// ---- groups, ranges -----------------------------------------------------------

struct Group {
    int first;   // sequences first .. end - 1
    int end;
    int prefix;  // tokens
};

__device__ __forceinline__ int clamp_to(int v, int hi) { return v < 0 ? 0 : v > hi ? hi : v; }

__device__ __forceinline__ int wave_max_int(int v) {
#pragma unroll
    for (int d = 1; d < kWaveSize; d <<= 1) v = max(v, __shfl_xor(v, d));
    return v;
}

/// The group of sequence s (uniform), or end = 0. Starts are taken as the
/// largest so far, so that groups never overlap whatever is stored.
__device__ Group group_of(const SharedArgs& a, int s) {
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    int first = 0;
    for (int base = 0; base <= a.groups; base += kWaveSize - 1) {  // one start is looked at twice
        const int g = base + lane;
        const bool there = g <= a.groups;
        const int start = there ? clamp_to(a.starts[g], a.sequences) : 0;
        const int prefix = g < a.groups ? clamp_to(a.prefix[g], a.capacity) : 0;
        const uint64_t above = __builtin_amdgcn_ballot_w64(there && start > s);
        if (above != 0) {
            const int at = __builtin_ctzll(above);  // the first start past s ends the group
            if (base + at == 0) return Group{0, 0, 0};
            first = max(first, wave_max_int(lane < at ? start : 0));
            return Group{first, __builtin_amdgcn_readlane(start, at), __builtin_amdgcn_readlane(prefix, at - 1)};
        }
        first = max(first, wave_max_int(start));
    }
    return Group{0, 0, 0};
}

__device__ __forceinline__ int context_of(const SharedArgs& a, int s) { return clamp_to(a.context[s], a.capacity); }

/// One XCD's share of the prefixes' work: a group, its row tile, and the place
/// of a (range, KV head) pair in the XCD's run of them.
struct PrefixItem {
    Group group;  // end = 0: no such item
    int tile;
    int place;
    int run;   // pairs per XCD
    int each;  // tokens per range
};

/// Item `index` (uniform) of an XCD, over all groups in turn: the groups' items
/// lie end to end, so the first workgroups have all the work. (Workgroups without
/// work among the others cost half of the GPU: they are dealt to the shader
/// engines in turn, and every second one was empty.)
__device__ PrefixItem prefix_item(const SharedArgs& a, int rows, int step, int least, int index) {
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    int before = 0;  // largest start so far
    for (int base = 0; base < a.groups; base += kWaveSize) {
        const int g = base + lane;
        const bool there = g < a.groups;
        int start = there ? clamp_to(a.starts[g], a.sequences) : 0;
        int end = there ? clamp_to(a.starts[g + 1], a.sequences) : 0;
        const int prefix = there ? clamp_to(a.prefix[g], a.capacity) : 0;
        if (lane == 0) start = max(start, before);
        if (a.groups > 1) {
#pragma unroll
            for (int d = 1; d < kWaveSize; d <<= 1) {
                const int o = __shfl_up(start, d);
                if (lane >= d) start = max(start, o);
            }
        }
        end = there ? max(start, end) : start;
        const int tiles = prefix > 0 ? ((end - start) * a.per + rows - 1) / rows : 0;
        const int each = split_length(max(prefix, 1), a.prefix_splits, step, least);
        const int run = (range_count(prefix, each) * a.kv_heads + 7) / 8;
        const int items = tiles * run;
        int total = items;
        if (a.groups > 1) {
#pragma unroll
            for (int d = 1; d < kWaveSize; d <<= 1) {
                const int o = __shfl_up(total, d);
                if (lane >= d) total += o;
            }
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(total > index);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            index -= __builtin_amdgcn_readlane(total - items, at);
            const int n = __builtin_amdgcn_readlane(tiles, at);
            return PrefixItem{Group{__builtin_amdgcn_readlane(start, at), __builtin_amdgcn_readlane(end, at),
                                    __builtin_amdgcn_readlane(prefix, at)},
                              index % n, index / n, __builtin_amdgcn_readlane(run, at),
                              __builtin_amdgcn_readlane(each, at)};
        }
        index -= __builtin_amdgcn_readlane(total, kWaveSize - 1);
        before = __builtin_amdgcn_readlane(start, kWaveSize - 1);
    }
    return PrefixItem{Group{0, 0, 0}, 0, 0, 0, 0};
}

/// LDS of a workgroup: its waves' own tiles (K and V each), or a ring of as many
/// shared ones; afterwards the waves' outputs.
template <typename T, int kD>
constexpr int lds_bytes() {
    using L = Tile<T, kD>;
    constexpr int tiles = kWaves * 2 * L::kBytes;
    constexpr int outputs = kWaves * L::kRows * L::kOutPitch * 4;
    return tiles > outputs ? tiles : outputs;
}

// ---- one work item ----------------------------------------------------------------

/// One workgroup's part: tokens lo .. hi - 1 of the cache behind `table`, for
/// query rows first_row .. of a set of sequences x heads of one KV head.
struct Item {
    const uint32_t* table;
    int lo, hi;
    int kv_head;
    int first_sequence;
    int sequences;   // rows are (sequence, head of the KV head)
    int first_row;
    int least;       // sequences with fewer tokens do not take part
    int last_block;  // of the range
    int slot;
};

/// The waves of a workgroup take different rows (kRows), different tokens of the
/// same rows (kTokens), or items of their own (kSolo: no barrier).
enum class Waves { kRows, kTokens, kSolo };

/// kRows: through a ring of kWaves tiles.
template <typename T, int kD, Waves kWork>
__device__ void attend(const SharedArgs& a, const Item& w, uint8_t* lds, float (*lds_m)[32], float (*lds_l)[32],
                       int (*lds_row)[32]) {
    using L = Tile<T, kD>;
    constexpr int kRowWaves = kWork == Waves::kRows ? kWaves : 1;
    constexpr int kTokenWaves = kWork == Waves::kTokens ? kWaves : 1;
    constexpr int kStages = kWaves;
    constexpr bool kSolo = kWork == Waves::kSolo;
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & (kWaveSize - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
    const int row_wave = kRowWaves == 1 ? 0 : wave;
    const int token_wave = kWork == Waves::kTokens ? wave : 0;
    const int total_rows = w.sequences * a.per;

    // Query rows of this wave; rows past the end are zeros.
    typename L::Query q[L::kQueries];
    const int row = w.first_row + row_wave * L::kRows + L::row_of(lane);
    {
        const bool inside = row < total_rows;
        const int seq = w.first_sequence + (inside ? row / a.per : 0);
        const int head = w.kv_head * a.per + (inside ? row % a.per : 0);
        const int out_row = seq * a.heads + head;
        const T* from = static_cast<const T*>(a.query) + static_cast<int64_t>(out_row) * a.head_dim;
        // Where the row's piece goes; nowhere for a sequence that takes no part.
        if (!kSolo && L::part_of(lane) == 0) {
            lds_row[wave][L::row_of(lane)] = inside && context_of(a, seq) >= w.least ? out_row : -1;
        }
#pragma unroll
        for (int u = 0; u < L::kQueries; ++u) {
            const int dim = L::query_dim(u, lane);
            u32x4_t raw = {0u, 0u, 0u, 0u};
            if (inside && dim < a.head_dim) raw = *reinterpret_cast<const u32x4_t*>(from + dim) ^ a.query_sign;
            q[u] = __builtin_bit_cast(typename L::Query, raw);
        }
    }
    if (a.head_dim < kD) {  // the copies leave the end of every row as it is
        constexpr int kPieces = 2 * L::kBytes / 16;  // of one stage, or of a wave's own tiles
        if constexpr (kSolo) {
            for (int i = lane; i < kPieces; i += kWaveSize) {
                reinterpret_cast<u32x4_t*>(lds)[wave * kPieces + i] = u32x4_t{0u, 0u, 0u, 0u};
            }
            wait_lds();
        } else {
            for (int i = tid; i < kStages * kPieces; i += kThreads) {
                reinterpret_cast<u32x4_t*>(lds)[i] = u32x4_t{0u, 0u, 0u, 0u};
            }
            __syncthreads();
        }
    }

    const uint32_t lds_base = __builtin_amdgcn_readfirstlane(lds_address(lds));
    const uint32_t token_bytes = static_cast<uint32_t>(a.kv_heads) * a.head_dim * sizeof(T);
    const uint32_t head_bytes = static_cast<uint32_t>(w.kv_head) * a.head_dim * sizeof(T);
    const uint8_t* k_head = static_cast<const uint8_t*>(a.k_cache) + head_bytes;
    const uint8_t* v_head = static_cast<const uint8_t*>(a.v_cache) + head_bytes;
    const int row_pieces = a.head_dim * static_cast<int>(sizeof(T)) / 16;
    // Tiles begin at multiples of kTokens; tokens before lo are masked.
    const int begin = w.lo / L::kTokens * L::kTokens;
    const int tiles = (w.hi - begin + L::kTokens - 1) / L::kTokens;

    // A copy takes kPerCopy neighbouring tokens. A wave's own tiles are copied
    // whole, K and V; of a ring's tile each wave copies a share of K or of V.
    // kSpan neighbouring tokens lie in one page (blocks of a power of two from 16
    // on).
    constexpr int kPerCopy = kWaveSize / L::kChunks;
    static_assert(kPerCopy >= 1, "a row within a copy");
    constexpr int kCopies = kRowWaves == 1 ? L::kCopies : 2 * L::kCopies / kWaves;
    static_assert(kRowWaves == 1 || 2 * L::kCopies % kWaves == 0, "copies per wave");
    constexpr int kSpan = kCopies * kPerCopy < 16 ? kCopies * kPerCopy : 16;
    constexpr int kSpanCopies = kSpan / kPerCopy;
    const bool ring_v = kRowWaves > 1 && wave >= kWaves / 2;
    const int first_copy = kRowWaves == 1 ? 0 : wave % (kWaves / 2) * kCopies;

    // 64 entries of the block table in lane registers: a token's page is a lane
    // read, not a load that would have to wait behind the copies. `sound`: all
    // entries of the range name pages.
    int window_base = static_cast<int>(static_cast<uint32_t>(begin) / a.block_size);
    auto load_window = [&]() { return w.table[min(window_base + lane, w.last_block)]; };
    uint32_t window = load_window();
    bool sound = __builtin_amdgcn_ballot_w64(window >= a.pages) == 0;
    for (int b = window_base + kWaveSize; b <= w.last_block && sound; b += kWaveSize) {
        sound = __builtin_amdgcn_ballot_w64(w.table[min(b + lane, w.last_block)] >= a.pages) == 0;
    }
    const bool fast = sound && a.block_shift >= 4 && a.page_bytes != 0;
    // Byte offset in the cache of token t, rounded to its span; tokens behind
    // the range's last page take that page.
    auto place_of = [&](int t) {
        const int block = min(t >> a.block_shift, w.last_block);
        if (block >= window_base + kWaveSize) {  // tiles are taken in ascending order
            window_base = block;
            window = load_window();
            // Waited for here: after the branch the compiler would wait for every
            // copy in flight, whether or not this ran.
            asm volatile("" : "+v"(window));
        }
        const uint32_t page = __builtin_amdgcn_readlane(window, block - window_base);
        return static_cast<uint64_t>(page) * a.page_bytes +
               (static_cast<uint32_t>(t) & (a.block_size - 1)) * token_bytes;
    };
    // This wave's copies of K or V of the tile at token `first` to LDS.
    auto fetch = [&](int first, uint32_t dst, bool is_v) {
#pragma unroll
        for (int n0 = 0; n0 < kCopies; n0 += kSpanCopies) {
            const uint8_t* base = (is_v ? v_head : k_head) + place_of(first + (first_copy + n0) * kPerCopy);
#pragma unroll
            for (int n = n0; n < n0 + kSpanCopies; ++n) {
                const int r = (first_copy + n) * kPerCopy + lane / L::kChunks;
                const int piece = (lane % L::kChunks) ^ (is_v ? L::v_swizzle(r) : L::k_swizzle(r));
                const uint32_t offset = static_cast<uint32_t>((n - n0) * kPerCopy + lane / L::kChunks) * token_bytes +
                                        static_cast<uint32_t>(piece) * 16;
                if (piece < row_pieces) {
                    copy16_to_lds(base, offset, dst + static_cast<uint32_t>(first_copy + n) * 16 * kWaveSize);
                }
            }
        }
    };

    float m = -INFINITY;  // the row's running maximum
    float l = 0.0f;       // this lane's share of the running sum
    typename L::Score acc[L::kAcc / L::kScores];
#pragma unroll
    for (int b = 0; b < L::kAcc / L::kScores; ++b) {
#pragma unroll
        for (int i = 0; i < L::kScores; ++i) acc[b][i] = 0.0f;
    }

    // The tokens of the tile at `first` that lie in the range, a bit each.
    constexpr uint32_t kAll = 0xFFFFFFFFu >> (32 - L::kTokens);
    auto in_range = [&](int first) {
        const int ahead = w.lo - first;
        const int count = w.hi - first;
        return (ahead > 0 ? kAll << ahead : kAll) & (count < L::kTokens ? (1u << count) - 1u : kAll);
    };
    auto mask = [&](typename L::Score& s, uint32_t valid) {
        const uint32_t mine = valid >> (4 * L::part_of(lane));
#pragma unroll
        for (int i = 0; i < L::kScores; ++i) s[i] = (mine & (1u << L::token_of(i))) != 0 ? s[i] : -INFINITY;
    };
    // Clear the V rows of tokens that are not there.
    auto clear = [&](uint8_t* v, uint32_t valid, int start, int step) {
        for (int i = start; i < L::kTokens * L::kChunks; i += step) {
            if (((valid >> (i / L::kChunks)) & 1) == 0) {
                reinterpret_cast<u32x4_t*>(v)[i] = u32x4_t{0u, 0u, 0u, 0u};
            }
        }
    };
    // Scores to probabilities, and the running values.
    auto soften = [&](typename L::Score& s) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < L::kScores; ++i) top = fmaxf(top, s[i]);
        top = groups_max<L::kRows>(top);
        const float m_new = fmaxf(m, top * a.c);
        if (__builtin_amdgcn_ballot_w64(m_new > m + L::kLag) != 0) {
            const float f = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.0f : m_new));
            l *= f;
#pragma unroll
            for (int b = 0; b < L::kAcc / L::kScores; ++b) {
#pragma unroll
                for (int i = 0; i < L::kScores; ++i) acc[b][i] *= f;
            }
            m = m_new;
        }
        const float shift = (m == -INFINITY ? 0.0f : m) - L::kLift;
#pragma unroll
        for (int i = 0; i < L::kScores; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.c, -shift));
            l += s[i];
        }
    };
    auto edge = [&](int first) { return first < w.lo || first + L::kTokens > w.hi; };

    if (!fast) {
        // Any block size, and tables with entries that name no page: every token
        // looked up by itself, a tile at a time.
        uint8_t* k = lds + (kRowWaves == 1 ? wave * 2 * L::kBytes : 0);
        uint8_t* v = k + L::kBytes;
        const uint32_t k_dst = lds_base + (kRowWaves == 1 ? static_cast<uint32_t>(wave) * 2 * L::kBytes : 0u);
        for (int i = token_wave; i < tiles; i += kTokenWaves) {
            const int t = begin + i * L::kTokens + (lane & (L::kTokens - 1));
            const uint32_t block = static_cast<uint32_t>(t) / a.block_size;
            const bool inside = t >= w.lo && t < w.hi;
            const uint32_t page = inside ? w.table[block] : a.pages;
            const uint32_t cache_row = page < a.pages ? page * a.block_size + static_cast<uint32_t>(t) - block * a.block_size : 0u;
            const uint32_t valid = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(page < a.pages)) & kAll;
            for (int n = kRowWaves == 1 ? 0 : wave; n < L::kCopies; n += kRowWaves) {
                const int r = n * kPerCopy + lane / L::kChunks;
                const uint64_t from = static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(cache_row), r))) * token_bytes;
                const uint32_t dst = k_dst + static_cast<uint32_t>(n) * 16 * kWaveSize;
                const int k_piece = (lane % L::kChunks) ^ L::k_swizzle(r);
                const int v_piece = (lane % L::kChunks) ^ L::v_swizzle(r);
                if (k_piece < row_pieces) copy16_to_lds(k_head + from + k_piece * 16, dst);
                if (v_piece < row_pieces) copy16_to_lds(v_head + from + v_piece * 16, dst + L::kBytes);
            }
            wait_vm<0>();
            if constexpr (kRowWaves > 1) __syncthreads();
            typename L::Score s = L::scores(k, q, lane);
            if (valid != kAll) mask(s, valid);
            soften(s);
            if (valid != kAll) {
                clear(v, valid, kRowWaves == 1 ? lane : tid, kRowWaves == 1 ? kWaveSize : kThreads);
                wait_lds();
                if constexpr (kRowWaves > 1) __syncthreads();
            }
            L::values(v, s, acc, lane);
            wait_lds();
            if constexpr (kRowWaves > 1) __syncthreads();
        }
    } else if constexpr (kRowWaves == 1) {
        // The wave's own K and V tile, one copied while the other is used.
        uint8_t* k = lds + wave * 2 * L::kBytes;
        uint8_t* v = k + L::kBytes;
        const uint32_t k_dst = lds_base + static_cast<uint32_t>(wave) * 2 * L::kBytes;
        const uint32_t v_dst = k_dst + L::kBytes;
        int t = begin + token_wave * L::kTokens;
        constexpr int kStep = kTokenWaves * L::kTokens;
        if (t < w.hi) {
            fetch(t, k_dst, false);
            fetch(t, v_dst, true);
        }
        for (; t < w.hi; t += kStep) {
            const bool more = t + kStep < w.hi;
            // K has landed: only V's copies may be in flight. (Copies that no
            // lane takes part in are not issued, so a head narrower than kD
            // waits for all.)
            if (a.head_dim == kD) wait_vm<kCopies>(); else wait_vm<0>();
            typename L::Score s = L::scores(k, q, lane);
            wait_lds();
            if (more) fetch(t + kStep, k_dst, false);
            const bool partial = edge(t);
            if (partial) mask(s, in_range(t));
            soften(s);
            if (more && a.head_dim == kD) wait_vm<kCopies>(); else wait_vm<0>();
            if (partial) {
                clear(v, in_range(t), lane, kWaveSize);
                wait_lds();
            }
            L::values(v, s, acc, lane);
            wait_lds();
            if (more) fetch(t + kStep, v_dst, true);
        }
    } else {
        // A ring of tiles, all but one of them in flight.
        constexpr int kStageBytes = 2 * L::kBytes;
        auto issue = [&](int tile) {
            const uint32_t dst = lds_base + static_cast<uint32_t>(tile % kStages) * kStageBytes;
            fetch(begin + tile * L::kTokens, ring_v ? dst + L::kBytes : dst, ring_v);
        };
        for (int i = 0; i < kStages - 1 && i < tiles; ++i) issue(i);
        // The ring's steps written out, so that LDS addresses are constants.
        auto step = [&](auto at, int i) {
            constexpr int kAt = decltype(at)::value;
            // This wave's copies of tile i have landed; those of the tiles behind
            // it (fewer at the end) are in flight.
            if (i + kStages - 2 < tiles && a.head_dim == kD) wait_vm<(kStages - 2) * kCopies>(); else wait_vm<0>();
            bare_barrier();  // and every wave is past tile i - 1, whose place is filled next
            if (i + kStages - 1 < tiles) issue(i + kStages - 1);
            uint8_t* k = lds + kAt * kStageBytes;
            uint8_t* v = k + L::kBytes;
            typename L::Score s = L::scores(k, q, lane);
            const int first = begin + i * L::kTokens;
            const bool partial = edge(first);
            if (partial) mask(s, in_range(first));
            soften(s);
            if (partial) {
                clear(v, in_range(first), tid, kThreads);
                __syncthreads();
            }
            L::values(v, s, acc, lane);
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

    const int64_t slot_rows = static_cast<int64_t>(w.slot) * a.sequences * a.heads;
    if constexpr (kSolo) {
#pragma unroll
        for (int d = L::kRows; d < kWaveSize; d <<= 1) l += __shfl_xor(l, d);
        if (row >= total_rows) return;
        const int64_t at = slot_rows + static_cast<int64_t>(w.first_sequence) * a.heads + w.kv_head * a.per + row;
        if (L::part_of(lane) == 0) {
            a.ml[2 * at] = m;
            a.ml[2 * at + 1] = l;
        }
#pragma unroll
        for (int i = 0; i < L::kAcc; i += 4) {
            f32x4_t four;
#pragma unroll
            for (int e = 0; e < 4; ++e) four[e] = acc[(i + e) / L::kScores][(i + e) % L::kScores];
            const int dim = L::dim_of(i, lane);
            if (dim < a.head_dim) *reinterpret_cast<f32x4_t*>(a.acc + at * a.pitch + dim) = four;
        }
        return;
    }
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
    __syncthreads();
    // Rows x groups of four dims, over the workgroup; token waves are joined.
    constexpr int kOutRows = kRowWaves * L::kRows;
    constexpr int kFours = kD / 4;
    constexpr int kRounds = (kOutRows * kFours + kThreads - 1) / kThreads;
#pragma unroll 4
    for (int n = 0; n < kRounds; ++n) {
        const int i = n * kThreads + tid;
        const int r = i / kFours;
        const int dim = (i % kFours) * 4;
        if (r >= kOutRows) break;
        const int owner = kRowWaves == 1 ? 0 : r / L::kRows;
        const int lr = r % L::kRows;
        const int out_row = lds_row[owner][lr];
        if (out_row < 0 || dim >= a.head_dim) continue;
        const int64_t at = slot_rows + out_row;
        float mm = lds_m[owner][lr];
#pragma unroll
        for (int t = 1; t < kTokenWaves; ++t) mm = fmaxf(mm, lds_m[t][lr]);
        float ll = 0.0f;
        f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < kTokenWaves; ++t) {
            const int src = owner + t;
            const float f = kTokenWaves == 1 ? 1.0f : lds_m[src][lr] == -INFINITY ? 0.0f : exp2f(lds_m[src][lr] - mm);
            // A wave without a finite score still passes its NaN on.
            ll += kTokenWaves > 1 && lds_m[src][lr] == -INFINITY ? lds_l[src][lr] : lds_l[src][lr] * f;
            const f32x4_t four = *reinterpret_cast<const f32x4_t*>(
                reinterpret_cast<const float*>(lds) + (src * L::kRows + lr) * L::kOutPitch + dim);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = fmaf(four[e], f, sum[e]);
        }
        if (dim == 0) {
            a.ml[2 * at] = mm;
            a.ml[2 * at + 1] = ll;
        }
        *reinterpret_cast<f32x4_t*>(a.acc + at * a.pitch + dim) = sum;
    }
}

/// Prefix tiles of four waves' rows, or of one's (kRowWaves 1: the four take
/// different tokens).
template <typename T, int kD, int kRowWaves>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(kD > 128 ? 1 : 2, 4))) void shared_attention_kernel(SharedArgs a) {
    using L = Tile<T, kD>;
    __shared__ __attribute__((aligned(16))) uint8_t lds[lds_bytes<T, kD>()];
    __shared__ float lds_m[kWaves][32];
    __shared__ float lds_l[kWaves][32];
    __shared__ int lds_row[kWaves][32];
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    Item w{};
    int id = static_cast<int>(blockIdx.x);
    if (id < a.prefix_items) {
        // Workgroup i runs on XCD i % 8. The (range, KV head) pairs of a prefix are
        // cut into eight runs, one per XCD, heads varying fastest: an XCD then
        // reads neighbouring tokens with all their heads, and all row tiles of a
        // pair, whose L2 serves them from one read.
        constexpr int kRows = kRowWaves * L::kRows;
        const PrefixItem p = prefix_item(a, kRows, a.prefix_step, a.prefix_least, id / 8);
        const Group& g = p.group;
        if (g.end == 0) return;
        const int pair = id % 8 * p.run + p.place;
        const int split = pair / a.kv_heads;
        w.kv_head = pair % a.kv_heads;
        const Range range = range_of(0, g.prefix, p.each, split);
        w.lo = range.lo;
        w.hi = range.hi;
        if (w.lo >= w.hi) return;
        // The pages of the first sequence that holds the whole prefix.
        int holder = -1;
        for (int s = g.first; s < g.end; s += kWaveSize) {
            const bool holds = s + lane < g.end && context_of(a, s + lane) >= g.prefix;
            const uint64_t any = __builtin_amdgcn_ballot_w64(holds);
            if (any != 0) {
                holder = s + __builtin_ctzll(any);
                break;
            }
        }
        if (holder < 0) return;
        w.table = a.tables + static_cast<int64_t>(holder) * a.max_blocks;
        w.last_block = static_cast<int>(static_cast<uint32_t>(w.hi - 1) / a.block_size);
        w.first_sequence = g.first;
        w.sequences = g.end - g.first;
        w.first_row = p.tile * kRows;
        w.least = g.prefix;
        w.slot = split;
        attend<T, kD, kRowWaves == 1 ? Waves::kTokens : Waves::kRows>(a, w, lds, lds_m, lds_l, lds_row);
    } else {
        // Where there are items enough, each wave has its own; else a workgroup.
        id -= a.prefix_items;
        const int rests = a.sequences * a.kv_heads * a.rest_tiles;
        const int per_layer = a.rest_solo ? (rests + kWaves - 1) / kWaves : rests;  // workgroups of one range index
        const int split = id / per_layer;
        id %= per_layer;
        if (per_layer % 8 == 0) id = id % 8 * (per_layer / 8) + id / 8;  // neighbours on one XCD, as above
        if (a.rest_solo) id = id * kWaves + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWaveSize);
        if (id >= rests) return;
        w.kv_head = id % a.kv_heads;
        id /= a.kv_heads;
        const int tile = id % a.rest_tiles;
        const int s = id / a.rest_tiles;
        const int context = context_of(a, s);
        const Group g = a.groups > 0 ? group_of(a, s) : Group{0, 0, 0};
        const int first = g.end > 0 && g.prefix <= context ? g.prefix : 0;
        const int each = split_length(context - first, a.rest_splits, a.rest_step, a.rest_least);
        const Range range = range_of(first, context - first, each, split);
        w.lo = range.lo;
        w.hi = range.hi;
        if (w.lo >= w.hi) return;
        w.table = a.tables + static_cast<int64_t>(s) * a.max_blocks;
        w.last_block = static_cast<int>(static_cast<uint32_t>(w.hi - 1) / a.block_size);
        w.first_sequence = s;
        w.sequences = 1;
        w.first_row = tile * L::kRows;
        w.least = 0;
        w.slot = a.prefix_splits + split;
        if (a.rest_solo) {
            attend<T, kD, Waves::kSolo>(a, w, lds, lds_m, lds_l, lds_row);
        } else {
            attend<T, kD, Waves::kTokens>(a, w, lds, lds_m, lds_l, lds_row);
        }
    }
}

/// Any head size and alignment: a wave per (sequence, head, range of the whole
/// context), a token at a time, dims over the lanes. No prefix is shared.
template <typename T, int kPer>
__global__ __launch_bounds__(kThreads) void shared_attention_any_kernel(SharedArgs a) {
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    const int64_t id = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWaveSize;
    if (id >= static_cast<int64_t>(a.sequences) * a.heads * a.rest_splits) return;
    const int split = static_cast<int>(id % a.rest_splits);
    const int64_t out_row = id / a.rest_splits;
    const int head = static_cast<int>(out_row % a.heads);
    const int s = static_cast<int>(out_row / a.heads);
    const int context = context_of(a, s);
    const int each = split_length(context, a.rest_splits, a.rest_step, a.rest_least);
    const Range range = range_of(0, context, each, split);
    const int lo = range.lo;
    const int hi = range.hi;
    if (lo >= hi) return;
    const T* q = static_cast<const T*>(a.query) + out_row * a.head_dim;
    float qv[kPer];
    float acc[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = lane + i * kWaveSize;
        qv[i] = d < a.head_dim ? Storage<T>::load(q + d) : 0.0f;
        acc[i] = 0.0f;
    }
    float m = -INFINITY;
    float l = 0.0f;
    for (int t = lo; t < hi; ++t) {
        const uint32_t page = a.tables[static_cast<int64_t>(s) * a.max_blocks + t / a.block_size];
        if (page >= a.pages) continue;
        const int64_t row = static_cast<int64_t>(page) * a.block_size + t % a.block_size;
        const int64_t at = (row * a.kv_heads + head / a.per) * a.head_dim;
        const T* k = static_cast<const T*>(a.k_cache) + at;
        const T* v = static_cast<const T*>(a.v_cache) + at;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int d = lane + i * kWaveSize;
            if (d < a.head_dim) dot = fmaf(qv[i], Storage<T>::load(k + d), dot);
        }
        const float y = wave_reduce_f32<AddF32>(dot) * (a.query_sign != 0 ? -a.c : a.c);
        const float m_new = fmaxf(m, y);
        const float shift = m_new == -INFINITY ? 0.0f : m_new;
        const float f = exp2f(m - shift);
        const float p = exp2f(y - shift);
        m = m_new;
        l = fmaf(l, f, p);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int d = lane + i * kWaveSize;
            if (d < a.head_dim) acc[i] = fmaf(acc[i], f, p * Storage<T>::load(v + d));
        }
    }
    const int64_t slot_row = static_cast<int64_t>(split) * a.sequences * a.heads + out_row;
    if (lane == 0) {
        a.ml[2 * slot_row] = m;
        a.ml[2 * slot_row + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = lane + i * kWaveSize;
        if (d < a.head_dim) a.acc[slot_row * a.pitch + d] = acc[i];
    }
}

/// Joins the pieces of one (sequence, head): four waves each, or one where there
/// are rows enough to fill the GPU with that.
template <typename T, int kD, int kRowWaves>
__global__ __launch_bounds__(kThreads) void shared_attention_join_kernel(SharedArgs a) {
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    const int64_t rows = static_cast<int64_t>(a.sequences) * a.heads;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWaveSize);
    const int row = static_cast<int>(blockIdx.x) * (kWaves / kRowWaves) + (kRowWaves == 1 ? wave : 0);
    if (row >= rows) return;
    const int s = row / a.heads;
    const int context = context_of(a, s);
    int first = 0;
    int prefix_pieces = 0;
    if (a.prefix_step > 0) {
        const Group g = group_of(a, s);
        if (g.end > 0 && g.prefix <= context && g.prefix > 0) {
            first = g.prefix;
            const int each = split_length(first, a.prefix_splits, a.prefix_step, a.prefix_least);
            prefix_pieces = range_count(first, each);
        }
    }
    int rest_pieces = 0;
    if (context > first) {
        const int each = split_length(context - first, a.rest_splits, a.rest_step, a.rest_least);
        rest_pieces = range_count(context - first, each);
    }
    const int pieces = prefix_pieces + rest_pieces;
    auto slot_of = [&](int i) { return i < prefix_pieces ? i : a.prefix_splits + i - prefix_pieces; };
    // Every wave weighs all pieces: lane i piece i (at most 2 x 64).
    static_assert(kMaxSplits <= kWaveSize, "two pieces per lane");
    float pm[2], pl[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int i = lane + n * kWaveSize;
        pm[n] = -INFINITY;
        pl[n] = 0.0f;
        if (i < pieces) {
            const int64_t at = slot_of(i) * rows + row;
            pm[n] = a.ml[2 * at];
            pl[n] = a.ml[2 * at + 1];
        }
    }
    // Threads: groups of kLanes lanes take the pieces in turn, four dims a lane.
    constexpr int kLanes = kD / 4;
    constexpr int kTeams = kRowWaves * kWaveSize / kLanes;
    constexpr int kAhead = 4;
    const int thread = kRowWaves == 1 ? lane : static_cast<int>(threadIdx.x);
    const int team = thread / kLanes;
    const int dim = (thread % kLanes) * 4;
    f32x4_t part[kAhead];
    auto load = [&](int i0) {
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const int i = i0 + n * kTeams + team;
            part[n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (i < pieces && dim < a.head_dim) {
                part[n] = *reinterpret_cast<const f32x4_t*>(a.acc + (slot_of(i) * rows + row) * a.pitch + dim);
            }
        }
    };
    load(0);  // in flight while the weights are found
    const float m = wave_reduce_f32<MaxF32>(fmaxf(pm[0], pm[1]));
    float weight[2];
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        weight[n] = pm[n] == -INFINITY ? 0.0f : exp2f(pm[n] - m);
        sum += pm[n] == -INFINITY ? pl[n] : pl[n] * weight[n];
    }
    const float l = wave_reduce_f32<AddF32>(sum);
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = 0; i0 < pieces; i0 += kAhead * kTeams) {
        if (i0 > 0) load(i0);
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const int i = i0 + n * kTeams + team;
            const float low = __shfl(weight[0], i & (kWaveSize - 1));
            const float high = __shfl(weight[1], i & (kWaveSize - 1));
            const float f = i < kWaveSize ? low : high;
            if (i < pieces) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(part[n][e], f, o[e]);
            }
        }
    }
    __shared__ __attribute__((aligned(16))) float all_teams[kWaves / kRowWaves][kTeams][kD];
    auto& teams = all_teams[kRowWaves == 1 ? wave : 0];
    *reinterpret_cast<f32x4_t*>(&teams[team][dim]) = o;
    if constexpr (kRowWaves == 1) wait_lds(); else __syncthreads();
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(row) * a.head_dim;
    for (int d = thread; d < a.head_dim; d += kRowWaves * kWaveSize) {
        float v = teams[0][d];
#pragma unroll
        for (int t = 1; t < kTeams; ++t) v += teams[t][d];
        Storage<T>::store(out + d, l == 0.0f ? 0.0f : v * inverse);
    }
}

// ---- host -----------------------------------------------------------------------

struct Plan {
    int dim;        // head size of the matrix kernel, or 0: the general kernel
    int row_waves;  // prefix tiles of 1 or 4 waves' rows
    int prefix_least;
    int prefix_splits;
    int rest_splits;
    int prefix_tiles;
    int rest_tiles;
    int prefix_step;
    int rest_step;
    int rest_least;
    bool rest_solo;
};

Plan plan_of(cf_dtype dtype, int64_t sequences, int64_t groups, int64_t heads, int64_t kv_heads, int64_t head_dim,
             int64_t capacity) {
    Plan p{};
    const int64_t per = heads / kv_heads;
    const bool wide = dtype == CF_F32;
    const int64_t vec = wide ? 4 : 8;
    if (head_dim % vec == 0 && head_dim <= (wide ? 128 : 256)) p.dim = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    auto splits = [&](int64_t items, int64_t target, int64_t least) {
        int64_t n = items > 0 ? target / items : 1;
        const int64_t most = ceil_div<int64_t>(capacity, least);
        if (n > most) n = most;
        if (n > kMaxSplits) n = kMaxSplits;
        return static_cast<int>(n < 1 ? 1 : n);
    };
    if (p.dim == 0) {
        p.rest_splits = splits(sequences * heads, 4096, 64);
        p.rest_step = p.rest_least = 32;
        return p;
    }
    const int64_t wave_rows = wide ? 16 : 32;
    const int64_t rows = sequences * per;
    constexpr int64_t slots = 512;  // workgroups at two per CU
    p.row_waves = 1;
    if (groups > 0) {
        // Four waves of rows where the groups fill more than two waves' on
        // average; below, two tiles of one wave's rows, four waves over their
        // tokens (64 rows behind 2048 tokens, 8 KV heads of 128 in bf16: 14.4 ->
        // 10.1 us, 32 rows in fp32 14.0 -> 11.9). Eight waves of rows, a workgroup
        // per CU, were within 3% from 16384 shared tokens on and up to 16% slower
        // below.
        p.row_waves = rows > 2 * wave_rows * groups ? 4 : 1;
        // A tile has as many tokens as a wave has rows.
        p.prefix_step = static_cast<int>(p.row_waves == 4 ? wave_rows : kWaves * wave_rows);
        p.prefix_least = p.row_waves == 1 ? 128 : wide ? 64 : 256;
        const int64_t tile = p.row_waves * wave_rows;
        p.prefix_tiles = static_cast<int>((rows + groups * (tile - 1)) / tile);  // at most, however the groups lie
        const int64_t likely = ceil_div<int64_t>(rows, tile * groups) * groups;
        p.prefix_splits = splits(likely * kv_heads, slots, p.prefix_least);
    }
    p.rest_tiles = static_cast<int>(ceil_div<int64_t>(per, wave_rows));
    // A wave for every rest where that fills the GPU (2048 waves at two per
    // SIMD) well enough; its ranges are then whole tiles.
    const int64_t rests = sequences * kv_heads * p.rest_tiles;
    p.rest_solo = rests >= 256;
    p.rest_least = p.rest_solo ? 256 : 128;
    p.rest_splits = splits(rests, p.rest_solo ? slots * kWaves : slots, p.rest_least);
    p.rest_step = static_cast<int>(wave_rows) * (p.rest_solo ? 1 : kWaves);
    return p;
}

int64_t capacity_of(int64_t max_blocks, int64_t block_size) {
    return max_blocks > kMostTokens / block_size ? kMostTokens : max_blocks * block_size;
}

size_t workspace_of(const Plan& p, int64_t sequences, int64_t heads, int64_t head_dim) {
    const size_t slots = static_cast<size_t>(p.prefix_splits) + p.rest_splits;
    const size_t rows = static_cast<size_t>(sequences) * heads;
    return (slots * rows * 8 + 15) / 16 * 16 + slots * rows * ((head_dim + 3) / 4 * 4) * 4;
}

bool sizes_ok(int64_t sequences, int64_t groups, int64_t heads, int64_t kv_heads, int64_t head_dim,
              int64_t block_size, int64_t max_blocks) {
    return sequences > 0 && groups >= 0 && heads > 0 && kv_heads > 0 && head_dim > 0 && head_dim <= 1024 &&
           block_size > 0 && max_blocks > 0 && heads % kv_heads == 0;
}

/// A wave per row from a round of the GPU's waves on (2048 rows: 9.4 -> 6.5 us).
bool join_by_wave(int64_t rows, int64_t head_dim) { return rows >= 1024 && head_dim <= 256; }

template <typename T, int kD>
void run_matrix(const SharedArgs& a, const Plan& p, dim3 grid, hipStream_t stream) {
    if (p.row_waves == 4) {
        launch(shared_attention_kernel<T, kD, 4>, grid, dim3(kThreads), 0, stream, a);
    } else {
        launch(shared_attention_kernel<T, kD, 1>, grid, dim3(kThreads), 0, stream, a);
    }
}

template <typename T>
void run(const SharedArgs& a, const Plan& p, hipStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.sequences) * a.heads;
    if (p.dim == 0) {
        const dim3 grid(static_cast<unsigned>(ceil_div<int64_t>(rows * a.rest_splits, kWaves)));
        if (a.head_dim <= 128) {
            launch(shared_attention_any_kernel<T, 2>, grid, dim3(kThreads), 0, stream, a);
        } else {
            launch(shared_attention_any_kernel<T, 16>, grid, dim3(kThreads), 0, stream, a);
        }
    } else {
        int64_t rest = static_cast<int64_t>(a.sequences) * a.kv_heads * a.rest_tiles;
        if (a.rest_solo) rest = ceil_div<int64_t>(rest, kWaves);
        rest *= a.rest_splits;
        const dim3 grid(static_cast<unsigned>(a.prefix_items + rest));
        if (p.dim == 64) {
            run_matrix<T, 64>(a, p, grid, stream);
        } else if (p.dim == 128) {
            run_matrix<T, 128>(a, p, grid, stream);
        } else if constexpr (sizeof(T) == 2) {
            run_matrix<T, 256>(a, p, grid, stream);
        }
    }
    const bool one_wave = join_by_wave(rows, a.head_dim);
    auto* join = one_wave ? (a.head_dim <= 64    ? shared_attention_join_kernel<T, 64, 1>
                             : a.head_dim <= 128 ? shared_attention_join_kernel<T, 128, 1>
                                                 : shared_attention_join_kernel<T, 256, 1>)
                          : (a.head_dim <= 64    ? shared_attention_join_kernel<T, 64, 4>
                             : a.head_dim <= 128 ? shared_attention_join_kernel<T, 128, 4>
                             : a.head_dim <= 256 ? shared_attention_join_kernel<T, 256, 4>
                                                 : shared_attention_join_kernel<T, 1024, 4>);
    launch(join, dim3(static_cast<unsigned>(one_wave ? ceil_div<int64_t>(rows, kWaves) : rows)), dim3(kThreads), 0,
           stream, a);
}

}  // namespace
}  // namespace cf

extern "C" {

size_t cf_paged_attention_shared_workspace_bytes(cf_dtype dtype, int64_t num_sequences, int64_t num_groups,
                                                 int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                                 int64_t block_size, int64_t max_blocks_per_sequence) {
    if (!cf::valid_dtype(dtype) || !cf::sizes_ok(num_sequences, num_groups, num_heads, num_kv_heads, head_dim,
                                                 block_size, max_blocks_per_sequence)) {
        return 0;
    }
    const cf::Plan p = cf::plan_of(dtype, num_sequences, num_groups, num_heads, num_kv_heads, head_dim,
                                   cf::capacity_of(max_blocks_per_sequence, block_size));
    return cf::workspace_of(p, num_sequences, num_heads, head_dim);
}

cf_status cf_paged_attention_shared(const void* query, const void* k_cache, const void* v_cache,
                                    const int32_t* group_starts, const int32_t* prefix_lens,
                                    const uint32_t* block_tables, const int32_t* context_lens, void* out,
                                    cf_dtype dtype, int64_t num_pages, int64_t num_sequences, int64_t num_groups,
                                    int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                    int64_t max_blocks_per_sequence, float scale, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    CF_ENTRY();
    const char* who = "cf_paged_attention_shared";
    if (num_sequences <= 0 || num_heads <= 0 || head_dim <= 0) return CF_OK;
    CF_REQUIRE(cf::valid_dtype(dtype), "%s: unknown dtype %d", who, static_cast<int>(dtype));
    CF_REQUIRE(cf::sizes_ok(num_sequences, num_groups, num_heads, num_kv_heads, head_dim, block_size,
                            max_blocks_per_sequence) && num_pages > 0,
               "%s: %lld heads over %lld KV heads of %lld (at most 1024), blocks of %lld, %lld per sequence, %lld "
               "pages, %lld groups",
               who, static_cast<long long>(num_heads), static_cast<long long>(num_kv_heads),
               static_cast<long long>(head_dim), static_cast<long long>(block_size),
               static_cast<long long>(max_blocks_per_sequence), static_cast<long long>(num_pages),
               static_cast<long long>(num_groups));
    CF_REQUIRE(query != nullptr && k_cache != nullptr && v_cache != nullptr && block_tables != nullptr &&
                   context_lens != nullptr && out != nullptr,
               "%s: null pointer", who);
    CF_REQUIRE(num_groups == 0 || (group_starts != nullptr && prefix_lens != nullptr), "%s: null pointer", who);
    const size_t size = cf::dtype_size(dtype);
    CF_REQUIRE(cf::host_aligned(query, size) && cf::host_aligned(k_cache, size) && cf::host_aligned(v_cache, size) &&
                   cf::host_aligned(out, size),
               "%s: misaligned pointer", who);
    // Cache rows, token positions and work items are counted in 32 bits.
    constexpr int64_t kMost = cf::kMostTokens;
    CF_REQUIRE(num_pages <= kMost / block_size && max_blocks_per_sequence <= kMost && num_kv_heads <= (1 << 14) && num_groups <= (1 << 20) &&
                   num_sequences <= kMost / num_heads,
               "%s: %lld pages of %lld tokens, %lld sequences of %lld heads, %lld KV heads or %lld groups exceed 32-bit counts", who,
               static_cast<long long>(num_pages), static_cast<long long>(block_size),
               static_cast<long long>(num_sequences), static_cast<long long>(num_heads),
               static_cast<long long>(num_kv_heads), static_cast<long long>(num_groups));
    cf::Plan p = cf::plan_of(dtype, num_sequences, num_groups, num_heads, num_kv_heads, head_dim,
                             cf::capacity_of(max_blocks_per_sequence, block_size));
    const size_t needed = cf::workspace_of(p, num_sequences, num_heads, head_dim);
    CF_REQUIRE(workspace != nullptr && workspace_bytes >= needed && cf::host_aligned(workspace, 16),
               "%s: needs %zu bytes of 16-byte aligned workspace", who, needed);
    if (p.dim != 0 && !(cf::host_aligned(query, 16) && cf::host_aligned(k_cache, 16) && cf::host_aligned(v_cache, 16))) {
        p.dim = 0;  // same workspace, read as ranges of whole contexts
        p.prefix_splits = p.prefix_step = 0;
        p.rest_step = p.rest_least = 32;
    }
    cf::SharedArgs a{};
    a.query = query;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.starts = group_starts;
    a.prefix = prefix_lens;
    a.tables = block_tables;
    a.context = context_lens;
    a.out = out;
    a.pages = static_cast<uint32_t>(num_pages);
    a.block_size = static_cast<uint32_t>(block_size);
    a.block_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctzll(static_cast<uint64_t>(block_size)) : -1;
    const uint64_t page_bytes = static_cast<uint64_t>(block_size) * num_kv_heads * head_dim * size;
    a.page_bytes = page_bytes < (uint64_t{1} << 32) ? static_cast<uint32_t>(page_bytes) : 0;
    a.sequences = static_cast<int>(num_sequences);
    a.heads = static_cast<int>(num_heads);
    a.kv_heads = static_cast<int>(num_kv_heads);
    a.per = static_cast<int>(num_heads / num_kv_heads);
    a.head_dim = static_cast<int>(head_dim);
    a.pitch = (a.head_dim + 3) / 4 * 4;
    a.groups = p.dim != 0 ? static_cast<int>(num_groups) : 0;
    a.max_blocks = static_cast<int>(max_blocks_per_sequence);
    a.capacity = static_cast<int>(cf::capacity_of(max_blocks_per_sequence, block_size));
    a.prefix_splits = p.prefix_splits;
    a.rest_splits = p.rest_splits;
    a.prefix_tiles = p.prefix_tiles;
    a.rest_tiles = p.rest_tiles;
    a.prefix_step = p.prefix_step;
    a.prefix_least = p.prefix_least;
    a.rest_step = p.rest_step;
    a.rest_least = p.rest_least;
    a.rest_solo = p.rest_solo;
    const int64_t prefix_items =
        a.groups > 0 ? (num_kv_heads * p.prefix_splits + 7) / 8 * 8 * p.prefix_tiles : 0;
    const int64_t rest_items = num_sequences * num_kv_heads * (p.rest_tiles > 0 ? p.rest_tiles : 1) * p.rest_splits;
    CF_REQUIRE(prefix_items + rest_items < kMost && num_sequences * num_heads * p.rest_splits < kMost,
               "%s: too many work items", who);
    const int64_t rows_in_all = num_sequences * num_heads;
    const int64_t workgroups =
        p.dim == 0 ? cf::ceil_div<int64_t>(rows_in_all * p.rest_splits, cf::kWaves)
                   : prefix_items + (p.rest_solo ? cf::ceil_div<int64_t>(rest_items / p.rest_splits, cf::kWaves) *
                                                       p.rest_splits
                                                 : rest_items);
    const int64_t joins =
        cf::join_by_wave(rows_in_all, head_dim) ? cf::ceil_div<int64_t>(rows_in_all, cf::kWaves) : rows_in_all;
    CF_REQUIRE(workgroups <= cf::kMaxWorkgroups && joins <= cf::kMaxWorkgroups,
               "%s: %lld sequences of %lld heads are too many for a launch", who,
               static_cast<long long>(num_sequences), static_cast<long long>(num_heads));
    a.prefix_items = static_cast<int>(prefix_items);
    // The kernels take maxima of unscaled scores, so the factor must not be
    // negative, nor 0 (which times a masked score is NaN).
    const float c = scale * cf::kLog2e;
    a.c = c == 0.0f ? 1.0e-37f : c < 0.0f ? -c : c;
    a.query_sign = c < 0.0f ? (dtype == CF_F32 ? 0x80000000u : 0x80008000u) : 0u;
    const size_t rows = static_cast<size_t>(num_sequences) * num_heads;
    const size_t slots = static_cast<size_t>(p.prefix_splits) + p.rest_splits;
    a.ml = static_cast<float*>(workspace);
    a.acc = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (slots * rows * 8 + 15) / 16 * 16);
    auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case CF_F32: cf::run<float>(a, p, s); break;
        case CF_F16: cf::run<cf::f16_t>(a, p, s); break;
        case CF_BF16: cf::run<cf::bf16_t>(a, p, s); break;
    }
    return cf::check_launch("launching shared-prefix paged attention", s);
}

}  // extern "C"
