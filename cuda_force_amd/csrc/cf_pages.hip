// Pages of a paged KV cache: copy, fork, extend, release, compact.
//
// State, all on the device: ref_counts [pages] (how many table rows name a
// page; a page with a count <= 0 is free), block_tables [sequences, width],
// context_lens [sequences]. Caches are tensors of `pages` pages of page_bytes
// bytes each (a K and a V per layer), whatever their type.
//
// Nothing is read back by the host, so every operator decides on the device:
// a planning kernel settles which entries of its list take part and which free
// pages they get (the lowest, in the order of the list), a second one moves the
// data. Results depend on the inputs alone: of two entries that claim the same
// row or page the earlier one wins (an integer minimum), reference counts are
// integer sums, and free pages come out of an ordered scan.
//   * The plan of a list runs in one workgroup of 1024 threads: phases divided
//     by barriers instead of launches, and nothing but the order of the phases
//     to keep between them. The search for free pages reads 16384 counts a step
//     and ends when it has enough. Bound by the chain of loads and atomics:
//     32 forks of 8 sequences 5.1 us, their extension 5.4 us, 1500 pairs of a copy
//     4.9 us; claims and short lists of pages are exchanged in LDS for that.
//   * Copies are bound by HBM: 16 KiB per workgroup and step, four 16-byte loads
//     in flight per lane, streamed past the caches. 1500 pages of 32 KiB in four
//     tensors (393 MB read and written) 78 us, 5.0 TB/s; 32 KiB per workgroup
//     took 80 us, and a grid that loops over the chunks 80 us.
//   * Compaction: 48 sequences' 195 MB read and written 37 us, after 11 us that
//     list the moves. Counting and listing in one launch where the pool is small
//     took 9 us of those 11 but left the whole as it was, so there is one way.
#include <type_traits>

#include "cf_common.hpp"

namespace cf {
namespace {

constexpr int kTensors = CF_CACHE_TENSORS_MAX;  // per launch
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWaveSize;
constexpr int kCountsPerThread = 16;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int64_t kChunkBytes = int64_t{kCopyThreads} * kCopyUnroll * 16;
constexpr int kTilePages = kCopyThreads * kCountsPerThread;  // counts per workgroup of the compaction's scan
/// Plans over at most so many rows (a copy: pages) exchange their claims in LDS,
/// those of forks and extensions if they want at most kPlanThreads pages: atomics
/// and loads past the CU's cache cost most of a plan's time otherwise (32 forks
/// 8.1 -> 5.6 us, 32 rows extended 8.0 -> 5.5, 1500 pairs copied 10.6 -> 4.9; these
/// take 14 us in a pool of 100000 pages).
constexpr int kSmallRows = 8192;
constexpr int kUnclaimed = 0x7FFFFFFF;
constexpr int kNamed = kUnclaimed - 1;

struct Tensors {
    uint8_t* p[kTensors];
};

// ---- memory that several waves of a plan exchange through ---------------------

/// Loads and stores at device scope: claims are made by atomics, which act
/// behind the CU's own cache.
__device__ __forceinline__ int peek(const int* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void poke(int* p, int v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
/// Barrier between two phases of a plan. One workgroup runs it, and all that
/// its threads exchange through memory goes by peek, poke and atomics, past the
/// CU's cache: it is enough that these have arrived. A fence at device scope
/// writes L2 back as well, microseconds each time.
__device__ __forceinline__ void phase() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

/// Numbers that a plan's threads exchange: in the workspace, or in LDS.
struct InMemory {
    int* p;
    __device__ __forceinline__ int get(int64_t i) const { return peek(p + i); }
    __device__ __forceinline__ void put(int64_t i, int v) const { poke(p + i, v); }
    __device__ __forceinline__ void lower(int64_t i, int v) const { atomicMin(p + i, v); }
    __device__ __forceinline__ static void phase() { cf::phase(); }
};
struct InLds {
    int* p;
    __device__ __forceinline__ int get(int64_t i) const { return p[i]; }
    __device__ __forceinline__ void put(int64_t i, int v) const { p[i] = v; }
    __device__ __forceinline__ void lower(int64_t i, int v) const { atomicMin(p + i, v); }
    __device__ __forceinline__ static void phase() { __syncthreads(); }
};

/// Sum of v over lower threads; `total` over all. Every thread calls it. Sums
/// of pages, entries or tokens wanted: at most kMostInts.
template <int kWaves>
__device__ __forceinline__ int scan_before(int v, int* slots, int& total) {
    const int lane = static_cast<int>(threadIdx.x) & (kWaveSize - 1);
    const int wave = static_cast<int>(threadIdx.x) / kWaveSize;
    int sum = v;
#pragma unroll
    for (int d = 1; d < kWaveSize; d <<= 1) {
        const int o = __shfl_up(sum, d);
        if (lane >= d) sum += o;
    }
    __syncthreads();  // the last call's slots have been read
    if (lane == kWaveSize - 1) slots[wave] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += slots[w];
        total += slots[w];
    }
    return before + sum - v;
}

/// Counts of pages first .. first + 15, 1 (taken) past the end.
__device__ __forceinline__ void load_counts(const int* counts, int64_t pages, int64_t first, bool aligned,
                                            int (&c)[kCountsPerThread]) {
    if (aligned && first + kCountsPerThread <= pages) {
#pragma unroll
        for (int i = 0; i < kCountsPerThread / 4; ++i) {
            const int4 four = reinterpret_cast<const int4*>(counts + first)[i];
            c[4 * i] = four.x;
            c[4 * i + 1] = four.y;
            c[4 * i + 2] = four.z;
            c[4 * i + 3] = four.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kCountsPerThread; ++i) c[i] = first + i < pages ? counts[first + i] : 1;
    }
}

/// The lowest `wanted` free pages into `list`, ascending; returns how many
/// there are (at most `wanted`). The whole planning workgroup calls it.
template <typename Ints>
__device__ int64_t find_free(const int* counts, int64_t pages, int64_t wanted, const Ints& list, int* slots) {
    int64_t found = 0;
    const bool aligned = aligned16(counts);
    for (int64_t base = 0; base < pages && found < wanted; base += int64_t{kPlanThreads} * kCountsPerThread) {
        const int64_t first = base + int64_t{threadIdx.x} * kCountsPerThread;
        int c[kCountsPerThread];
        load_counts(counts, pages, first, aligned, c);
        int mine = 0;
#pragma unroll
        for (int i = 0; i < kCountsPerThread; ++i) mine += c[i] <= 0 ? 1 : 0;
        int total;
        int64_t at = found + scan_before<kPlanWaves>(mine, slots, total);
#pragma unroll
        for (int i = 0; i < kCountsPerThread; ++i) {
            if (c[i] > 0) continue;
            if (at < wanted) list.put(at, static_cast<int>(first + i));
            ++at;
        }
        found += total;
    }
    return found < wanted ? found : wanted;
}

__device__ __forceinline__ bool within(int v, int64_t size) { return v >= 0 && v < size; }

// ---- copies -----------------------------------------------------------------

/// Bytes [begin, end) of a page of one cache, by the workgroup; kUnit bytes an
/// access. At most kChunkBytes.
template <int kUnit>
__device__ __forceinline__ void copy_bytes(const uint8_t* from, uint8_t* to, int64_t begin, int64_t end) {
    const int tid = static_cast<int>(threadIdx.x);
    if constexpr (kUnit == 16) {
        uint4 v[kCopyUnroll];
        const int64_t at = begin + tid * 16;
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) {
            const int64_t b = at + u * kCopyThreads * 16;
            if (b < end) v[u] = load_stream16(from + b);
        }
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) {
            const int64_t b = at + u * kCopyThreads * 16;
            if (b < end) store_stream16(to + b, v[u]);
        }
    } else if constexpr (kUnit == 4) {
        for (int64_t b = begin + tid * 4; b < end; b += kCopyThreads * 4) {
            *reinterpret_cast<uint32_t*>(to + b) = *reinterpret_cast<const uint32_t*>(from + b);
        }
    } else {
        for (int64_t b = begin + tid; b < end; b += kCopyThreads) to[b] = from[b];
    }
}

// ---- copy -------------------------------------------------------------------

/// Which pairs of a copy take part: status 0, or 1 for a pair out of range,
/// whose dst an earlier pair in range names, or whose src any pair names as its
/// dst (one out of range by its src too: such a dst is kNamed, claimed by none).
/// kSmall: claims in LDS.
template <bool kSmall>
__global__ __launch_bounds__(kPlanThreads) void copy_plan_kernel(const int* src, const int* dst, int64_t count,
                                                                 int64_t pages, int* claims_, int* status) {
    using Ints = typename std::conditional<kSmall, InLds, InMemory>::type;
    __shared__ int lds[kSmall ? kSmallRows : 1];
    const Ints claims{kSmall ? lds : claims_};
    for (int64_t i = threadIdx.x; i < count; i += kPlanThreads) {
        if (within(src[i], pages)) claims.put(src[i], kUnclaimed);
        if (within(dst[i], pages)) claims.put(dst[i], kUnclaimed);
    }
    Ints::phase();
    for (int64_t i = threadIdx.x; i < count; i += kPlanThreads) {
        if (within(dst[i], pages)) claims.lower(dst[i], within(src[i], pages) ? static_cast<int>(i) : kNamed);
    }
    Ints::phase();
    for (int64_t i = threadIdx.x; i < count; i += kPlanThreads) {
        const bool good = within(src[i], pages) && within(dst[i], pages) && claims.get(dst[i]) == i &&
                          claims.get(src[i]) == kUnclaimed;
        status[i] = good ? 0 : 1;
    }
}

template <int kUnit>
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(Tensors t, int tensors, int64_t page_bytes,
                                                                  int64_t chunks, const int* src, const int* dst,
                                                                  const int* status) {
    int64_t id = blockIdx.x;
    const int64_t chunk = id % chunks;
    id /= chunks;
    const int tensor = static_cast<int>(id % tensors);
    const int64_t pair = id / tensors;
    if (status[pair] != 0) return;
    const int64_t begin = chunk * kChunkBytes;
    const int64_t end = begin + kChunkBytes < page_bytes ? begin + kChunkBytes : page_bytes;
    copy_bytes<kUnit>(t.p[tensor] + src[pair] * page_bytes, t.p[tensor] + dst[pair] * page_bytes, begin, end);
}

// ---- fork and extend ----------------------------------------------------------

struct TableArgs {
    int* counts;
    uint32_t* tables;
    int* context;
    int64_t pages;
    int64_t block;
    int64_t sequences;
    int64_t width;
    int64_t capacity;  // tokens of a table row
};

/// Fork's plan. `fresh[i]`: the page that pair i's child gets in the place of
/// its parent's partial last page, -1 for none. kSmall: a pair a thread at most,
/// and claims and free pages in LDS.
template <bool kSmall>
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(TableArgs a, const int* parents, const int* children,
                                                                 int64_t count, int* claims_, int* fresh,
                                                                 int* free_list, int* status) {
    using Ints = typename std::conditional<kSmall, InLds, InMemory>::type;
    __shared__ int slots[kPlanWaves];
    __shared__ int lds[kSmall ? kSmallRows + kPlanThreads : 1];
    const Ints claims{kSmall ? lds : claims_};
    const Ints list{kSmall ? lds + kSmallRows : free_list};
    const int64_t rounds = kSmall ? 1 : (count + kPlanThreads - 1) / kPlanThreads;
    // A pair's parent's length where it may be forked, else 0.
    auto eligible = [&](int64_t i) {
        if (i >= count || !within(parents[i], a.sequences) || !within(children[i], a.sequences)) return 0;
        const int length = a.context[parents[i]];
        return length > 0 && length <= a.capacity && a.context[children[i]] <= 0 ? length : 0;
    };
    int mine = 0;  // kSmall: the thread's pair's
    for (int64_t r = 0; r < rounds; ++r) {
        const int64_t i = r * kPlanThreads + threadIdx.x;
        if (i < count && within(children[i], a.sequences)) claims.put(children[i], kUnclaimed);
    }
    if (kSmall) mine = eligible(threadIdx.x);
    Ints::phase();
    for (int64_t r = 0; r < rounds; ++r) {
        const int64_t i = r * kPlanThreads + threadIdx.x;
        if (kSmall ? mine > 0 : eligible(i) > 0) claims.lower(children[i], static_cast<int>(i));
    }
    Ints::phase();
    // Which pairs need a page, and how many before each do.
    int64_t wanted = 0;
    int rank = -1;
    bool wins = false;
    for (int64_t r = 0; r < rounds; ++r) {
        const int64_t i = r * kPlanThreads + threadIdx.x;
        const int length = kSmall ? mine : eligible(i);
        wins = length > 0 && claims.get(children[i]) == i;
        const bool needs = wins && static_cast<uint32_t>(length) % static_cast<uint32_t>(a.block) != 0;
        int total;
        const int64_t before = wanted + scan_before<kPlanWaves>(needs ? 1 : 0, slots, total);
        rank = needs ? static_cast<int>(before) : -1;
        if (!kSmall && i < count) {
            poke(fresh + i, rank);
            poke(status + i, wins ? 0 : 1);
        }
        wanted += total;
    }
    const int64_t found = find_free(a.counts, a.pages, wanted < a.pages ? wanted : a.pages, list, slots);
    Ints::phase();
    for (int64_t r = 0; r < rounds; ++r) {
        const int64_t i = r * kPlanThreads + threadIdx.x;
        if (i >= count) break;
        if (!kSmall) {
            wins = peek(status + i) == 0;
            rank = peek(fresh + i);
        }
        const bool enough = rank < found;
        int page = -1;
        if (wins && enough) {
            if (rank >= 0) {
                page = list.get(rank);
                a.counts[page] = 1;
            }
            a.context[children[i]] = a.context[parents[i]];
        }
        fresh[i] = page;
        status[i] = !wins ? 1 : enough ? 0 : 2;
    }
}

/// Table rows, counts (workgroup 0 of a pair) and the partial page's tokens.
template <int kUnit>
__global__ __launch_bounds__(kCopyThreads) void fork_move_kernel(TableArgs a, Tensors t, int tensors,
                                                                 int64_t page_bytes, int64_t chunks, bool with_tables,
                                                                 const int* parents, const int* children,
                                                                 const int* fresh, const int* status) {
    const int64_t pieces = chunks * tensors + (with_tables ? 1 : 0);
    const int64_t pair = blockIdx.x / pieces;
    int64_t piece = blockIdx.x % pieces;
    if (status[pair] != 0) return;
    const int64_t length = a.context[children[pair]];
    const int64_t whole = length / a.block;
    const uint32_t* from = a.tables + parents[pair] * a.width;
    const int page = fresh[pair];
    if (with_tables && piece-- == 0) {
        uint32_t* to = a.tables + children[pair] * a.width;
        for (int64_t i = threadIdx.x; i < whole; i += kCopyThreads) {
            const uint32_t p = from[i];
            to[i] = p;
            if (p < a.pages) atomicAdd(a.counts + p, 1);
        }
        if (threadIdx.x == 0 && page >= 0) to[whole] = static_cast<uint32_t>(page);
        return;
    }
    if (page < 0) return;
    const uint32_t old = from[whole];
    if (old >= a.pages) return;
    const int64_t begin = piece % chunks * kChunkBytes;
    const int64_t used = length % a.block * (page_bytes / a.block);
    const int64_t end = begin + kChunkBytes < used ? begin + kChunkBytes : used;
    uint8_t* cache = t.p[piece / chunks];
    copy_bytes<kUnit>(cache + old * page_bytes, cache + page * page_bytes, begin, end);
}

/// The flat slot of token `at` of a table row; -1 where the row names no page.
__device__ __forceinline__ int64_t slot_of(const TableArgs& a, int64_t sequence, int64_t at) {
    const uint32_t block = static_cast<uint32_t>(a.block);
    const uint32_t token = static_cast<uint32_t>(at);  // below the capacity
    const uint32_t page = a.tables[sequence * a.width + token / block];
    return page < a.pages ? page * a.block + token % block : -1;
}

/// Extend, whole for one token a sequence (slots then holds count entries);
/// else slots are left to extend_slots_kernel. kSmall: an entry a thread at
/// most, and claims and free pages in LDS.
template <bool kSmall>
__global__ __launch_bounds__(kPlanThreads) void extend_kernel(TableArgs a, const int* sequences, int64_t count,
                                                              int64_t tokens, int* claims_, int64_t* ranks,
                                                              int* free_list, int* status, int64_t* slots_out) {
    using Ints = typename std::conditional<kSmall, InLds, InMemory>::type;
    __shared__ int slots[kPlanWaves];
    __shared__ int lds[kSmall ? kSmallRows + kPlanThreads : 1];
    const Ints claims{kSmall ? lds : claims_};
    const Ints list{kSmall ? lds + kSmallRows : free_list};
    const int64_t rounds = kSmall ? 1 : (count + kPlanThreads - 1) / kPlanThreads;
    for (int64_t r = 0; r < rounds; ++r) {
        const int64_t i = r * kPlanThreads + threadIdx.x;
        if (i < count && within(sequences[i], a.sequences)) claims.put(sequences[i], kUnclaimed);
    }
    Ints::phase();
    for (int64_t r = 0; r < rounds; ++r) {
        const int64_t i = r * kPlanThreads + threadIdx.x;
        if (i < count && within(sequences[i], a.sequences)) claims.lower(sequences[i], static_cast<int>(i));
    }
    Ints::phase();
    auto length_of = [&](int64_t i) { return static_cast<int64_t>(a.context[sequences[i]] > 0 ? a.context[sequences[i]] : 0); };
    // Lengths up to the capacity fit 31 bits, and the block 30.
    const uint32_t block = static_cast<uint32_t>(a.block);
    auto pages_of = [&](int64_t n) { return static_cast<int>((static_cast<uint32_t>(n) + block - 1) / block); };
    int64_t wanted = 0;
    int64_t rank = 0;
    bool wins = false;
    for (int64_t r = 0; r < rounds; ++r) {
        const int64_t i = r * kPlanThreads + threadIdx.x;
        wins = i < count && within(sequences[i], a.sequences) && claims.get(sequences[i]) == i &&
               length_of(i) + tokens <= a.capacity;
        const int need = wins ? pages_of(length_of(i) + tokens) - pages_of(length_of(i)) : 0;
        int total;
        rank = wanted + scan_before<kPlanWaves>(need, slots, total);
        if (!kSmall && i < count) {
            ranks[i] = rank;  // read by this thread alone
            poke(status + i, wins ? 0 : 1);
        }
        wanted += total;
    }
    const int64_t found = find_free(a.counts, a.pages, wanted < a.pages ? wanted : a.pages, list, slots);
    Ints::phase();
    for (int64_t r = 0; r < rounds; ++r) {
        const int64_t i = r * kPlanThreads + threadIdx.x;
        if (i >= count) break;
        if (!kSmall) {
            wins = peek(status + i) == 0;
            rank = ranks[i];
        }
        bool good = wins;
        int64_t length = 0;
        if (good) {
            length = length_of(i);
            const int64_t first = pages_of(length);
            const int need = pages_of(length + tokens) - static_cast<int>(first);
            if (need > 0 && rank + need > found) {
                good = false;
            } else {
                for (int k = 0; k < need; ++k) {
                    const int page = list.get(rank + k);
                    a.tables[sequences[i] * a.width + first + k] = static_cast<uint32_t>(page);
                    a.counts[page] = 1;
                }
                a.context[sequences[i]] = static_cast<int>(length + tokens);
            }
        }
        status[i] = good ? 0 : wins ? 2 : 1;
        if (tokens == 1) slots_out[i] = good ? slot_of(a, sequences[i], length) : -1;
    }
}

__global__ __launch_bounds__(kCopyThreads) void extend_slots_kernel(TableArgs a, const int* sequences, int64_t count,
                                                                    int64_t tokens, const int* status,
                                                                    int64_t* slots) {
    const int64_t id = int64_t{blockIdx.x} * kCopyThreads + threadIdx.x;
    if (id >= count * tokens) return;
    const int64_t i = id / tokens;
    slots[id] = status[i] == 0 ? slot_of(a, sequences[i], a.context[sequences[i]] - tokens + id % tokens) : -1;
}

// ---- release ------------------------------------------------------------------

__global__ __launch_bounds__(kCopyThreads) void release_kernel(TableArgs a, const int* sequences) {
    __shared__ int64_t held;
    const int s = sequences[blockIdx.x];
    if (!within(s, a.sequences)) return;
    if (threadIdx.x == 0) {
        // A sequence listed twice is empty the second time.
        const int64_t length = atomicExch(a.context + s, 0);
        const int64_t reach = length <= 0 ? 0 : (length + a.block - 1) / a.block;
        held = reach < a.width ? reach : a.width;
    }
    __syncthreads();
    for (int64_t i = threadIdx.x; i < held; i += kCopyThreads) {
        const uint32_t page = a.tables[s * a.width + i];
        // Not below 0: a count that was 0 already gets its 1 back.
        if (page < a.pages && atomicSub(a.counts + page, 1) <= 0) atomicAdd(a.counts + page, 1);
    }
}

// ---- compact ------------------------------------------------------------------

struct CompactArgs {
    const int* counts;
    const uint32_t* tables;
    const int* context;
    int* new_counts;
    uint32_t* new_tables;
    int* live;
    int64_t pages;
    int64_t block;
    int64_t sequences;
    int64_t width;
    int64_t tiles;
    int* tile_live;    // [tiles]
    int* holes;        // [pages]: free pages below the live count, ascending
    int* movers;       // [pages]: live pages from the live count on
    int* mover_count;  // [pages]: their reference counts
    int* rank;         // [pages]: a mover's place among them, else -1
    int* moves;        // [1]
};

__global__ __launch_bounds__(kCopyThreads) void compact_count_kernel(CompactArgs a) {
    __shared__ int slots[kCopyThreads / kWaveSize];
    const int64_t first = int64_t{blockIdx.x} * kTilePages + int64_t{threadIdx.x} * kCountsPerThread;
    int c[kCountsPerThread];
    load_counts(a.counts, a.pages, first, aligned16(a.counts), c);
    int live = 0;
#pragma unroll
    for (int i = 0; i < kCountsPerThread; ++i) live += c[i] > 0 && first + i < a.pages ? 1 : 0;
    int total;
    scan_before<kCopyThreads / kWaveSize>(live, slots, total);
    if (threadIdx.x == 0) a.tile_live[blockIdx.x] = static_cast<int>(total);
}

/// Every workgroup: the lists' entries of one tile of pages.
__global__ __launch_bounds__(kCopyThreads) void compact_list_kernel(CompactArgs a) {
    constexpr int kWaves = kCopyThreads / kWaveSize;
    __shared__ int slots[kWaves];
    const int64_t tile = blockIdx.x;
    // Live pages in all, before this tile, and before the tile that the live
    // count falls into.
    int all = 0, before = 0;
    for (int64_t i = threadIdx.x; i < a.tiles; i += kCopyThreads) {
        all += a.tile_live[i];
        if (i < tile) before += a.tile_live[i];
    }
    int live, base, unused;
    scan_before<kWaves>(all, slots, live);
    scan_before<kWaves>(before, slots, base);
    const bool aligned = aligned16(a.counts);
    int c[kCountsPerThread];
    // Live pages below the live count: what is not moved.
    const int64_t edge = live / kTilePages;
    int low = 0;
    for (int64_t i = threadIdx.x; i < edge && i < a.tiles; i += kCopyThreads) low += a.tile_live[i];
    if (edge < a.tiles) {
        const int64_t first = edge * kTilePages + int64_t{threadIdx.x} * kCountsPerThread;
        load_counts(a.counts, a.pages, first, aligned, c);
#pragma unroll
        for (int i = 0; i < kCountsPerThread; ++i) low += c[i] > 0 && first + i < live ? 1 : 0;
    }
    int kept;
    scan_before<kWaves>(low, slots, kept);
    const int64_t first = tile * kTilePages + int64_t{threadIdx.x} * kCountsPerThread;
    load_counts(a.counts, a.pages, first, aligned, c);
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kCountsPerThread; ++i) mine += c[i] > 0 && first + i < a.pages ? 1 : 0;
    int64_t at = base + scan_before<kWaves>(mine, slots, unused);  // live pages before the thread's first
#pragma unroll
    for (int i = 0; i < kCountsPerThread; ++i) {
        const int64_t page = first + i;
        if (page >= a.pages) break;
        const bool used = c[i] > 0;
        if (!used && page < live) a.holes[page - at] = static_cast<int>(page);
        int place = -1;
        if (used && page >= live) {
            place = static_cast<int>(at - kept);
            a.movers[place] = static_cast<int>(page);
            a.mover_count[place] = c[i];
        }
        a.rank[page] = place;
        at += used ? 1 : 0;
    }
    if (tile == 0 && threadIdx.x == 0) {
        *a.live = static_cast<int>(live);
        *a.moves = static_cast<int>(live - kept);
    }
}

/// Counts and table rows (first launch), and pages. A grid of any size.
template <int kUnit>
__global__ __launch_bounds__(kCopyThreads) void compact_move_kernel(CompactArgs a, Tensors t, int tensors,
                                                                    int64_t page_bytes, int64_t chunks,
                                                                    bool with_tables) {
    const int64_t moves = *a.moves;
    const int64_t items = moves * tensors * chunks;
    for (int64_t id = blockIdx.x; id < items; id += gridDim.x) {
        const int64_t begin = id % chunks * kChunkBytes;
        const int64_t end = begin + kChunkBytes < page_bytes ? begin + kChunkBytes : page_bytes;
        const int64_t move = id / chunks / tensors;
        uint8_t* cache = t.p[id / chunks % tensors];
        copy_bytes<kUnit>(cache + a.movers[move] * page_bytes, cache + a.holes[move] * page_bytes, begin, end);
    }
    if (!with_tables) return;
    const int64_t thread = int64_t{blockIdx.x} * kCopyThreads + threadIdx.x;
    const int64_t threads = int64_t{gridDim.x} * kCopyThreads;
    const int64_t live = *a.live;
    // A page's count is read and written by one thread: the arrays may be one.
    for (int64_t p = thread; p < a.pages; p += threads) {
        const int c = a.counts[p];
        if (p >= live) {
            a.new_counts[p] = 0;
        } else if (c > 0) {
            a.new_counts[p] = c;
        }
    }
    for (int64_t j = thread; j < moves; j += threads) a.new_counts[a.holes[j]] = a.mover_count[j];
    for (int64_t i = thread; i < a.sequences * a.width; i += threads) {
        const int64_t length = a.context[i / a.width];
        uint32_t page = a.tables[i];
        if (i % a.width * a.block < length && page < a.pages) {
            const int place = a.rank[page];
            if (place >= 0) page = static_cast<uint32_t>(a.holes[place]);
        }
        a.new_tables[i] = page;
    }
}

// ---- host -----------------------------------------------------------------------

constexpr int64_t kMostInts = int64_t{1} << 30;  // pages, rows, list entries: int32 with room to add

size_t align_up(size_t bytes) { return (bytes + 255) / 256 * 256; }

/// Bytes per access that pages of every tensor allow.
int unit_of(void* const* caches, int64_t tensors, int64_t page_bytes, int64_t token_bytes) {
    int unit = page_bytes % 16 == 0 && token_bytes % 16 == 0 ? 16 : page_bytes % 4 == 0 && token_bytes % 4 == 0 ? 4 : 1;
    for (int64_t i = 0; i < tensors; ++i) {
        while (!host_aligned(caches[i], static_cast<size_t>(unit))) unit = unit == 16 ? 4 : 1;
    }
    return unit;
}

cf_status check_caches(const char* who, void* const* caches, int64_t tensors, int64_t page_bytes) {
    CF_REQUIRE(tensors >= 0 && (tensors == 0 || caches != nullptr), "%s: %lld cache tensors", who,
               static_cast<long long>(tensors));
    for (int64_t i = 0; i < tensors; ++i) CF_REQUIRE(caches[i] != nullptr, "%s: null cache pointer", who);
    CF_REQUIRE(tensors == 0 || (page_bytes > 0 && page_bytes < (int64_t{1} << 40)), "%s: pages of %lld bytes", who,
               static_cast<long long>(page_bytes));
    return CF_OK;
}

cf_status check_tables(const char* who, const void* counts, const void* tables, const void* context,
                       const TableArgs& a) {
    CF_REQUIRE(counts != nullptr && tables != nullptr && context != nullptr, "%s: null pointer", who);
    CF_REQUIRE(a.pages > 0 && a.pages <= kMostInts && a.block > 0 && a.block <= kMostInts && a.sequences > 0 &&
                   a.sequences <= kMostInts && a.width > 0 && a.width <= kMostInts,
               "%s: %lld pages of %lld tokens, tables [%lld, %lld]", who, static_cast<long long>(a.pages),
               static_cast<long long>(a.block), static_cast<long long>(a.sequences), static_cast<long long>(a.width));
    return CF_OK;
}

TableArgs table_args(int32_t* counts, uint32_t* tables, int32_t* context, int64_t pages, int64_t block,
                     int64_t sequences, int64_t width) {
    // Lengths are int32, so a row's reach is cut there.
    const int64_t capacity = block > 0 && width > 0x7FFFFFFF / block ? 0x7FFFFFFF : width * block;
    return TableArgs{counts, tables, context, pages, block, sequences, width, capacity};
}

/// Runs `body` with up to kTensors tensors at a time.
template <typename Body>
void by_tensors(void* const* caches, int64_t tensors, Body body) {
    for (int64_t first = 0; first < tensors || first == 0; first += kTensors) {
        Tensors t{};
        const int64_t n = tensors - first < kTensors ? tensors - first : kTensors;
        for (int64_t i = 0; i < n; ++i) t.p[i] = static_cast<uint8_t*>(caches[first + i]);
        body(t, static_cast<int>(n), first == 0);
    }
}

/// Whether a launch takes the workgroups of one entry: every chunk of its page in
/// every tensor, and one for its tables.
bool one_entry_fits(int64_t tensors, int64_t chunks) {
    return (tensors < kTensors ? tensors : kTensors) * chunks + 1 <= kMaxWorkgroups;
}

/// Runs `body` with entries [first, first + n) of a list of `count`, each of
/// which takes `each` workgroups, in launches of no more than there may be.
template <typename Body>
void by_entries(int64_t count, int64_t each, Body body) {
    const int64_t most = kMaxWorkgroups / each;
    for (int64_t first = 0; first < count; first += most) {
        body(first, count - first < most ? count - first : most);
    }
}

}  // namespace
}  // namespace cf

extern "C" {

size_t cf_cache_workspace_bytes(int64_t num_pages, int64_t num_sequences, int64_t count) {
    if (num_pages <= 0 || num_pages > cf::kMostInts || num_sequences < 0 || num_sequences > cf::kMostInts ||
        count < 0 || count > cf::kMostInts) {
        return 0;
    }
    // A list's claims (pages or rows), ranks, pages and status; a compaction's
    // four lists and its tiles.
    const size_t pages = static_cast<size_t>(num_pages);
    const size_t list = cf::align_up((pages > static_cast<size_t>(num_sequences) ? pages : num_sequences) * 4) +
                        2 * cf::align_up(static_cast<size_t>(count) * 8) + cf::align_up(pages * 4);
    const size_t compact = 4 * cf::align_up(pages * 4) + cf::align_up((pages / cf::kTilePages + 2) * 4) + 256;
    return list > compact ? list : compact;
}

cf_status cf_cache_copy(void* const* caches, int64_t num_caches, int64_t page_bytes, int64_t num_pages,
                        const int32_t* src, const int32_t* dst, int64_t count, int32_t* status, void* workspace,
                        size_t workspace_bytes, void* stream) {
    CF_ENTRY();
    const char* who = "cf_cache_copy";
    if (count <= 0) return CF_OK;
    const cf_status st = cf::check_caches(who, caches, num_caches, page_bytes);
    if (st != CF_OK) return st;
    CF_REQUIRE(src != nullptr && dst != nullptr && status != nullptr, "%s: null pointer", who);
    CF_REQUIRE(num_pages > 0 && num_pages <= cf::kMostInts && count <= cf::kMostInts, "%s: %lld pairs of %lld pages",
               who, static_cast<long long>(count), static_cast<long long>(num_pages));
    const size_t needed = cf_cache_workspace_bytes(num_pages, 0, count);
    CF_REQUIRE(workspace != nullptr && workspace_bytes >= needed && cf::host_aligned(workspace, 16),
               "%s: needs %zu bytes of 16-byte aligned workspace", who, needed);
    const int64_t chunks = cf::ceil_div<int64_t>(page_bytes, cf::kChunkBytes);
    CF_REQUIRE(cf::one_entry_fits(num_caches, chunks), "%s: pages of %lld bytes", who,
               static_cast<long long>(page_bytes));
    auto s = static_cast<hipStream_t>(stream);
    const bool small = num_pages <= cf::kSmallRows;
    cf::launch(small ? cf::copy_plan_kernel<true> : cf::copy_plan_kernel<false>, dim3(1), dim3(cf::kPlanThreads), 0, s, src, dst, count, num_pages,
               static_cast<int*>(workspace), status);
    if (num_caches > 0) {
        const int unit = cf::unit_of(caches, num_caches, page_bytes, page_bytes);
        cf::by_tensors(caches, num_caches, [&](const cf::Tensors& t, int n, bool) {
            auto* kernel = unit == 16 ? cf::copy_pages_kernel<16>
                           : unit == 4 ? cf::copy_pages_kernel<4> : cf::copy_pages_kernel<1>;
            cf::by_entries(count, n * chunks, [&](int64_t at, int64_t pairs) {
                cf::launch(kernel, dim3(static_cast<unsigned>(pairs * n * chunks)), dim3(cf::kCopyThreads), 0, s, t, n,
                           page_bytes, chunks, src + at, dst + at, static_cast<const int*>(status + at));
            });
        });
    }
    return cf::check_launch("launching the page copies", s);
}

cf_status cf_cache_fork(void* const* caches, int64_t num_caches, int64_t page_bytes, int32_t* ref_counts,
                        uint32_t* block_tables, int32_t* context_lens, int64_t num_pages, int64_t block_size,
                        int64_t num_sequences, int64_t max_blocks_per_sequence, const int32_t* parents,
                        const int32_t* children, int64_t count, int32_t* status, void* workspace,
                        size_t workspace_bytes, void* stream) {
    CF_ENTRY();
    const char* who = "cf_cache_fork";
    if (count <= 0) return CF_OK;
    cf_status st = cf::check_caches(who, caches, num_caches, page_bytes);
    if (st != CF_OK) return st;
    const cf::TableArgs a = cf::table_args(ref_counts, block_tables, context_lens, num_pages, block_size,
                                           num_sequences, max_blocks_per_sequence);
    st = cf::check_tables(who, ref_counts, block_tables, context_lens, a);
    if (st != CF_OK) return st;
    CF_REQUIRE(parents != nullptr && children != nullptr && status != nullptr, "%s: null pointer", who);
    CF_REQUIRE(num_caches == 0 || page_bytes % block_size == 0, "%s: pages of %lld bytes do not hold %lld tokens", who,
               static_cast<long long>(page_bytes), static_cast<long long>(block_size));
    CF_REQUIRE(count <= cf::kMostInts, "%s: %lld pairs", who, static_cast<long long>(count));
    const size_t needed = cf_cache_workspace_bytes(num_pages, num_sequences, count);
    CF_REQUIRE(workspace != nullptr && workspace_bytes >= needed && cf::host_aligned(workspace, 16),
               "%s: needs %zu bytes of 16-byte aligned workspace", who, needed);
    const int64_t chunks = num_caches > 0 ? cf::ceil_div<int64_t>(page_bytes, cf::kChunkBytes) : 1;
    CF_REQUIRE(cf::one_entry_fits(num_caches, chunks), "%s: pages of %lld bytes", who,
               static_cast<long long>(page_bytes));
    auto* claims = static_cast<int*>(workspace);
    const int64_t rows = num_pages > num_sequences ? num_pages : num_sequences;
    auto* fresh = reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + cf::align_up(static_cast<size_t>(rows) * 4));
    auto* free_list = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(fresh) + cf::align_up(static_cast<size_t>(count) * 8));
    auto s = static_cast<hipStream_t>(stream);
    const bool small = count <= cf::kPlanThreads && num_sequences <= cf::kSmallRows;
    cf::launch(small ? cf::fork_plan_kernel<true> : cf::fork_plan_kernel<false>, dim3(1), dim3(cf::kPlanThreads), 0, s, a, parents, children, count, claims, fresh,
               free_list, status);
    const int unit = num_caches > 0 ? cf::unit_of(caches, num_caches, page_bytes, page_bytes / block_size) : 16;
    cf::by_tensors(caches, num_caches, [&](const cf::Tensors& t, int n, bool first) {
        auto* kernel = unit == 16 ? cf::fork_move_kernel<16>
                       : unit == 4 ? cf::fork_move_kernel<4> : cf::fork_move_kernel<1>;
        const int64_t pieces = n * chunks + (first ? 1 : 0);
        cf::by_entries(count, pieces, [&](int64_t at, int64_t pairs) {
            cf::launch(kernel, dim3(static_cast<unsigned>(pairs * pieces)), dim3(cf::kCopyThreads), 0, s, a, t, n,
                       page_bytes, chunks, first, parents + at, children + at, static_cast<const int*>(fresh + at),
                       static_cast<const int*>(status + at));
        });
    });
    return cf::check_launch("launching the fork", s);
}

cf_status cf_cache_extend(int32_t* ref_counts, uint32_t* block_tables, int32_t* context_lens, int64_t num_pages,
                          int64_t block_size, int64_t num_sequences, int64_t max_blocks_per_sequence,
                          const int32_t* sequences, int64_t count, int64_t tokens, int64_t* slots, void* workspace,
                          size_t workspace_bytes, void* stream) {
    CF_ENTRY();
    const char* who = "cf_cache_extend";
    if (count <= 0) return CF_OK;
    const cf::TableArgs a = cf::table_args(ref_counts, block_tables, context_lens, num_pages, block_size,
                                           num_sequences, max_blocks_per_sequence);
    const cf_status st = cf::check_tables(who, ref_counts, block_tables, context_lens, a);
    if (st != CF_OK) return st;
    CF_REQUIRE(sequences != nullptr && slots != nullptr, "%s: null pointer", who);
    CF_REQUIRE(tokens >= 1 && count <= cf::kMostInts && tokens <= cf::kMostInts / count, "%s: %lld sequences by %lld tokens",
               who, static_cast<long long>(count), static_cast<long long>(tokens));
    const size_t needed = cf_cache_workspace_bytes(num_pages, num_sequences, count);
    CF_REQUIRE(workspace != nullptr && workspace_bytes >= needed && cf::host_aligned(workspace, 16),
               "%s: needs %zu bytes of 16-byte aligned workspace", who, needed);
    auto* claims = static_cast<int*>(workspace);
    const int64_t rows = num_pages > num_sequences ? num_pages : num_sequences;
    uint8_t* at = static_cast<uint8_t*>(workspace) + cf::align_up(static_cast<size_t>(rows) * 4);
    auto* ranks = reinterpret_cast<int64_t*>(at);
    at += cf::align_up(static_cast<size_t>(count) * 8);
    auto* status = reinterpret_cast<int*>(at);
    at += cf::align_up(static_cast<size_t>(count) * 8);
    auto* free_list = reinterpret_cast<int*>(at);
    auto s = static_cast<hipStream_t>(stream);
    const bool small = num_sequences <= cf::kSmallRows &&
                       count * cf::ceil_div<int64_t>(tokens, block_size) <= cf::kPlanThreads;  // pages wanted
    cf::launch(small ? cf::extend_kernel<true> : cf::extend_kernel<false>, dim3(1), dim3(cf::kPlanThreads), 0, s, a, sequences, count, tokens, claims, ranks,
               free_list, status, slots);
    if (tokens > 1) {
        cf::launch(cf::extend_slots_kernel,
                   dim3(static_cast<unsigned>(cf::ceil_div<int64_t>(count * tokens, cf::kCopyThreads))),
                   dim3(cf::kCopyThreads), 0, s, a, sequences, count, tokens, static_cast<const int*>(status), slots);
    }
    return cf::check_launch("launching the extension", s);
}

cf_status cf_cache_release(int32_t* ref_counts, uint32_t* block_tables, int32_t* context_lens, int64_t num_pages,
                           int64_t block_size, int64_t num_sequences, int64_t max_blocks_per_sequence,
                           const int32_t* sequences, int64_t count, void* stream) {
    CF_ENTRY();
    const char* who = "cf_cache_release";
    if (count <= 0) return CF_OK;
    const cf::TableArgs a = cf::table_args(ref_counts, block_tables, context_lens, num_pages, block_size,
                                           num_sequences, max_blocks_per_sequence);
    const cf_status st = cf::check_tables(who, ref_counts, block_tables, context_lens, a);
    if (st != CF_OK) return st;
    CF_REQUIRE(sequences != nullptr, "%s: null pointer", who);
    CF_REQUIRE(count <= cf::kMostInts, "%s: %lld sequences", who, static_cast<long long>(count));
    auto s = static_cast<hipStream_t>(stream);
    cf::by_entries(count, 1, [&](int64_t at, int64_t rows) {
        cf::launch(cf::release_kernel, dim3(static_cast<unsigned>(rows)), dim3(cf::kCopyThreads), 0, s, a,
                   sequences + at);
    });
    return cf::check_launch("launching the release", s);
}

cf_status cf_cache_compact(void* const* caches, int64_t num_caches, int64_t page_bytes, const int32_t* ref_counts,
                           const uint32_t* block_tables, const int32_t* context_lens, int64_t num_pages,
                           int64_t block_size, int64_t num_sequences, int64_t max_blocks_per_sequence,
                           int32_t* new_ref_counts, uint32_t* new_block_tables, int32_t* live_pages, void* workspace,
                           size_t workspace_bytes, void* stream) {
    CF_ENTRY();
    const char* who = "cf_cache_compact";
    cf_status st = cf::check_caches(who, caches, num_caches, page_bytes);
    if (st != CF_OK) return st;
    CF_REQUIRE(ref_counts != nullptr && new_ref_counts != nullptr && live_pages != nullptr, "%s: null pointer", who);
    const bool rows = num_sequences > 0 && max_blocks_per_sequence > 0;
    CF_REQUIRE(!rows || (block_tables != nullptr && new_block_tables != nullptr && context_lens != nullptr),
               "%s: null pointer", who);
    CF_REQUIRE(num_pages > 0 && num_pages <= cf::kMostInts && block_size > 0 && block_size <= cf::kMostInts &&
                   num_sequences >= 0 && num_sequences <= cf::kMostInts && max_blocks_per_sequence >= 0 &&
                   max_blocks_per_sequence <= cf::kMostInts,
               "%s: %lld pages of %lld tokens, tables [%lld, %lld]", who, static_cast<long long>(num_pages),
               static_cast<long long>(block_size), static_cast<long long>(num_sequences),
               static_cast<long long>(max_blocks_per_sequence));
    const size_t needed = cf_cache_workspace_bytes(num_pages, num_sequences, 0);
    CF_REQUIRE(workspace != nullptr && workspace_bytes >= needed && cf::host_aligned(workspace, 16),
               "%s: needs %zu bytes of 16-byte aligned workspace", who, needed);
    cf::CompactArgs a{};
    a.counts = ref_counts;
    a.tables = block_tables;
    a.context = context_lens;
    a.new_counts = new_ref_counts;
    a.new_tables = new_block_tables;
    a.live = live_pages;
    a.pages = num_pages;
    a.block = block_size;
    a.sequences = rows ? num_sequences : 0;
    a.width = rows ? max_blocks_per_sequence : 1;
    a.tiles = cf::ceil_div<int64_t>(num_pages, cf::kTilePages);
    uint8_t* at = static_cast<uint8_t*>(workspace);
    const size_t list = cf::align_up(static_cast<size_t>(num_pages) * 4);
    a.holes = reinterpret_cast<int*>(at);
    a.movers = reinterpret_cast<int*>(at + list);
    a.mover_count = reinterpret_cast<int*>(at + 2 * list);
    a.rank = reinterpret_cast<int*>(at + 3 * list);
    a.tile_live = reinterpret_cast<int*>(at + 4 * list);
    a.moves = a.tile_live + a.tiles;
    auto s = static_cast<hipStream_t>(stream);
    const dim3 tiles(static_cast<unsigned>(a.tiles));
    cf::launch(cf::compact_count_kernel, tiles, dim3(cf::kCopyThreads), 0, s, a);
    cf::launch(cf::compact_list_kernel, tiles, dim3(cf::kCopyThreads), 0, s, a);
    const int64_t chunks = num_caches > 0 ? cf::ceil_div<int64_t>(page_bytes, cf::kChunkBytes) : 1;
    const int unit = num_caches > 0 ? cf::unit_of(caches, num_caches, page_bytes, page_bytes) : 16;
    cf::by_tensors(caches, num_caches, [&](const cf::Tensors& t, int n, bool first) {
        auto* kernel = unit == 16 ? cf::compact_move_kernel<16>
                       : unit == 4 ? cf::compact_move_kernel<4> : cf::compact_move_kernel<1>;
        cf::launch(kernel, dim3(static_cast<unsigned>(8 * cf::cu_count())), dim3(cf::kCopyThreads), 0, s, a, t, n,
                   page_bytes, chunks, first);
    });
    return cf::check_launch("launching the compaction", s);
}

}  // extern "C"
