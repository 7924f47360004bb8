// Storing keys and values into a paged cache, as they are or in 8 bits with a
// scale per row, and reading them back.
//
// A row is one token's head_dim values of one KV head, of K or of V; places in
// the cache come as slots. Both directions are bound by HBM: a bf16 row of 128
// is read once (256 bytes) and written once (128 + 4).
//   * A row belongs to a group of 8 to 64 lanes that holds it in registers,
//     16 bytes of the given type a lane and step, so the largest magnitude is a
//     reduction over the group and the row is never read twice.
//   * Of tokens with one slot the last one stays, as if they were written one
//     after the other. A workgroup owns neighbouring tokens; it puts their slots
//     into a hash table in LDS and looks up those of all later tokens in it,
//     while its first rows are on their way.
// 8192 tokens of 8 heads of 128, bf16 to e4m3: 17.7 us written (2.9 TB/s, behind
// that search), 11.3 us read back (4.5 TB/s); to bf16 15.2 and 14.4 us.
// 64 tokens, 4.4 and 2.8 us, are a launch and its chain of loads.
#include "cf_codes.hpp"
#include "cf_common.hpp"
#include "cf_ranges.hpp"

namespace cf {
namespace {

constexpr int kThreads = 256;
constexpr int kManyThreads = 1024;
constexpr int kMaxOwn = 1024;  // tokens per workgroup at most: 52 KiB of LDS

struct StoreArgs {
    const void* x[2];  // keys, values (read: the results)
    int64_t token_stride[2];
    int64_t head_stride[2];
    void* cache[2];
    float* scales[2];
    const int64_t* slots;
    int64_t num_slots;
    int64_t tokens;
    int kv_heads;
    int dim;
    int own;    // tokens per workgroup
    int table;  // entries of the hash table, a power of two, 2 own at least
    int bits;   // of the filter before it, a power of two
};

/// The largest over groups of kLanes lanes (8 to 64) of magnitudes' bits.
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    v = group_reduce_u32<(kLanes < 16 ? kLanes : 16), MaxU32>(v);
#pragma unroll
    for (int d = 16; d < kLanes; d <<= 1) {
        const uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d));
        v = o > v ? o : v;
    }
    return v;
}

__device__ __forceinline__ uint32_t abs_of(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

/// Which of the workgroup's tokens are written: those whose slot lies in the
/// cache and is no later token's. The own slots are set in a hash table, and in a
/// filter of one bit per slot modulo its size, which nearly all slots of later
/// tokens miss (8192 tokens: the search took 7 of 21 us with the table alone).
struct Own {
    int32_t* slot;     // [own] -1: left out
    int32_t* key;      // [table] slot or -1
    int32_t* last;     // [table] the last own token of that slot; `own` behind a later workgroup's
    uint32_t* filter;  // [bits / 32]
};

__device__ __forceinline__ uint32_t place_of(uint32_t slot, int table) {
    return (slot * 2654435761u >> 8) & static_cast<uint32_t>(table - 1);
}

__device__ void find_kept(const StoreArgs& a, const Own& own, int64_t first, int count) {
    const int tid = static_cast<int>(threadIdx.x);
    const int threads = static_cast<int>(blockDim.x);
    if (a.own == 1) {  // one token: its slot against all later ones
        const int64_t s = a.slots[first];
        bool again = false;
        for (int64_t j = first + 1 + tid; j < a.tokens; j += threads) again = again || a.slots[j] == s;
        if (tid == 0) own.slot[0] = s >= 0 && s < a.num_slots ? static_cast<int>(s) : -1;
        __syncthreads();
        if (again) own.slot[0] = -1;
        __syncthreads();
        return;
    }
    for (int i = tid; i < a.table; i += threads) {
        own.key[i] = -1;
        own.last[i] = -1;
    }
    for (int i = tid; i < a.bits / 32; i += threads) own.filter[i] = 0;
    __syncthreads();
    const uint32_t mask = static_cast<uint32_t>(a.bits - 1);
    for (int i = tid; i < count; i += threads) {
        const int64_t s = a.slots[first + i];
        const int slot = s >= 0 && s < a.num_slots ? static_cast<int>(s) : -1;
        own.slot[i] = slot;
        if (slot < 0) continue;
        uint32_t at = place_of(static_cast<uint32_t>(slot), a.table);
        for (;;) {  // half of the table at least stays empty
            const int held = atomicCAS(&own.key[at], -1, slot);
            if (held == -1 || held == slot) break;
            at = (at + 1) & static_cast<uint32_t>(a.table - 1);
        }
        atomicMax(&own.last[at], i);
        atomicOr(&own.filter[(static_cast<uint32_t>(slot) & mask) >> 5], 1u << (slot & 31));
    }
    __syncthreads();
    constexpr int kBatch = 8;  // loads of a thread in flight
    for (int64_t j0 = first + count + tid; j0 < a.tokens; j0 += kBatch * threads) {
        int64_t later[kBatch];
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
            const int64_t j = j0 + n * threads;
            later[n] = j < a.tokens ? a.slots[j] : -1;
        }
        uint32_t hits = 0;
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
            const uint32_t low = static_cast<uint32_t>(later[n]);
            hits |= ((own.filter[(low & mask) >> 5] >> (low & 31)) & 1u) << n;
        }
        if (hits == 0) continue;
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
            if ((hits >> n & 1) == 0 || later[n] < 0 || later[n] >= a.num_slots) continue;
            const int slot = static_cast<int>(later[n]);
            uint32_t at = place_of(static_cast<uint32_t>(slot), a.table);
            for (;;) {
                const int held = own.key[at];
                if (held == slot) own.last[at] = a.own;
                if (held == slot || held == -1) break;
                at = (at + 1) & static_cast<uint32_t>(a.table - 1);
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < count; i += threads) {
        const int slot = own.slot[i];
        if (slot < 0) continue;
        uint32_t at = place_of(static_cast<uint32_t>(slot), a.table);
        while (own.key[at] != slot) at = (at + 1) & static_cast<uint32_t>(a.table - 1);
        if (own.last[at] != i) own.slot[i] = -1;
    }
    __syncthreads();
}

/// The rows of K or of V that a group of lanes takes in turn: (token, head) pairs
/// of the workgroup, `step` apart, without a division or product per row.
struct Rows {
    int token;
    int head;
    int step_tokens, step_heads, heads;

    __device__ __forceinline__ Rows(int first, int step, int kv_heads)
        : token(first / kv_heads), head(first - token * kv_heads), step_tokens(step / kv_heads),
          step_heads(step - step_tokens * kv_heads), heads(kv_heads) {}
    __device__ __forceinline__ void next() {
        token += step_tokens;
        head += step_heads;
        const bool wraps = head >= heads;
        token += wraps ? 1 : 0;
        head -= wraps ? heads : 0;
    }
};

/// kVecs 16-byte vectors per lane of a group of kLanes; kVecs 0: rows of any
/// length and alignment, a wave each, read twice. The first half of a workgroup
/// takes keys, the second values.
template <typename T, cf_cache_format kFormat, int kLanes, int kVecs>
__global__ __launch_bounds__(kManyThreads) void cache_write_kernel(StoreArgs a) {
    extern __shared__ int32_t lds[];
    const Own own{lds, lds + a.own, lds + a.own + a.table, reinterpret_cast<uint32_t*>(lds) + a.own + 2 * a.table};
    const int half = static_cast<int>(blockDim.x) / 2;
    const int which = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >= half ? 1 : 0);
    const int tid = static_cast<int>(threadIdx.x) - which * half;  // of the half
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.own;
    const int count = static_cast<int>(a.tokens - first < a.own ? a.tokens - first : a.own);
    const int64_t token_stride = which ? a.token_stride[1] : a.token_stride[0];
    const int64_t head_stride = which ? a.head_stride[1] : a.head_stride[0];
    const T* given = static_cast<const T*>(which ? a.x[1] : a.x[0]) + first * token_stride;
    void* const cache = which ? a.cache[1] : a.cache[0];
    float* const scales = which ? a.scales[1] : a.scales[0];
    const int groups = half / kLanes;
    const int part = tid % kLanes;
    Rows row(tid / kLanes, groups, a.kv_heads);
    if constexpr (kVecs > 0) {
        constexpr int kPer = Storage<T>::kPerVec;
        constexpr int kAhead = kVecs == 1 ? 4 : 1;  // rows per group of lanes on their way
        struct Given {
            int token;
            int head;
            uint4 raw[kVecs];
        };
        Given now[kAhead];
        auto load = [&](Given& g) {
            g.token = row.token;
            g.head = row.head;
            const T* x = given + row.token * token_stride + row.head * head_stride;
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                const int d = (v * kLanes + part) * kPer;
                g.raw[v] = make_uint4(0, 0, 0, 0);
                if (row.token < count && d < a.dim) g.raw[v] = load_stream16(x + d);
            }
            row.next();
        };
#pragma unroll
        for (int n = 0; n < kAhead; ++n) load(now[n]);
        find_kept(a, own, first, count);
        while (now[0].token < count) {
#pragma unroll
            for (int n = 0; n < kAhead; ++n) {
                // A row is stored while those behind it, the next round's among them, are
                // on their way.
                const Given g = now[n];
                load(now[n]);
                const int slot = g.token < count ? own.slot[g.token] : -1;
                const int64_t at = static_cast<int64_t>(slot) * a.kv_heads + g.head;
                if constexpr (kFormat == CF_CACHE_PLAIN) {
                    T* to = static_cast<T*>(cache) + at * a.dim;
#pragma unroll
                    for (int v = 0; v < kVecs; ++v) {
                        const int d = (v * kLanes + part) * kPer;
                        if (slot >= 0 && d < a.dim) *reinterpret_cast<uint4*>(to + d) = g.raw[v];
                    }
                } else {
                    float f[kVecs][kPer];
                    uint32_t top = 0;
#pragma unroll
                    for (int v = 0; v < kVecs; ++v) {
                        top = MaxU32::apply(top, largest16<T>(g.raw[v]));
                        unpack16<T>(g.raw[v], f[v]);
                    }
                    const RowScale s = row_scale<kFormat>(lanes_max<kLanes>(top));
                    const bool ordinary = ordinary_rows(s);
                    uint8_t* to = static_cast<uint8_t*>(cache) + at * a.dim;
#pragma unroll
                    for (int v = 0; v < kVecs; ++v) {
                        const int d = (v * kLanes + part) * kPer;
                        uint32_t w[kPer / 4];
#pragma unroll
                        for (int e = 0; e < kPer / 4; ++e) {
                            w[e] = ordinary ? pack4_codes<kFormat, false>(f[v] + 4 * e, s)
                                            : pack4_codes<kFormat, true>(f[v] + 4 * e, s);
                        }
                        if (slot >= 0 && d < a.dim) {
                            if constexpr (kPer == 8) {
                                *reinterpret_cast<uint2*>(to + d) = make_uint2(w[0], w[1]);
                            } else {
                                *reinterpret_cast<uint32_t*>(to + d) = w[0];
                            }
                        }
                    }
                    if (slot >= 0 && part == 0) scales[at] = s.s;
                }
            }
        }
    } else {
        find_kept(a, own, first, count);
        for (; row.token < count; row.next()) {
            const int slot = own.slot[row.token];
            if (slot < 0) continue;
            const T* x = given + row.token * token_stride + row.head * head_stride;
            const int64_t at = static_cast<int64_t>(slot) * a.kv_heads + row.head;
            if constexpr (kFormat == CF_CACHE_PLAIN) {
                for (int d = part; d < a.dim; d += kLanes) static_cast<T*>(cache)[at * a.dim + d] = x[d];
            } else {
                uint32_t top = 0;
                for (int d = part; d < a.dim; d += kLanes) top = MaxU32::apply(top, abs_of(Storage<T>::load(x + d)));
                const RowScale s = row_scale<kFormat>(lanes_max<kLanes>(top));
                uint8_t* to = static_cast<uint8_t*>(cache) + at * a.dim;
                for (int d = part; d < a.dim; d += kLanes) {
                    const float f[4] = {Storage<T>::load(x + d), 0.0f, 0.0f, 0.0f};
                    to[d] = static_cast<uint8_t>(pack4_codes<kFormat, true>(f, s));
                }
                if (part == 0) scales[at] = s.s;
            }
        }
    }
}

template <typename T, cf_cache_format kFormat, int kLanes, int kVecs>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(StoreArgs a) {
    constexpr int kPer = Storage<T>::kPerVec;
    constexpr int kGroups = kThreads / kLanes;
    const int tid = static_cast<int>(threadIdx.x);
    const int part = tid % kLanes;
    const int per_token = 2 * a.kv_heads;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.own;
    const int count = static_cast<int>(a.tokens - first < a.own ? a.tokens - first : a.own);
    const int rows = count * per_token;
    for (int r = tid / kLanes; r < rows; r += kGroups) {
        const int64_t token = first + r / per_token;
        const int64_t slot = a.slots[token];
        const bool there = slot >= 0 && slot < a.num_slots;
        const int which = r % per_token / a.kv_heads;
        const int head = r % a.kv_heads;
        const int64_t row = (there ? slot : 0) * a.kv_heads + head;
        T* x = static_cast<T*>(const_cast<void*>(which ? a.x[1] : a.x[0])) +
               (token * a.kv_heads + head) * a.dim;
        const void* cache = which ? a.cache[1] : a.cache[0];
        float s = 1.0f;
        if constexpr (kFormat != CF_CACHE_PLAIN) s = there ? (which ? a.scales[1] : a.scales[0])[row] : 0.0f;
        if constexpr (kVecs > 0) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                const int d = (v * kLanes + part) * kPer;
                if (d >= a.dim) continue;
                uint4 out = make_uint4(0, 0, 0, 0);
                if constexpr (kFormat == CF_CACHE_PLAIN) {
                    if (there) out = load_stream16(static_cast<const T*>(cache) + row * a.dim + d);
                } else {
                    const uint8_t* from = static_cast<const uint8_t*>(cache) + row * a.dim + d;
                    float f[kPer];
                    if constexpr (kPer == 8) {
                        const uint2 w = there ? load_stream8(from) : make_uint2(0, 0);
                        unpack4_codes<kFormat>(w.x, f);
                        unpack4_codes<kFormat>(w.y, f + 4);
                    } else {
                        unpack4_codes<kFormat>(there ? load_stream4(from) : 0u, f);
                    }
#pragma unroll
                    for (int e = 0; e < kPer; ++e) f[e] *= s;
                    out = pack16<T>(f);
                }
                store_stream16(x + d, out);
            }
        } else {
            for (int d = part; d < a.dim; d += kLanes) {
                if constexpr (kFormat == CF_CACHE_PLAIN) {
                    x[d] = there ? static_cast<const T*>(cache)[row * a.dim + d] : T{};
                } else {
                    float f[4];
                    unpack4_codes<kFormat>(there ? static_cast<const uint8_t*>(cache)[row * a.dim + d] : 0u, f);
                    Storage<T>::store(x + d, f[0] * s);
                }
            }
        }
    }
}

// ---- host -----------------------------------------------------------------------

/// Groups of lanes: vectors of 16 bytes of the given type a row holds, over at
/// most 64 lanes and 4 steps (rows of 4 KiB); 0: the kernel for any row.
template <template <typename, cf_cache_format, int, int> class Kernel, typename T, cf_cache_format kFormat>
void launch_rows(const StoreArgs& a, bool vectors, dim3 grid, dim3 block, uint32_t lds_bytes, hipStream_t stream) {
    const int vecs = a.dim / Storage<T>::kPerVec;
    if (!vectors || vecs > 256) {
        launch(Kernel<T, kFormat, 64, 0>::get(), grid, block, lds_bytes, stream, a);
    } else if (vecs <= 8) {
        launch(Kernel<T, kFormat, 8, 1>::get(), grid, block, lds_bytes, stream, a);
    } else if (vecs <= 16) {
        launch(Kernel<T, kFormat, 16, 1>::get(), grid, block, lds_bytes, stream, a);
    } else if (vecs <= 32) {
        launch(Kernel<T, kFormat, 32, 1>::get(), grid, block, lds_bytes, stream, a);
    } else if (vecs <= 64) {
        launch(Kernel<T, kFormat, 64, 1>::get(), grid, block, lds_bytes, stream, a);
    } else {
        launch(Kernel<T, kFormat, 64, 4>::get(), grid, block, lds_bytes, stream, a);
    }
}

template <typename T, cf_cache_format kFormat, int kLanes, int kVecs>
struct Write {
    static constexpr auto get() { return &cache_write_kernel<T, kFormat, kLanes, kVecs>; }
};
template <typename T, cf_cache_format kFormat, int kLanes, int kVecs>
struct Read {
    static constexpr auto get() { return &cache_read_kernel<T, kFormat, kLanes, kVecs>; }
};

template <template <typename, cf_cache_format, int, int> class Kernel, typename T>
void launch_format(cf_cache_format format, const StoreArgs& a, bool vectors, dim3 grid, dim3 block,
                   uint32_t lds_bytes, hipStream_t stream) {
    switch (format) {
        case CF_CACHE_PLAIN: launch_rows<Kernel, T, CF_CACHE_PLAIN>(a, vectors, grid, block, lds_bytes, stream); break;
        case CF_CACHE_INT8: launch_rows<Kernel, T, CF_CACHE_INT8>(a, vectors, grid, block, lds_bytes, stream); break;
        case CF_CACHE_E4M3: launch_rows<Kernel, T, CF_CACHE_E4M3>(a, vectors, grid, block, lds_bytes, stream); break;
    }
}

template <template <typename, cf_cache_format, int, int> class Kernel>
void launch_all(cf_dtype dtype, cf_cache_format format, const StoreArgs& a, bool vectors, dim3 grid, dim3 block,
                uint32_t lds_bytes, hipStream_t stream) {
    switch (dtype) {
        case CF_F32: launch_format<Kernel, float>(format, a, vectors, grid, block, lds_bytes, stream); break;
        case CF_F16: launch_format<Kernel, f16_t>(format, a, vectors, grid, block, lds_bytes, stream); break;
        case CF_BF16: launch_format<Kernel, bf16_t>(format, a, vectors, grid, block, lds_bytes, stream); break;
    }
}

/// Checks that both directions share.
cf_status check_store(const char* who, cf_dtype dtype, cf_cache_format format, int64_t tokens, int64_t kv_heads,
                      int64_t head_dim, int64_t num_slots, const void* const (&pointers)[5], const float* k_scales,
                      const float* v_scales) {
    CF_REQUIRE(valid_dtype(dtype), "%s: unknown dtype %d", who, static_cast<int>(dtype));
    CF_REQUIRE(valid_format(format), "%s: unknown cache format %d", who, static_cast<int>(format));
    CF_REQUIRE(kv_heads <= (1 << 14) && head_dim <= (1 << 20) && num_slots >= 0 && num_slots <= kMostTokens,
               "%s: %lld KV heads of %lld over %lld slots (at most 2^14, 2^20 and 2^31 - 4096)", who,
               static_cast<long long>(kv_heads), static_cast<long long>(head_dim), static_cast<long long>(num_slots));
    for (const void* p : pointers) CF_REQUIRE(p != nullptr, "%s: null pointer", who);
    CF_REQUIRE(format == CF_CACHE_PLAIN || (k_scales != nullptr && v_scales != nullptr),
               "%s: an 8-bit cache needs scales", who);
    const size_t size = dtype_size(dtype);
    const size_t held = format == CF_CACHE_PLAIN ? size : 1;
    CF_REQUIRE(host_aligned(pointers[0], size) && host_aligned(pointers[1], size) && host_aligned(pointers[2], held) &&
                   host_aligned(pointers[3], held) && host_aligned(pointers[4], 8) && host_aligned(k_scales, 4) &&
                   host_aligned(v_scales, 4),
               "%s: misaligned pointer", who);
    return CF_OK;
}

/// Bytes from `begin` to `end`, of rows a stride of elements apart.
struct Bytes {
    uintptr_t begin, end;

    bool meet(const Bytes& o) const { return begin < end && o.begin < o.end && begin < o.end && o.begin < end; }
};
Bytes bytes_of(const void* p, size_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return Bytes{at, at + bytes};
}
Bytes bytes_of_rows(const void* p, int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride, int64_t dim,
                    size_t size) {
    const int64_t reach[2] = {(tokens - 1) * token_stride, (heads - 1) * head_stride};
    int64_t first = 0, last = dim;
    for (const int64_t r : reach) (r < 0 ? first : last) += r;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return Bytes{at + static_cast<uintptr_t>(first * static_cast<int64_t>(size)),
                 at + static_cast<uintptr_t>(last * static_cast<int64_t>(size))};
}

/// Whole vectors: of the given type, and as many codes of the cache.
bool whole_vectors(const StoreArgs& a, cf_dtype dtype, cf_cache_format format, bool strided) {
    const int64_t per = dtype == CF_F32 ? 4 : 8;
    const size_t held = format == CF_CACHE_PLAIN ? 16 : static_cast<size_t>(per);
    bool good = a.dim % per == 0;
    for (int i = 0; i < 2; ++i) {
        good = good && host_aligned(a.x[i], 16) && host_aligned(a.cache[i], held);
        if (strided) good = good && a.token_stride[i] % per == 0 && a.head_stride[i] % per == 0;
    }
    return good;
}

}  // namespace
}  // namespace cf

extern "C" {

cf_status cf_cache_write(const void* keys, const void* values, cf_dtype dtype, int64_t tokens, int64_t num_kv_heads,
                         int64_t head_dim, int64_t key_token_stride, int64_t key_head_stride,
                         int64_t value_token_stride, int64_t value_head_stride, const int64_t* slots, void* k_cache,
                         void* v_cache, cf_cache_format format, float* k_scales, float* v_scales, int64_t num_slots,
                         void* stream) {
    CF_ENTRY();
    const char* who = "cf_cache_write";
    if (tokens <= 0 || num_kv_heads <= 0 || head_dim <= 0) return CF_OK;
    const cf_status st = cf::check_store(who, dtype, format, tokens, num_kv_heads, head_dim, num_slots,
                                         {keys, values, k_cache, v_cache, slots}, k_scales, v_scales);
    if (st != CF_OK) return st;
    {
        const size_t size = cf::dtype_size(dtype);
        const size_t rows = static_cast<size_t>(num_slots) * static_cast<size_t>(num_kv_heads);
        const size_t cache_bytes = rows * static_cast<size_t>(head_dim) * (format == CF_CACHE_PLAIN ? size : 1);
        const size_t scale_bytes = format == CF_CACHE_PLAIN ? 0 : rows * 4;
        const cf::Bytes written[4] = {cf::bytes_of(k_cache, cache_bytes), cf::bytes_of(v_cache, cache_bytes),
                                      cf::bytes_of(k_scales, scale_bytes), cf::bytes_of(v_scales, scale_bytes)};
        const cf::Bytes given[2] = {
            cf::bytes_of_rows(keys, tokens, key_token_stride, num_kv_heads, key_head_stride, head_dim, size),
            cf::bytes_of_rows(values, tokens, value_token_stride, num_kv_heads, value_head_stride, head_dim, size)};
        const int many = format == CF_CACHE_PLAIN ? 2 : 4;
        for (int i = 0; i < many; ++i) {
            for (int j = 0; j < i; ++j) {
                CF_REQUIRE(!written[i].meet(written[j]), "%s: caches or scales share memory", who);
            }
            for (const cf::Bytes& g : given) {
                CF_REQUIRE(!written[i].meet(g), "%s: keys or values share memory with what is written", who);
            }
        }
    }
    cf::StoreArgs a{};
    a.x[0] = keys;
    a.x[1] = values;
    a.token_stride[0] = key_token_stride;
    a.token_stride[1] = value_token_stride;
    a.head_stride[0] = key_head_stride;
    a.head_stride[1] = value_head_stride;
    a.cache[0] = k_cache;
    a.cache[1] = v_cache;
    a.scales[0] = k_scales;
    a.scales[1] = v_scales;
    a.slots = slots;
    a.num_slots = num_slots;
    a.tokens = tokens;
    a.kv_heads = static_cast<int>(num_kv_heads);
    a.dim = static_cast<int>(head_dim);
    // A workgroup a CU, so that few read the list of later slots.
    const int64_t own = cf::ceil_div<int64_t>(tokens, 256);
    a.own = static_cast<int>(own > cf::kMaxOwn ? cf::kMaxOwn : own);
    a.table = 64;
    while (a.table < 2 * a.own) a.table *= 2;
    const int64_t workgroups = cf::ceil_div<int64_t>(tokens, a.own);
    CF_REQUIRE(workgroups <= cf::kMaxWorkgroups, "%s: %lld tokens are too many", who, static_cast<long long>(tokens));
    a.bits = 32768;
    while (a.bits < 262144 && a.bits < 256 * a.own) a.bits *= 2;
    const uint32_t lds_bytes = static_cast<uint32_t>(a.own + 2 * a.table) * 4 + static_cast<uint32_t>(a.bits) / 8;
    // Large workgroups where each has values for them (bf16 to int8, 8 heads of 128: 1024
    // tokens 8.2 us with 256 threads and 9.6 with 1024, 2048 tokens 10.9 and 10.4, 8192
    // tokens 29 and 19).
    const int threads = int64_t{a.own} * num_kv_heads * head_dim >= 8 * cf::kManyThreads ? cf::kManyThreads : cf::kThreads;
    auto s = static_cast<hipStream_t>(stream);
    cf::launch_all<cf::Write>(dtype, format, a, cf::whole_vectors(a, dtype, format, true),
                              dim3(static_cast<unsigned>(workgroups)), dim3(threads), lds_bytes, s);
    return cf::check_launch("launching the cache write", s);
}

cf_status cf_cache_read(const void* k_cache, const void* v_cache, cf_cache_format format, const float* k_scales,
                        const float* v_scales, int64_t num_slots, const int64_t* slots, int64_t tokens,
                        int64_t num_kv_heads, int64_t head_dim, void* keys, void* values, cf_dtype dtype,
                        void* stream) {
    CF_ENTRY();
    const char* who = "cf_cache_read";
    if (tokens <= 0 || num_kv_heads <= 0 || head_dim <= 0) return CF_OK;
    const cf_status st = cf::check_store(who, dtype, format, tokens, num_kv_heads, head_dim, num_slots,
                                         {keys, values, k_cache, v_cache, slots}, k_scales, v_scales);
    if (st != CF_OK) return st;
    cf::StoreArgs a{};
    a.x[0] = keys;
    a.x[1] = values;
    a.cache[0] = const_cast<void*>(k_cache);
    a.cache[1] = const_cast<void*>(v_cache);
    a.scales[0] = const_cast<float*>(k_scales);
    a.scales[1] = const_cast<float*>(v_scales);
    a.slots = slots;
    a.num_slots = num_slots;
    a.tokens = tokens;
    a.kv_heads = static_cast<int>(num_kv_heads);
    a.dim = static_cast<int>(head_dim);
    int64_t own = cf::ceil_div<int64_t>(tokens, 2048);
    if (own > cf::kMaxOwn) own = cf::kMaxOwn;
    a.own = static_cast<int>(own);
    const int64_t workgroups = cf::ceil_div<int64_t>(tokens, own);
    CF_REQUIRE(workgroups <= cf::kMaxWorkgroups, "%s: %lld tokens are too many", who, static_cast<long long>(tokens));
    auto s = static_cast<hipStream_t>(stream);
    cf::launch_all<cf::Read>(dtype, format, a, cf::whole_vectors(a, dtype, format, false),
                             dim3(static_cast<unsigned>(workgroups)), dim3(cf::kThreads), 0, s);
    return cf::check_launch("launching the cache read", s);
}

}  // extern "C"
