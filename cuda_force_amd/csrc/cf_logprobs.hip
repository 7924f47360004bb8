// Log probabilities of given tokens, entropy and the likeliest tokens of rows
// of logits, and the gradient of the first two.
//
// With x = scale * logits[row] (fp32) and L = ln sum_j e^(x_j):
//   logprob(t) = x_t - L;   p_j = e^(x_j - L);   entropy = -sum_j p_j ln p_j;
//   top: the largest x_j - L, equal logits in the order of their ids.
// Backward, with g the gradients of the given tokens' log probabilities,
// G = sum g, h the entropy's gradient and H the entropy:
//   d logits_j = scale * (sum_{i: token_i = j} g_i - p_j (G + h (ln p_j + H))).
//
// Bound by HBM: the forward reads each logit once (no probabilities are
// written), the backward reads it once more and writes its gradient.
//   * A row is cut into chunks of whole 16-byte vectors, one workgroup each:
//     few rows still fill the GPU, and a thread's share stays short. Every
//     thread keeps a running maximum, sum and (for the entropy) weighted sum
//     over its vectors; threads, then chunks are joined with the rescaling
//     rule. A row of one chunk is finished by its own workgroup, others by a
//     second kernel from the chunks' partial results.
//   * Sums are in base 2 on e = exp2(fma(x, c, -m c)), c = scale log2(e): one
//     fma and one v_exp_f32 a logit. A thread's m c is rounded, and the rounding
//     taken out when threads are joined (by an exact fma), so a common offset of
//     the logits costs no precision. Chunks whose maximum is so large that m c could
//     overflow (rows of the type's lowest value), or that hold a NaN, are
//     summed again by a loop that subtracts before it multiplies.
//   * The likeliest tokens need no second pass over the row. Every thread
//     knows its own best logit, and so does every team of four threads. A logit
//     can be among the row's top k only if its team's best is among the k best
//     teams' (otherwise k larger ones exist), so only those k teams' vectors
//     (k / 64 of the chunk) are read again, from L2, and filtered by the k-th
//     best team's logit. Teams of four against single threads: 64 keys to rank
//     and not 256 (5 of 131072, 600 rows in fp16 cut in four: 41 -> 38 us, with the
//     batches below); a row of equal logits leaves more keys, which are sieved twice.
//   * Measured: 4096 rows of 32000 bf16 logits (262 MB) with entropy 52 us, 5.0
//     TB/s, from memory that nothing has written to before; 78 us straight after a
//     kernel that wrote as much, whose lines are then written back meanwhile.
//     1001 rows of 32000 floats (128 MB) 24.7 us a call, 5.2 TB/s. A batch of four
//     vectors with one maximum and the next on its way, against a vector at a
//     time: 27 -> 24 us (two workgroups a row). Few rows are bound by the chain of
//     steps behind the loads: 8 rows of 50257 with 20 tokens 7 to 9 us, and 5.1 us
//     to join them.
#include <type_traits>

#include "cf_common.hpp"

namespace cf {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWaveSize;
constexpr int kTopMax = 64;
/// Threads whose logits are looked through together by the search for the
/// likeliest: as many teams as tokens may be asked for.
constexpr int kTeam = kThreads / kTopMax;
constexpr int kTokensMax = 1024;
/// Keys that the filter may keep before the slow search takes over. Logits that
/// are all equal (a masked row) leave the first vector of each thread of as many
/// teams as tokens are asked for, and up to seven logits before the first vector:
/// 2031 in 16 bits. (With room for 1024, 600 rows of 131072 in fp16, all but 100
/// logits masked, took 1904 us for 64 tokens and take 99 now, like any others.)
constexpr int kCandidates = 2048;
static_assert(kTopMax * kTeam * 8 <= kCandidates, "equal 16-bit logits");
constexpr int kChunksMax = 1024;  // of a row
static_assert(kChunksMax + kTopMax <= kCandidates, "the joining kernel holds the first keys of every chunk");
constexpr int kUnroll = 4;  // vectors of a batch; two batches are in flight
constexpr int kHeld = 8;           // keys that a thread of the joining kernel keeps in registers
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
/// Below every exponent that leaves something in fp32: a stand-in for the
/// logarithm of a probability that is 0.
constexpr float kNothing = -256.0f;
constexpr float kLowest = -3.0e38f;
/// Most logits per row: a row's chunks (at most 128 vectors a thread) then
/// stay within kChunksMax.
constexpr int64_t kVocabMax = int64_t{1} << 27;
static_assert(kVocabMax * 4 / 16 / (128 * kThreads) <= kChunksMax, "chunks of the longest row");

typedef unsigned long long u64;

struct RowArgs {
    const void* logits;
    const int64_t* tokens;
    float* logprobs;
    float* stats;    // [rows, 2]: maximum logit, log2 of sum e^(x - scale max); may be null
    float* entropy;  // may be null
    float* top_logprobs;
    int64_t* top_tokens;
    float* partial;  // [rows, chunks, 4]: maximum, sum, weighted sum, unused
    u64* keys;       // [rows, chunks, top]
    int64_t rows;
    int64_t vocab;
    int64_t stride;
    int64_t count;
    int64_t vectors_per_chunk;
    int chunks;
    int top;
    float scale;
    float c;  // scale * log2(e)
};

/// A logit's place in the order "larger first, then lower index", as an
/// unsigned number: larger is earlier. NaN counts as the largest; -0 as 0.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    if (v != v) return 0xFFFFFFFFu;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
    if (o == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ u64 key_of(float v, uint32_t index) {
    return (static_cast<u64>(ordered(v)) << 32) | static_cast<uint32_t>(~index);
}

/// Where the 16-byte vectors of a row lie, and which of them are a chunk's.
template <typename T>
struct Span {
    static constexpr int kVec = Storage<T>::kPerVec;
    const T* row;
    uint32_t vocab;
    uint32_t head;   // elements before the first aligned vector
    uint32_t v_lo, v_hi;
    uint32_t tail;   // first element behind the last vector
    bool first, last;

    __device__ Span(const void* base, int64_t vocab_, int64_t row_offset, int64_t per_chunk, int chunk, int chunks) {
        row = static_cast<const T*>(base) + row_offset;
        vocab = static_cast<uint32_t>(vocab_);
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15u);
        head = off == 0 ? 0u : (16u - off) / sizeof(T);
        if (head > vocab) head = vocab;
        const uint32_t vectors = (vocab - head) / kVec;
        tail = head + vectors * kVec;
        const int64_t lo = per_chunk * chunk;
        const int64_t hi = lo + per_chunk;
        v_lo = lo < vectors ? static_cast<uint32_t>(lo) : vectors;
        v_hi = hi < vectors ? static_cast<uint32_t>(hi) : vectors;
        first = chunk == 0;
        last = chunk == chunks - 1;
        if (last) v_hi = vectors;
    }
    __device__ uint32_t base_of(uint32_t vector) const { return head + vector * kVec; }
    __device__ uint4 load(uint32_t vector) const {
        return *reinterpret_cast<const uint4*>(row + base_of(vector));
    }
    /// The thread's elements outside the vectors: index, or vocab for none.
    __device__ uint32_t head_element(int tid) const {
        return first && static_cast<uint32_t>(tid) < head ? static_cast<uint32_t>(tid) : vocab;
    }
    __device__ uint32_t tail_element(int tid) const {
        const uint32_t e = tail + static_cast<uint32_t>(tid);
        return last && e < vocab ? e : vocab;
    }
};

/// A partial result: maximum logit m, l = sum e^(scale (x - m)), and t = the
/// sum of e^.. * scale (x - m) log2(e). Nothing yet: m = -inf, l = t = 0.
struct Sums {
    float m, l, t;
};

__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float c) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    r.l = 0.0f;
    r.t = 0.0f;
    const Sums* parts[2] = {&a, &b};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const Sums& s = *parts[i];
        if (s.m == -INFINITY) {  // nothing, or a NaN
            r.l += s.l;
            r.t += s.t;
            continue;
        }
        const float d = (s.m - r.m) * c;
        const float f = exp2f(d);
        r.l = fmaf(s.l, f, r.l);
        r.t += fmaf(s.l, fmaxf(d, kNothing), s.t) * f;
        if (d != d) r.l = d;  // a maximum of +inf
    }
    return r;
}

__device__ __forceinline__ u64 wave_max_u64(u64 v) {
#pragma unroll
    for (int d = 1; d < kWaveSize; d <<= 1) {
        const u64 o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}

struct Shared {
    float f[kWaves];
    Sums waves[kWaves];
    u64 best[kTopMax];
    u64 candidates[kCandidates];
    u64 sorted[kTopMax];
    int selected[kTopMax];
    u64 threshold;
    int kept;
};

/// How many teams of kTeam neighbouring threads have a better best key than
/// the thread's team; `best` becomes the team's own. Keys differ (0: none).
/// Each thread of a team looks at a quarter of the teams.
__device__ __forceinline__ int rank_of_team(u64& best, u64* bests) {
    const int tid = static_cast<int>(threadIdx.x);
    static_assert(kTeam == 4 && kThreads / kTeam == kTopMax, "two exchanges");
#pragma unroll
    for (int d = 1; d < kTeam; d <<= 1) {
        const u64 o = __shfl_xor(best, d);
        best = o > best ? o : best;
    }
    if (tid % kTeam == 0) bests[tid / kTeam] = best;
    __syncthreads();
    int rank = 0;
#pragma unroll
    for (int i = 0; i < kTopMax / kTeam; ++i) rank += bests[i * kTeam + tid % kTeam] > best ? 1 : 0;
#pragma unroll
    for (int d = 1; d < kTeam; d <<= 1) rank += __shfl_xor(rank, d);
    return rank;
}

/// The `top` largest of the keys (which differ) into their places: each key
/// against all others by four threads.
__device__ __forceinline__ void rank_keys(const u64* keys, int count, int top, u64* out) {
    const int tid = static_cast<int>(threadIdx.x);
    for (int i = tid / kTeam; i < count; i += kThreads / kTeam) {
        const u64 key = keys[i];
        int place = 0;
#pragma unroll 4
        for (int j = tid % kTeam; j < count; j += kTeam) place += keys[j] > key ? 1 : 0;
#pragma unroll
        for (int d = 1; d < kTeam; d <<= 1) place += __shfl_xor(place, d);
        if (tid % kTeam == 0 && place < top) out[place] = key;
    }
}

/// The k best keys of the chunk in descending order into out[0 .. top) (0
/// where the chunk has fewer elements). `best` is the thread's own best
/// logit's vector: its value and the index of the vector's first element.
template <typename T>
__device__ void chunk_top(const Span<T>& s, u64 best, int top, Shared& sh, u64* out) {
    constexpr int kVec = Span<T>::kVec;
    const int tid = static_cast<int>(threadIdx.x);
    if (tid == 0) {
        sh.kept = 0;
        sh.threshold = 0;
    }
    if (tid < top) sh.selected[tid] = -1;
    int rank = rank_of_team(best, sh.best);
    if (best != 0 && rank < top && tid % kTeam == 0) {
        sh.selected[rank] = tid;
        // The team's best element lies within its vector: at most kVec - 1
        // places later than the vector's first.
        if (rank == top - 1) {
            const uint32_t low = static_cast<uint32_t>(best);
            sh.threshold = (best & 0xFFFFFFFF00000000ull) | (low >= kVec - 1 ? low - (kVec - 1) : 0u);
        }
    }
    __syncthreads();
    const u64 threshold = sh.threshold;
    const uint32_t per_thread = (s.v_hi - s.v_lo + kThreads - 1) / kThreads + 1;  // vectors, and the loose elements
    auto offer = [&](float v, uint32_t index) {
        const u64 key = key_of(v, index);
        if (key >= threshold) {
            const int at = atomicAdd(&sh.kept, 1);
            if (at < kCandidates) sh.candidates[at] = key;
        }
    };
    const uint32_t per_team = per_thread * kTeam;
    for (uint32_t item = tid; item < per_team * static_cast<uint32_t>(top); item += kThreads) {
        const int first = sh.selected[item / per_team];
        if (first < 0) continue;
        const uint32_t i = item % per_team / kTeam;
        const int owner = first + static_cast<int>(item % kTeam);
        if (i + 1 == per_thread) {
            const uint32_t h = s.head_element(owner);
            const uint32_t e = s.tail_element(owner);
            if (h < s.vocab) offer(Storage<T>::load(s.row + h), h);
            if (e < s.vocab) offer(Storage<T>::load(s.row + e), e);
            continue;
        }
        const uint32_t v = s.v_lo + i * kThreads + owner;
        if (v >= s.v_hi) continue;
        float x[kVec];
        unpack16<T>(s.load(v), x);
#pragma unroll
        for (int e = 0; e < kVec; ++e) offer(x[e], s.base_of(v) + e);
    }
    __syncthreads();
    int kept = sh.kept;
    if (kept <= kCandidates) {
        if (kept > 2 * kThreads / kTeam) {
            // Many equal logits (a masked row): the same sieve once more, over
            // the keys, since ranking them costs their number squared. They
            // lie as the waves brought them, neighbours beside each other; a
            // team takes every kSpread-th (the golden section of them all), so
            // that each has some of the best.
            constexpr int kEach = kCandidates / kThreads;
            constexpr int kSpread = 1265;
            static_assert(kCandidates == 2048, "kSpread");
            u64 held[kEach];
            best = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int from = (tid * kEach + i) * kSpread % kCandidates;
                held[i] = from < kept ? sh.candidates[from] : 0;
                best = held[i] > best ? held[i] : best;
            }
            if (tid == 0) sh.threshold = 0;
            __syncthreads();  // all have read the number and the keys
            if (tid == 0) sh.kept = 0;
            rank = rank_of_team(best, sh.best);
            if (best != 0 && rank == top - 1 && tid % kTeam == 0) sh.threshold = best;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                if (held[i] != 0 && held[i] >= sh.threshold) sh.candidates[atomicAdd(&sh.kept, 1)] = held[i];
            }
            __syncthreads();
            kept = sh.kept;
        }
        rank_keys(sh.candidates, kept, top, out);
        for (int i = kept + tid; i < top; i += kThreads) out[i] = 0;
        return;
    }
    // More logits than fit (they would have to be dealt so that the same few
    // teams hold them): one search over the chunk for each place.
    u64 previous = 0;  // of the place before; the first has none (a NaN as token 0 has the largest key there is)
    for (int place = 0; place < top; ++place) {
        u64 mine = 0;
        auto look = [&](float v, uint32_t index) {
            const u64 key = key_of(v, index);
            if ((place == 0 || key < previous) && key > mine) mine = key;
        };
        const uint32_t h = s.head_element(tid);
        const uint32_t e = s.tail_element(tid);
        if (h < s.vocab) look(Storage<T>::load(s.row + h), h);
        if (e < s.vocab) look(Storage<T>::load(s.row + e), e);
        for (uint32_t v = s.v_lo + tid; v < s.v_hi; v += kThreads) {
            float x[kVec];
            unpack16<T>(s.load(v), x);
#pragma unroll
            for (int k = 0; k < kVec; ++k) look(x[k], s.base_of(v) + k);
        }
        mine = wave_max_u64(mine);
        __syncthreads();  // the previous round's reads are done
        if ((tid & (kWaveSize - 1)) == 0) sh.best[tid / kWaveSize] = mine;
        __syncthreads();
        previous = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) previous = sh.best[w] > previous ? sh.best[w] : previous;
        if (tid == 0) out[place] = previous;
    }
}

/// The thread's given token and its logit, asked for long before they are used.
template <typename T>
struct Given {
    int64_t id = -1;  // none
    float logit = 0.0f;

    __device__ void token(const RowArgs& a, int64_t row) {
        if (threadIdx.x < a.count) id = a.tokens[row * a.count + threadIdx.x];
    }
    __device__ void fetch(const RowArgs& a, int64_t row) {
        if (id >= 0 && id < a.vocab) logit = Storage<T>::load(static_cast<const T*>(a.logits) + row * a.stride + id);
    }
};

/// The row's results from its joined sums and its sorted top keys.
template <typename T>
__device__ void finish_row(const RowArgs& a, int64_t row, const Sums& s, const Given<T>& given, const u64* top_keys) {
    const int tid = static_cast<int>(threadIdx.x);
    const float log2l = log2f(s.l);
    if (tid == 0) {
        if (a.stats != nullptr) {
            a.stats[2 * row] = s.m;
            a.stats[2 * row + 1] = log2l;
        }
        if (a.entropy != nullptr) a.entropy[row] = (log2l - s.t / s.l) * kLn2;
    }
    for (int64_t i = tid; i < a.count; i += kThreads) {
        int64_t id = given.id;
        float logit = given.logit;
        if (i >= kThreads) {
            id = a.tokens[row * a.count + i];
            if (id >= 0 && id < a.vocab) logit = Storage<T>::load(static_cast<const T*>(a.logits) + row * a.stride + id);
        }
        float r = 0.0f;  // padding
        if (id >= a.vocab) {
            r = __uint_as_float(0x7FC00000u);
        } else if (id >= 0) {
            r = fmaf(logit - s.m, a.scale, -log2l * kLn2);
        }
        a.logprobs[row * a.count + i] = r;
    }
    for (int i = tid; i < a.top; i += kThreads) {
        const u64 key = top_keys[i];
        a.top_tokens[row * a.top + i] = static_cast<uint32_t>(~static_cast<uint32_t>(key));
        a.top_logprobs[row * a.top + i] =
            fmaf(unordered(static_cast<uint32_t>(key >> 32)) - s.m, a.scale, -log2l * kLn2);
    }
}

template <typename T, bool kEntropy, bool kTop>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(RowArgs a) {
    constexpr int kVec = Span<T>::kVec;
    __shared__ Shared sh;
    const int tid = static_cast<int>(threadIdx.x);
    const int chunk = static_cast<int>(blockIdx.x % a.chunks);
    const int64_t row = blockIdx.x / a.chunks;
    const Span<T> s(a.logits, a.vocab, row * a.stride, a.vectors_per_chunk, chunk, a.chunks);
    const float c = a.c;

    // The thread's own maximum logit and where it first stands; sums relative
    // to mc = m c as rounded.
    float m = -INFINITY;
    float mc = kLowest;
    float l = 0.0f;
    float t = 0.0f;
    uint32_t where = s.vocab;
    auto raise = [&](float vmax, uint32_t index) {
        if (kTop && (vmax > m || where == s.vocab)) where = index;
        if (vmax > m) {
            m = vmax;
            // Not below the start: rows masked with the type's lowest value.
            const float next = fmaxf(vmax * c, kLowest);
            const float d = mc - next;
            const float f = exp2f(d);
            if (kEntropy) t = fmaf(l, fmaxf(d, kNothing), t) * f;
            l *= f;
            mc = next;
        }
    };
    auto add = [&](float x) {
        const float d = fmaf(x, c, -mc);
        const float e = __builtin_amdgcn_exp2f(d);
        l += e;
        if (kEntropy) t = fmaf(e, fmaxf(d, kNothing), t);
    };
    Given<T> given;
    if (a.chunks == 1) given.token(a, row);
    const uint32_t h = s.head_element(tid);
    const uint32_t tail = s.tail_element(tid);
    if (h < s.vocab) {
        const float x = Storage<T>::load(s.row + h);
        raise(x, h);
        add(x);
    }
    // Batches of vectors: one maximum, and rarely a raise, for a whole batch; two
    // sums, so that neither is one long chain of additions. The next batch is
    // under way meanwhile; behind the chunk's end it reads the last vector again.
    if (s.v_lo + tid < s.v_hi) {
        constexpr uint32_t kBatch = kUnroll * kThreads;
        const uint32_t last = s.v_hi - 1;
        uint4 next[kUnroll];
        auto fetch = [&](uint32_t v) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const uint32_t at = v + u * kThreads;
                next[u] = s.load(at < last ? at : last);
            }
        };
        fetch(s.v_lo + tid);
        for (uint32_t v = s.v_lo + tid; v < s.v_hi; v += kBatch) {
            uint4 raw[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) raw[u] = next[u];
            if (v + kBatch < s.v_hi) fetch(v + kBatch);
            if (v + (kBatch - kThreads) >= s.v_hi) {
                constexpr uint32_t kNone = Storage<T>::kPerVec == 4                ? 0xFF800000u
                                           : std::is_same<T, bf16_t>::value ? 0xFF80FF80u
                                                                            : 0xFC00FC00u;  // -inf
#pragma unroll
                for (int u = 1; u < kUnroll; ++u) {
                    if (v + u * kThreads >= s.v_hi) raw[u] = uint4{kNone, kNone, kNone, kNone};
                }
            }
            float best[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                float x[kVec];
                unpack16<T>(raw[u], x);
                best[u] = x[0];
#pragma unroll
                for (int e = 1; e < kVec; ++e) best[u] = fmaxf(best[u], x[e]);
            }
            float top = best[0];
#pragma unroll
            for (int u = 1; u < kUnroll; ++u) top = fmaxf(top, best[u]);
            if (top > m || (kTop && where == s.vocab)) {
                uint32_t index = s.base_of(v);  // the first vector that holds the maximum
                if (kTop) {
#pragma unroll
                    for (int u = kUnroll - 1; u > 0; --u) {
                        if (best[u] == top) index = s.base_of(v + u * kThreads);
                    }
                    if (best[0] == top) index = s.base_of(v);
                }
                raise(top, index);
            }
            float l2 = 0.0f;
            float t2 = 0.0f;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                float x[kVec];
                unpack16<T>(raw[u], x);
#pragma unroll
                for (int e = 0; e < kVec; e += 2) {
                    const float d0 = fmaf(x[e], c, -mc);
                    const float d1 = fmaf(x[e + 1], c, -mc);
                    const float e0 = __builtin_amdgcn_exp2f(d0);
                    const float e1 = __builtin_amdgcn_exp2f(d1);
                    l += e0;
                    l2 += e1;
                    if (kEntropy) {
                        t = fmaf(e0, fmaxf(d0, kNothing), t);
                        t2 = fmaf(e1, fmaxf(d1, kNothing), t2);
                    }
                }
            }
            l += l2;
            if (kEntropy) t += t2;
        }
    }
    if (tail < s.vocab) {
        const float x = Storage<T>::load(s.row + tail);
        raise(x, tail);
        add(x);
    }
    if (a.chunks == 1) given.fetch(a, row);  // on its way while the threads are joined

    // From the threads' rounded m c to the exact one of their wave, then all waves.
    Sums sum;
    sum.m = wave_reduce_f32<MaxF32>(m);
    if (m != -INFINITY) {
        const float d = fmaf(-sum.m, c, mc);
        const float f = exp2f(d);
        if (kEntropy) t = fmaf(l, fmaxf(d, kNothing), t) * f;
        l *= f;
    } else if (kEntropy) {
        t = l;  // 0, or a NaN
    }
    sum.l = wave_reduce_f32<AddF32>(l);
    sum.t = kEntropy ? wave_reduce_f32<AddF32>(t) : 0.0f;
    if (tid % kWaveSize == 0) sh.waves[tid / kWaveSize] = sum;
    __syncthreads();
    sum = sh.waves[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum = join(sum, sh.waves[w], c);
    u64 best = kTop && where < s.vocab ? key_of(m, where) : 0;
    // Rows at the ends of the number range, and NaN.
    if (!(fabsf(sum.m) * fmaxf(c, 1.0f) < 1.0e38f || sum.m == -INFINITY) || sum.l != sum.l) {
        float ls = 0.0f;
        float ts = 0.0f;
        best = 0;
        auto again = [&](float x, uint32_t index) {
            const float d = sum.m == -INFINITY ? x : (x - sum.m) * c;  // a NaN stays one
            const float e = exp2f(d);
            ls += e;
            ts = fmaf(e, fmaxf(d, kNothing), ts);
            const u64 key = key_of(x, index);
            if (key > best) best = key;
        };
        if (h < s.vocab) again(Storage<T>::load(s.row + h), h);
        for (uint32_t w = s.v_lo + tid; w < s.v_hi; w += kThreads) {
            float x[kVec];
            unpack16<T>(s.load(w), x);
#pragma unroll
            for (int e = 0; e < kVec; ++e) again(x[e], s.base_of(w) + e);
        }
        if (tail < s.vocab) again(Storage<T>::load(s.row + tail), tail);
        sum.l = block_reduce_f32<kWaves, AddF32>(ls, sh.f);
        sum.t = kEntropy ? block_reduce_f32<kWaves, AddF32>(ts, sh.f) : 0.0f;
    }

    const int64_t at = row * a.chunks + chunk;
    if (kTop) chunk_top<T>(s, best, a.top, sh, a.chunks == 1 ? sh.sorted : a.keys + at * a.top);
    if (a.chunks == 1) {
        if (kTop) __syncthreads();
        finish_row<T>(a, row, sum, given, sh.sorted);
        return;
    }
    if (tid == 0) {
        a.partial[4 * at] = sum.m;
        a.partial[4 * at + 1] = sum.l;
        a.partial[4 * at + 2] = sum.t;
    }
}

/// One workgroup per row joins its chunks. The top keys: the smallest of any
/// top keys is a threshold that the answer lies above. Two such sets are taken
/// from the chunks' sorted lists (the first few of every list; the whole of
/// the best list), and the keys above the higher threshold are ranked against
/// each other.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(RowArgs a) {
    __shared__ Shared sh;
    __shared__ Sums joined;
    const int tid = static_cast<int>(threadIdx.x);
    const int64_t row = blockIdx.x;
    const u64* keys = a.keys + row * a.chunks * a.top;
    const int total = a.chunks * a.top;
    const int each = a.top > 0 ? (a.top + a.chunks - 1) / a.chunks : 0;  // of every list: at least top keys in all
    const int heads = each * a.chunks;
    Given<T> given;
    given.token(a, row);
    // Read at once what will be needed.
    u64 held[kHeld];
    u64 last = 0;  // the largest last key of the lists
    if (a.top > 0) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) held[i] = keys[min(i * kThreads + tid, total - 1)];
        for (int i = tid; i < a.chunks; i += kThreads) {
            const u64 key = keys[(i + 1) * a.top - 1];
            last = key > last ? key : last;
        }
        for (int i = tid; i < heads; i += kThreads) sh.candidates[i] = keys[i / each * a.top + i % each];
    }
    given.fetch(a, row);
    if (tid < kWaveSize) {
        Sums s{-INFINITY, 0.0f, 0.0f};
        for (int i = tid; i < a.chunks; i += kWaveSize) {
            const float4 p = *reinterpret_cast<const float4*>(a.partial + 4 * (row * a.chunks + i));
            s = join(s, Sums{p.x, p.y, p.z}, a.c);
        }
        // The lanes' sums to the largest maximum, as join() does, then added up.
        Sums all;
        all.m = wave_reduce_f32<MaxF32>(s.m);
        if (s.m != -INFINITY) {
            const float d = (s.m - all.m) * a.c;
            const float f = exp2f(d);
            s.t = fmaf(s.l, fmaxf(d, kNothing), s.t) * f;
            s.l = d == d ? s.l * f : d;
        }
        all.l = wave_reduce_f32<AddF32>(s.l);
        all.t = wave_reduce_f32<AddF32>(s.t);
        if (tid == 0) joined = all;
    }
    if (a.top > 0) {
        auto each_key = [&](auto&& f) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (i * kThreads + tid < total) f(held[i]);
            }
            for (int i = kHeld * kThreads + tid; i < total; i += kThreads) f(keys[i]);
        };
        const u64 best = wave_max_u64(last);
        if (tid % kWaveSize == 0) sh.best[tid / kWaveSize] = best;
        if (tid == 0) {
            sh.kept = 0;
            sh.threshold = 0;
        }
        __syncthreads();
        for (int i = tid / kTeam; i < heads; i += kThreads / kTeam) {
            const u64 key = sh.candidates[i];
            int rank = 0;
#pragma unroll 4
            for (int j = tid % kTeam; j < heads; j += kTeam) rank += sh.candidates[j] > key ? 1 : 0;
#pragma unroll
            for (int d = 1; d < kTeam; d <<= 1) rank += __shfl_xor(rank, d);
            if (key != 0 && rank == a.top - 1 && tid % kTeam == 0) sh.threshold = key;
        }
        __syncthreads();
        u64 threshold = sh.threshold;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) threshold = sh.best[w] > threshold ? sh.best[w] : threshold;
        each_key([&](u64 key) {
            if (key >= threshold && key != 0) {
                const int at = atomicAdd(&sh.kept, 1);
                if (at < kCandidates) sh.candidates[at] = key;
            }
        });
        __syncthreads();
        const int kept = sh.kept;
        if (kept <= kCandidates) {
            rank_keys(sh.candidates, kept, a.top, sh.sorted);
        } else {
            for (int i = tid; i < total; i += kThreads) {
                const u64 key = keys[i];
                if (key < threshold || key == 0) continue;
                int place = 0;
                for (int j = 0; j < total; ++j) place += keys[j] > key ? 1 : 0;
                if (place < a.top) sh.sorted[place] = key;
            }
        }
    }
    __syncthreads();
    finish_row<T>(a, row, joined, given, sh.sorted);
}

struct GradArgs {
    const void* logits;
    const int64_t* tokens;
    const float* stats;
    const float* entropy;
    const float* grad_logprobs;  // null: zeros
    const float* grad_entropy;   // null: zeros
    void* grad;
    int64_t vocab;
    int64_t stride;
    int64_t grad_stride;
    int64_t count;
    int64_t vectors_per_chunk;
    int chunks;
    float scale;
    float c;
};

/// The gradient of one chunk of a row. The tokens' own terms are added after a
/// barrier by recomputing those elements whole: a token given twice gets the
/// sum of its gradients in the order given, once rounded.
template <typename T, bool kEntropy>
__global__ __launch_bounds__(kThreads) void logprobs_grad_kernel(GradArgs a) {
    constexpr int kVec = Span<T>::kVec;
    __shared__ float slots[kWaves];
    __shared__ int flags[kWaves];
    const int tid = static_cast<int>(threadIdx.x);
    const int chunk = static_cast<int>(blockIdx.x % a.chunks);
    const int64_t row = blockIdx.x / a.chunks;
    const Span<T> s(a.logits, a.vocab, row * a.stride, a.vectors_per_chunk, chunk, a.chunks);
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
    const int64_t* tokens = a.tokens + row * a.count;
    const float* given = a.grad_logprobs == nullptr ? nullptr : a.grad_logprobs + row * a.count;

    // Given token i's part of G: none where no log probability is differentiated.
    auto weight = [&](int64_t i, int64_t token) {
        return given == nullptr ? 0.0f : token >= a.vocab ? __uint_as_float(0x7FC00000u) : given[i];
    };
    float total = 0.0f;
    bool any = false;
    for (int64_t i = tid; i < a.count; i += kThreads) {
        const int64_t token = tokens[i];
        if (token < 0) continue;
        any = true;
        total += weight(i, token);
    }
    if (a.count > 1) {
        total = block_reduce_f32<kWaves, AddF32>(total, slots);
        any = workgroup_any<kWaves>(any, flags);
    } else {
        const int64_t token = tokens[0];
        any = token >= 0;
        total = any ? weight(0, token) : 0.0f;
    }
    const float h = kEntropy ? a.grad_entropy[row] : 0.0f;
    const float big_h = kEntropy ? a.entropy[row] : 0.0f;
    const float m = a.stats[2 * row];
    const float log2l = a.stats[2 * row + 1];
    const float neg_scale = -a.scale;
    auto grad = [&](float x) {
        const float d = fmaf(x - m, a.c, -log2l);
        const float p = __builtin_amdgcn_exp2f(d) * neg_scale;
        if (kEntropy) return p * fmaf(h, fmaf(fmaxf(d, kNothing), kLn2, big_h), total);
        return p * total;
    };
    // A row of padding alone has no gradient: nothing is read.
    const bool empty = !any && h == 0.0f;
    const uint32_t edges[2] = {s.head_element(tid), s.tail_element(tid)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (edges[i] < s.vocab) Storage<T>::store(out + edges[i], empty ? 0.0f : grad(Storage<T>::load(s.row + edges[i])));
    }
    const bool aligned = aligned16(out + s.head);
    for (uint32_t v = s.v_lo + tid; v < s.v_hi; v += kThreads) {
        float x[kVec];
        if (empty) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) x[e] = 0.0f;
        } else {
            unpack16<T>(s.load(v), x);
#pragma unroll
            for (int e = 0; e < kVec; ++e) x[e] = grad(x[e]);
        }
        T* to = out + s.base_of(v);
        if (aligned) {
            *reinterpret_cast<uint4*>(to) = pack16<T>(x);
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) Storage<T>::store(to + e, x[e]);
        }
    }
    if (given == nullptr) return;
    __syncthreads();
    const uint32_t lo = s.first ? 0u : s.base_of(s.v_lo);
    const uint32_t hi = s.last ? s.vocab : s.base_of(s.v_hi);
    for (int64_t i = tid; i < a.count; i += kThreads) {
        const int64_t token = tokens[i];
        if (token < static_cast<int64_t>(lo) || token >= static_cast<int64_t>(hi)) continue;
        float own = 0.0f;
        bool mine = true;
        for (int64_t j = 0; j < a.count; ++j) {
            if (tokens[j] != token) continue;
            if (j < i) {
                mine = false;
                break;
            }
            own += given[j];
        }
        if (mine) Storage<T>::store(out + token, fmaf(own, a.scale, grad(Storage<T>::load(s.row + token))));
    }
}

/// Chunks per row: the given number of workgroups in all where there are few
/// rows, but no chunk under a vector a thread, and none above 128 vectors a thread.
int chunks_of(int64_t rows, int64_t vocab, size_t size, int64_t workgroups) {
    const int64_t vectors = ceil_div<int64_t>(vocab * static_cast<int64_t>(size), 16);
    const int64_t many = ceil_div<int64_t>(workgroups, rows);
    const int64_t wanted = many < kChunksMax ? many : kChunksMax;
    const int64_t most = ceil_div<int64_t>(vectors, kThreads);
    const int64_t least = ceil_div<int64_t>(vectors, 128 * kThreads);
    int64_t chunks = wanted < most ? wanted : most;
    if (chunks < least) chunks = least;
    return static_cast<int>(chunks < 1 ? 1 : chunks);
}

/// The forward: 512 workgroups, since a row that is not cut needs no join. Many
/// of the likeliest tokens of long rows: 2048, since a chunk's sieve reads its
/// teams' vectors again, and takes the longer the more there are. Whole calls in
/// us at 512 | 1024 | 2048 workgroups, rows of bf16 out of memory:
///   600 x 32000, none of the likeliest  12.1 | 15.5 | 15.1;   5: 16.6 | 22.5 | 22.7
///   1001 x 32000                        16.9 | 20.7 | 22.6;      21.9 | 28.1 | 32.2
///   600 x 131072                        32.9 | 36.3 | 35.3;      43.0 | 47.0 | 44.5
///   600 x 131072, 20 of the likeliest   57.9 | 58.3 | 54.2;  48: 89.5 | 78.7 | 74.6
/// Against 2048 throughout, over 1 to 3000 rows of 4099 to 131072 in bf16 and
/// fp32 with 0 to 64 of the likeliest, calls take 14% less on average, 9% more at
/// most (200 rows of 131072 floats) and a third at least (1001 rows of 4099).
int64_t forward_groups(int64_t vocab, size_t size, int64_t top) {
    return top > 8 && vocab * static_cast<int64_t>(size) / 16 > 32 * kThreads ? 2048 : 512;
}

/// The backward joins nothing, and is bound by its stores: 1024 workgroups (300
/// rows of 131072 in bf16 39.2 us at 512, 28.9 at 1024, 32.2 at 2048; 600 rows 77.3,
/// 56.7 and 60.0; 1700 rows of 32000 39.4, 39.3 and 37.4).
constexpr int64_t kBackwardGroups = 1024;

int64_t vectors_per_chunk(int64_t vocab, size_t size, int chunks) {
    return ceil_div<int64_t>(ceil_div<int64_t>(vocab * static_cast<int64_t>(size), 16), chunks);
}

size_t round_up(size_t bytes) { return (bytes + 15) / 16 * 16; }

cf_status validate(const char* who, const void* logits, cf_dtype dtype, int64_t rows, int64_t vocab,
                   int64_t row_stride, const int64_t* tokens, int64_t token_count, float scale) {
    CF_REQUIRE(valid_dtype(dtype), "%s: unknown dtype %d", who, static_cast<int>(dtype));
    CF_REQUIRE(logits != nullptr && tokens != nullptr, "%s: null pointer", who);
    CF_REQUIRE(vocab <= kVocabMax, "%s: vocab %lld is above %lld", who, static_cast<long long>(vocab),
               static_cast<long long>(kVocabMax));
    CF_REQUIRE(row_stride >= vocab, "%s: row_stride %lld is below vocab %lld", who, static_cast<long long>(row_stride),
               static_cast<long long>(vocab));
    CF_REQUIRE(token_count >= 1 && token_count <= kTokensMax, "%s: token_count %lld is not in 1 .. %d", who,
               static_cast<long long>(token_count), kTokensMax);
    CF_REQUIRE(scale > 0.0f && scale * kLog2e < 1.0e30f, "%s: scale must be positive and finite", who);
    CF_REQUIRE(host_aligned(logits, dtype_size(dtype)) && host_aligned(tokens, 8), "%s: misaligned pointer", who);
    CF_REQUIRE(rows * chunks_of(rows, vocab, dtype_size(dtype), 1) < (1LL << 31), "%s: %lld rows are too many", who,
               static_cast<long long>(rows));
    return CF_OK;
}

/// p + n, or null.
template <typename P>
P* at(P* p, int64_t n) {
    return p == nullptr ? nullptr : p + n;
}

/// As many rows a launch as it takes workgroups.
template <typename T>
void run_forward(const RowArgs& all, hipStream_t stream) {
    const int64_t most = kMaxWorkgroups / all.chunks;
    for (int64_t row = 0; row < all.rows; row += most) {
        RowArgs a = all;
        a.rows = all.rows - row < most ? all.rows - row : most;
        a.logits = static_cast<const T*>(all.logits) + row * all.stride;
        a.tokens = all.tokens + row * all.count;
        a.logprobs = all.logprobs + row * all.count;
        a.stats = at(all.stats, 2 * row);
        a.entropy = at(all.entropy, row);
        a.top_logprobs = at(all.top_logprobs, row * all.top);
        a.top_tokens = at(all.top_tokens, row * all.top);
        a.partial = at(all.partial, 4 * row * all.chunks);
        a.keys = at(all.keys, row * all.chunks * all.top);
        const dim3 grid(static_cast<unsigned>(a.rows * a.chunks));
        const dim3 block(kThreads);
        const bool entropy = a.entropy != nullptr;
        if (a.top > 0) {
            launch(entropy ? logprobs_kernel<T, true, true> : logprobs_kernel<T, false, true>, grid, block, 0, stream,
                   a);
        } else {
            launch(entropy ? logprobs_kernel<T, true, false> : logprobs_kernel<T, false, false>, grid, block, 0,
                   stream, a);
        }
        if (a.chunks > 1) {
            launch(logprobs_join_kernel<T>, dim3(static_cast<unsigned>(a.rows)), block, 0, stream, a);
        }
    }
}

template <typename T>
void run_backward(const GradArgs& all, int64_t rows, hipStream_t stream) {
    const int64_t most = kMaxWorkgroups / all.chunks;
    for (int64_t row = 0; row < rows; row += most) {
        GradArgs a = all;
        a.logits = static_cast<const T*>(all.logits) + row * all.stride;
        a.tokens = all.tokens + row * all.count;
        a.stats = all.stats + 2 * row;
        a.entropy = at(all.entropy, row);
        a.grad_logprobs = at(all.grad_logprobs, row * all.count);
        a.grad_entropy = at(all.grad_entropy, row);
        a.grad = static_cast<T*>(all.grad) + row * all.grad_stride;
        const dim3 grid(static_cast<unsigned>((rows - row < most ? rows - row : most) * a.chunks));
        launch(a.grad_entropy != nullptr ? logprobs_grad_kernel<T, true> : logprobs_grad_kernel<T, false>, grid,
               dim3(kThreads), 0, stream, a);
    }
}

}  // namespace
}  // namespace cf

extern "C" {

size_t cf_token_logprobs_workspace_bytes(cf_dtype dtype, int64_t rows, int64_t vocab, int64_t top) {
    if (!cf::valid_dtype(dtype) || rows <= 0 || vocab <= 0 || top < 0) return 0;
    const size_t size = cf::dtype_size(dtype);
    const int chunks = cf::chunks_of(rows, vocab, size, cf::forward_groups(vocab, size, top));
    if (chunks == 1) return 0;
    return cf::round_up(static_cast<size_t>(rows) * chunks * 16) + static_cast<size_t>(rows) * chunks * top * 8;
}

cf_status cf_token_logprobs(const void* logits, cf_dtype dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                            const int64_t* tokens, int64_t token_count, float scale, float* logprobs,
                            float* row_stats, float* entropy, int64_t top, float* top_logprobs, int64_t* top_tokens,
                            void* workspace, size_t workspace_bytes, void* stream) {
    CF_ENTRY();
    if (rows <= 0 || vocab <= 0) return CF_OK;
    const char* who = "cf_token_logprobs";
    const cf_status st = cf::validate(who, logits, dtype, rows, vocab, row_stride, tokens, token_count, scale);
    if (st != CF_OK) return st;
    CF_REQUIRE(logprobs != nullptr, "%s: null pointer", who);
    CF_REQUIRE(top >= 0 && top <= cf::kTopMax && top <= vocab, "%s: top %lld is not in 0 .. %d, or above vocab", who,
               static_cast<long long>(top), cf::kTopMax);
    CF_REQUIRE(top == 0 || (top_logprobs != nullptr && top_tokens != nullptr), "%s: null pointer", who);
    const size_t needed = cf_token_logprobs_workspace_bytes(dtype, rows, vocab, top);
    CF_REQUIRE(needed == 0 || (workspace != nullptr && workspace_bytes >= needed && cf::host_aligned(workspace, 16)),
               "%s: needs %zu bytes of 16-byte aligned workspace", who, needed);
    cf::RowArgs a{};
    a.logits = logits;
    a.tokens = tokens;
    a.logprobs = logprobs;
    a.stats = row_stats;
    a.entropy = entropy;
    a.top_logprobs = top_logprobs;
    a.top_tokens = top_tokens;
    a.rows = rows;
    a.vocab = vocab;
    a.stride = row_stride;
    a.count = token_count;
    const size_t size = cf::dtype_size(dtype);
    a.chunks = cf::chunks_of(rows, vocab, size, cf::forward_groups(vocab, size, top));
    a.vectors_per_chunk = cf::vectors_per_chunk(vocab, cf::dtype_size(dtype), a.chunks);
    a.top = static_cast<int>(top);
    a.scale = scale;
    a.c = scale * cf::kLog2e;
    a.partial = static_cast<float*>(workspace);
    if (a.chunks > 1) {
        a.keys = reinterpret_cast<cf::u64*>(static_cast<uint8_t*>(workspace) +
                                            cf::round_up(static_cast<size_t>(rows) * a.chunks * 16));
    }
    auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case CF_F32: cf::run_forward<float>(a, s); break;
        case CF_F16: cf::run_forward<cf::f16_t>(a, s); break;
        case CF_BF16: cf::run_forward<cf::bf16_t>(a, s); break;
    }
    return cf::check_launch("launching the token log probabilities", s);
}

cf_status cf_token_logprobs_backward(const void* logits, cf_dtype dtype, int64_t rows, int64_t vocab,
                                     int64_t row_stride, const int64_t* tokens, int64_t token_count, float scale,
                                     const float* row_stats, const float* entropy, const float* grad_logprobs,
                                     const float* grad_entropy, void* grad_logits, int64_t grad_row_stride,
                                     void* stream) {
    CF_ENTRY();
    if (rows <= 0 || vocab <= 0) return CF_OK;
    const char* who = "cf_token_logprobs_backward";
    const cf_status st = cf::validate(who, logits, dtype, rows, vocab, row_stride, tokens, token_count, scale);
    if (st != CF_OK) return st;
    CF_REQUIRE(row_stats != nullptr && grad_logits != nullptr, "%s: null pointer", who);
    CF_REQUIRE(grad_entropy == nullptr || entropy != nullptr, "%s: an entropy gradient needs the entropy", who);
    CF_REQUIRE(grad_row_stride >= vocab, "%s: grad_row_stride %lld is below vocab %lld", who,
               static_cast<long long>(grad_row_stride), static_cast<long long>(vocab));
    CF_REQUIRE(cf::host_aligned(grad_logits, cf::dtype_size(dtype)), "%s: misaligned pointer", who);
    cf::GradArgs a{};
    a.logits = logits;
    a.tokens = tokens;
    a.stats = row_stats;
    a.entropy = entropy;
    a.grad_logprobs = grad_logprobs;
    a.grad_entropy = grad_entropy;
    a.grad = grad_logits;
    a.vocab = vocab;
    a.stride = row_stride;
    a.grad_stride = grad_row_stride;
    a.count = token_count;
    a.chunks = cf::chunks_of(rows, vocab, cf::dtype_size(dtype), cf::kBackwardGroups);
    a.vectors_per_chunk = cf::vectors_per_chunk(vocab, cf::dtype_size(dtype), a.chunks);
    a.scale = scale;
    a.c = scale * cf::kLog2e;
    auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case CF_F32: cf::run_backward<float>(a, rows, s); break;
        case CF_F16: cf::run_backward<cf::f16_t>(a, rows, s); break;
        case CF_BF16: cf::run_backward<cf::bf16_t>(a, rows, s); break;
    }
    return cf::check_launch("launching the token log probabilities' gradient", s);
}

}  // extern "C"
