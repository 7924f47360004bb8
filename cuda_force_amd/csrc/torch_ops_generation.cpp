// Dispatcher registration of the operators of token generation: pages of a
// paged cache, attention over it behind shared prompts, and log probabilities
// of tokens with their gradient. Same conventions as
// torch_ops.cpp: ATen on the CPU, the C ABI of libcudaforge_hip.so on
// PyTorch's current HIP stream on the GPU, never synchronising; workspaces
// from torch's caching allocator.
#include "torch_ops_common.hpp"

#include <algorithm>

namespace cudaforge_amd {
namespace {

// ---- token log probabilities -------------------------------------------------

using LogprobsResult = std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>;

void check_logits(const torch::Tensor& logits, const torch::Tensor& tokens, double scale) {
    check_2d(logits, "logits");
    TORCH_CHECK(logits.size(1) <= 1 || logits.stride(1) == 1, "logits must be dense along the vocabulary");
    TORCH_CHECK(logits.size(0) <= 1 || logits.stride(0) >= logits.size(1),
                "logits' rows overlap: call .contiguous() first");
    check_2d(tokens, "tokens");
    check_contiguous(tokens, "tokens");
    check_same_device(logits, tokens, "tokens");
    TORCH_CHECK(tokens.scalar_type() == torch::kInt64, "tokens must be int64, got ", tokens.scalar_type());
    TORCH_CHECK(tokens.size(0) == logits.size(0), "tokens has ", tokens.size(0), " rows but logits has ",
                logits.size(0));
    TORCH_CHECK(tokens.size(1) >= 1, "tokens must name at least one token per row");
    TORCH_CHECK(scale > 0, "scale must be positive, got ", scale);
}

int64_t row_stride(const torch::Tensor& rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

/// The results for tokens [rows, n], the first of them as `shape` has it.
LogprobsResult logprobs_of(const torch::Tensor& logits, const torch::Tensor& tokens, torch::IntArrayRef shape,
                           double scale, bool entropy, int64_t top) {
    check_logits(logits, tokens, scale);
    const at::DeviceGuard guard(logits.device());
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    TORCH_CHECK(top >= 0 && top <= vocab, "top ", top, " is not in 0 .. ", vocab, " (the vocabulary)");
    const auto f32 = logits.options().dtype(torch::kFloat32);
    torch::Tensor logprobs = torch::empty(shape, f32);
    torch::Tensor stats = torch::empty({rows, 2}, f32);
    torch::Tensor h = torch::empty({entropy ? rows : 0}, f32);
    torch::Tensor top_logprobs = torch::empty({top > 0 ? rows : 0, top}, f32);
    torch::Tensor top_tokens = torch::empty({top > 0 ? rows : 0, top}, tokens.options());
    const cf_dtype dtype = to_cf(logits, "logits");
    const size_t bytes = cf_token_logprobs_workspace_bytes(dtype, rows, vocab, top);
    torch::Tensor workspace;
    if (bytes > 0) workspace = torch::empty({static_cast<int64_t>(bytes)}, logits.options().dtype(torch::kUInt8));
    check_status(cf_token_logprobs(logits.data_ptr(), dtype, rows, vocab, row_stride(logits),
                                   tokens.data_ptr<int64_t>(), tokens.size(1), static_cast<float>(scale),
                                   logprobs.data_ptr<float>(), stats.data_ptr<float>(),
                                   entropy ? h.data_ptr<float>() : nullptr, top,
                                   top > 0 ? top_logprobs.data_ptr<float>() : nullptr,
                                   top > 0 ? top_tokens.data_ptr<int64_t>() : nullptr,
                                   bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_for(logits)));
    return {logprobs, stats, h, top_logprobs, top_tokens};
}

LogprobsResult token_logprobs_hip(const torch::Tensor& logits, const torch::Tensor& tokens, double scale,
                                  bool entropy, int64_t top) {
    return logprobs_of(logits, tokens, tokens.sizes(), scale, entropy, top);
}

/// Contiguous fp32 gradient of the expected shape, or null where it is absent.
const float* gradient(const std::optional<torch::Tensor>& g, const torch::Tensor& like, torch::IntArrayRef sizes,
                      const char* name, torch::Tensor& held) {
    if (!g.has_value() || !g->defined()) return nullptr;
    check_same_device(like, *g, name);
    TORCH_CHECK(g->sizes() == sizes, name, " has shape ", g->sizes(), ", expected ", sizes);
    TORCH_CHECK(g->scalar_type() == torch::kFloat32, name, " must be float32, got ", g->scalar_type());
    held = g->contiguous();
    return held.data_ptr<float>();
}

torch::Tensor token_logprobs_backward_hip(const torch::Tensor& logits, const torch::Tensor& tokens, double scale,
                                          const torch::Tensor& stats, const torch::Tensor& entropy,
                                          const std::optional<torch::Tensor>& grad_logprobs,
                                          const std::optional<torch::Tensor>& grad_entropy) {
    check_logits(logits, tokens, scale);
    const at::DeviceGuard guard(logits.device());
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    check_same_device(logits, stats, "stats");
    check_contiguous(stats, "stats");
    TORCH_CHECK(stats.scalar_type() == torch::kFloat32 && stats.numel() == 2 * rows, "stats must be float32 [", rows,
                ", 2]");
    torch::Tensor held_lp, held_h;
    const float* g = gradient(grad_logprobs, logits, tokens.sizes(), "grad_logprobs", held_lp);
    const float* h = gradient(grad_entropy, logits, {rows}, "grad_entropy", held_h);
    if (h != nullptr) {
        check_same_device(logits, entropy, "entropy");
        check_contiguous(entropy, "entropy");
        TORCH_CHECK(entropy.scalar_type() == torch::kFloat32 && entropy.numel() == rows, "entropy must be float32 [",
                    rows, "]");
    }
    // Laid out as the logits where their rows are padded to an aligned pitch, so
    // that the gradient's are aligned too; not where they are a small part of a
    // larger tensor's rows (the last position of each sequence), which it would
    // take the memory of.
    const int64_t pitch = row_stride(logits) - vocab <= 128 ? row_stride(logits) : vocab;
    torch::Tensor grad = torch::empty_strided(logits.sizes(), {pitch, 1}, logits.options());
    check_status(cf_token_logprobs_backward(logits.data_ptr(), to_cf(logits, "logits"), rows, vocab,
                                            row_stride(logits), tokens.data_ptr<int64_t>(), tokens.size(1),
                                            static_cast<float>(scale), stats.data_ptr<float>(),
                                            h != nullptr ? entropy.data_ptr<float>() : nullptr, g, h, grad.data_ptr(),
                                            row_stride(grad), stream_for(logits)));
    return grad;
}

LogprobsResult token_logprobs_cpu(const torch::Tensor& logits, const torch::Tensor& tokens, double scale,
                                  bool entropy, int64_t top) {
    check_logits(logits, tokens, scale);
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    TORCH_CHECK(top >= 0 && top <= vocab, "top ", top, " is not in 0 .. ", vocab, " (the vocabulary)");
    const torch::Tensor wide = logits.to(torch::kFloat32);
    const torch::Tensor shift = vocab > 0 ? std::get<0>(wide.max(1, true)) : torch::zeros({rows, 1}, wide.options());
    const torch::Tensor x = (wide - shift) * scale;
    const torch::Tensor log_sum = x.exp().sum(1, true).log();
    const torch::Tensor logp = x - log_sum;
    const torch::Tensor stats = torch::cat({shift, log_sum / std::log(2.0)}, 1);
    torch::Tensor picked = logp.gather(1, tokens.clamp(0, vocab - 1));
    picked = picked.masked_fill(tokens < 0, 0.0).masked_fill(tokens >= vocab, std::numeric_limits<float>::quiet_NaN());
    const torch::Tensor p = logp.exp();
    const torch::Tensor h = entropy ? -torch::where(p == 0, torch::zeros_like(p), p * logp).sum(1)
                                    : torch::empty({0}, wide.options());
    if (top == 0) {
        return {picked, stats, h, torch::empty({0, 0}, wide.options()), torch::empty({0, 0}, tokens.options())};
    }
    const torch::Tensor order = std::get<1>(wide.sort(/*stable=*/true, 1, /*descending=*/true)).slice(1, 0, top);
    return {picked, stats, h, logp.gather(1, order), order.contiguous()};
}

torch::Tensor token_logprobs_backward_cpu(const torch::Tensor& logits, const torch::Tensor& tokens, double scale,
                                          const torch::Tensor& stats, const torch::Tensor& entropy,
                                          const std::optional<torch::Tensor>& grad_logprobs,
                                          const std::optional<torch::Tensor>& grad_entropy) {
    check_logits(logits, tokens, scale);
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    const torch::Tensor wide = logits.to(torch::kFloat32);
    const torch::Tensor logp = (wide - stats.slice(1, 0, 1)) * scale - stats.slice(1, 1, 2) * std::log(2.0);
    const torch::Tensor p = logp.exp();
    torch::Tensor held;
    torch::Tensor grad = torch::zeros_like(p);
    torch::Tensor padding = (tokens < 0).all(1, true);  // of rows that have no gradient, whatever they hold
    if (gradient(grad_entropy, logits, {rows}, "grad_entropy", held) != nullptr) {
        const torch::Tensor kept = torch::where(p == 0, torch::zeros_like(p), logp);
        grad -= held.unsqueeze(1) * p * (kept + entropy.unsqueeze(1));
        padding = padding & (held == 0).unsqueeze(1);
    }
    if (gradient(grad_logprobs, logits, tokens.sizes(), "grad_logprobs", held) != nullptr) {
        torch::Tensor g = held.masked_fill(tokens < 0, 0.0);
        g = g.masked_fill(tokens >= vocab, std::numeric_limits<float>::quiet_NaN());
        grad -= g.sum(1, true) * p;
        grad.scatter_add_(1, tokens.clamp(0, vocab - 1), g);
    }
    return (scale * grad.masked_fill_(padding, 0.0)).to(logits.scalar_type());
}

// ---- pages of a paged cache ------------------------------------------------

void check_ints(const torch::Tensor& t, int64_t dim, const torch::Tensor& like, const char* name) {
    TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimensions, got ", t.dim());
    TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be int32, got ", t.scalar_type());
    check_contiguous(t, name);
    check_same_device(like, t, name);
}

/// Caches as the C ABI takes them: pointers, and the bytes of a page.
struct CacheList {
    std::vector<void*> pointers;
    int64_t page_bytes = 0;
    int64_t pages = 0;
    int64_t block = 0;
};

CacheList cache_list(at::TensorList caches, bool by_token) {
    TORCH_CHECK(!caches.empty(), "caches must name at least one tensor");
    const torch::Tensor& first = caches[0];
    TORCH_CHECK(first.dim() >= (by_token ? 2 : 1), "caches must be [pages, block, ...], got ", first.sizes());
    CacheList list;
    list.pages = first.size(0);
    list.block = first.dim() > 1 ? first.size(1) : 1;
    for (const torch::Tensor& t : caches) {
        check_contiguous(t, "a cache");
        check_same_device(first, t, "a cache");
        TORCH_CHECK(t.sizes() == first.sizes() && t.scalar_type() == first.scalar_type(),
                    "caches differ in shape or dtype: ", t.sizes(), " and ", first.sizes());
        list.pointers.push_back(t.data_ptr());
    }
    list.page_bytes = list.pages > 0 ? first.numel() / list.pages * first.element_size() : 0;
    return list;
}

/// Counts a write for autograd's saved-tensor checks, as the mutating
/// operators of torch do.
void mark_written(const torch::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

torch::Tensor page_workspace(const torch::Tensor& like, int64_t pages, int64_t sequences, int64_t count) {
    const size_t bytes = cf_cache_workspace_bytes(pages, sequences, count);
    return torch::empty({static_cast<int64_t>(bytes)}, like.options().dtype(torch::kUInt8));
}

void check_state(const torch::Tensor& counts, const torch::Tensor& tables, const torch::Tensor& context) {
    check_ints(counts, 1, counts, "ref_counts");
    check_ints(tables, 2, counts, "block_tables");
    check_ints(context, 1, counts, "context_lens");
    TORCH_CHECK(tables.size(0) == context.size(0), "block_tables has ", tables.size(0), " rows but context_lens ",
                context.size(0));
}

uint32_t* entries(const torch::Tensor& tables) { return reinterpret_cast<uint32_t*>(tables.data_ptr<int32_t>()); }

torch::Tensor cache_copy_hip(at::TensorList caches, const torch::Tensor& src, const torch::Tensor& dst) {
    const CacheList list = cache_list(caches, false);
    check_ints(src, 1, caches[0], "src");
    check_ints(dst, 1, caches[0], "dst");
    TORCH_CHECK(src.size(0) == dst.size(0), "src and dst differ in length: ", src.size(0), " and ", dst.size(0));
    const at::DeviceGuard guard(src.device());
    torch::Tensor status = torch::empty_like(src);
    if (src.numel() == 0) return status;
    if (list.page_bytes == 0) return status.fill_(list.pages == 0 ? 1 : 0);
    const torch::Tensor workspace = page_workspace(src, list.pages, 0, src.size(0));
    check_status(cf_cache_copy(list.pointers.data(), list.pointers.size(), list.page_bytes, list.pages,
                               src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(), src.size(0),
                               status.data_ptr<int32_t>(), workspace.data_ptr(), workspace.numel(), stream_for(src)));
    for (const torch::Tensor& t : caches) mark_written(t);
    return status;
}

torch::Tensor cache_fork_hip(at::TensorList caches, const torch::Tensor& counts, const torch::Tensor& tables,
                             const torch::Tensor& context, const torch::Tensor& parents,
                             const torch::Tensor& children) {
    const CacheList list = cache_list(caches, true);
    check_state(counts, tables, context);
    check_same_device(counts, caches[0], "a cache");
    check_ints(parents, 1, counts, "parents");
    check_ints(children, 1, counts, "children");
    TORCH_CHECK(counts.size(0) == list.pages, "ref_counts counts ", counts.size(0), " pages, the caches hold ",
                list.pages);
    TORCH_CHECK(parents.size(0) == children.size(0), "parents and children differ in length: ", parents.size(0),
                " and ", children.size(0));
    const at::DeviceGuard guard(counts.device());
    torch::Tensor status = torch::empty_like(parents);
    if (parents.numel() == 0) return status;
    if (list.page_bytes == 0 || tables.numel() == 0) return status.fill_(1);
    const torch::Tensor workspace = page_workspace(counts, list.pages, tables.size(0), parents.size(0));
    check_status(cf_cache_fork(list.pointers.data(), list.pointers.size(), list.page_bytes,
                               counts.data_ptr<int32_t>(), entries(tables), context.data_ptr<int32_t>(), list.pages,
                               list.block, tables.size(0), tables.size(1), parents.data_ptr<int32_t>(),
                               children.data_ptr<int32_t>(), parents.size(0), status.data_ptr<int32_t>(),
                               workspace.data_ptr(), workspace.numel(), stream_for(counts)));
    for (const torch::Tensor& t : caches) mark_written(t);
    for (const torch::Tensor* t : {&counts, &tables, &context}) mark_written(*t);
    return status;
}

torch::Tensor cache_extend_hip(const torch::Tensor& counts, const torch::Tensor& tables, const torch::Tensor& context,
                               const torch::Tensor& sequences, int64_t block, int64_t tokens) {
    check_state(counts, tables, context);
    check_ints(sequences, 1, counts, "sequences");
    TORCH_CHECK(block > 0 && tokens > 0, "block_size and tokens must be positive, got ", block, " and ", tokens);
    const at::DeviceGuard guard(counts.device());
    torch::Tensor slots = torch::empty({sequences.size(0), tokens}, sequences.options().dtype(torch::kInt64));
    if (sequences.numel() == 0) return slots;
    if (tables.numel() == 0 || counts.numel() == 0) return slots.fill_(-1);
    const torch::Tensor workspace = page_workspace(counts, counts.size(0), tables.size(0), sequences.size(0));
    check_status(cf_cache_extend(counts.data_ptr<int32_t>(), entries(tables), context.data_ptr<int32_t>(),
                                 counts.size(0), block, tables.size(0), tables.size(1), sequences.data_ptr<int32_t>(),
                                 sequences.size(0), tokens, slots.data_ptr<int64_t>(), workspace.data_ptr(),
                                 workspace.numel(), stream_for(counts)));
    for (const torch::Tensor* t : {&counts, &tables, &context}) mark_written(*t);
    return slots;
}

void cache_release_hip(const torch::Tensor& counts, const torch::Tensor& tables, const torch::Tensor& context,
                       const torch::Tensor& sequences, int64_t block) {
    check_state(counts, tables, context);
    check_ints(sequences, 1, counts, "sequences");
    TORCH_CHECK(block > 0, "block_size must be positive, got ", block);
    const at::DeviceGuard guard(counts.device());
    if (sequences.numel() == 0 || tables.numel() == 0 || counts.numel() == 0) return;
    check_status(cf_cache_release(counts.data_ptr<int32_t>(), entries(tables), context.data_ptr<int32_t>(),
                                  counts.size(0), block, tables.size(0), tables.size(1),
                                  sequences.data_ptr<int32_t>(), sequences.size(0), stream_for(counts)));
    for (const torch::Tensor* t : {&counts, &context}) mark_written(*t);
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> cache_compact_hip(at::TensorList caches,
                                                                          const torch::Tensor& counts,
                                                                          const torch::Tensor& tables,
                                                                          const torch::Tensor& context) {
    const CacheList list = cache_list(caches, true);
    check_state(counts, tables, context);
    check_same_device(counts, caches[0], "a cache");
    TORCH_CHECK(counts.size(0) == list.pages, "ref_counts counts ", counts.size(0), " pages, the caches hold ",
                list.pages);
    const at::DeviceGuard guard(counts.device());
    torch::Tensor new_counts = torch::empty_like(counts);
    torch::Tensor new_tables = torch::empty_like(tables);
    torch::Tensor live = torch::empty({1}, counts.options());
    if (list.pages == 0 || list.block == 0) {
        new_tables.copy_(tables);
        return {new_counts.copy_(counts), new_tables, live.fill_(0)};
    }
    const torch::Tensor workspace = page_workspace(counts, list.pages, tables.size(0), 0);
    check_status(cf_cache_compact(list.pointers.data(), list.page_bytes > 0 ? list.pointers.size() : 0,
                                  list.page_bytes, counts.data_ptr<int32_t>(), entries(tables),
                                  context.data_ptr<int32_t>(), list.pages, list.block, tables.size(0), tables.size(1),
                                  new_counts.data_ptr<int32_t>(), entries(new_tables), live.data_ptr<int32_t>(),
                                  workspace.data_ptr(), workspace.numel(), stream_for(counts)));
    for (const torch::Tensor& t : caches) mark_written(t);
    return {new_counts, new_tables, live};
}

// ---- paged attention behind shared prompts -----------------------------------

void check_shared(const torch::Tensor& query, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                  const torch::Tensor& starts, const torch::Tensor& prefix, const torch::Tensor& tables,
                  const torch::Tensor& context) {
    TORCH_CHECK(query.dim() == 3, "query must be [sequences, heads, head_dim], got ", query.dim(), " dimensions");
    TORCH_CHECK(k_cache.dim() == 4, "k_cache must be [pages, block, kv_heads, head_dim], got ", k_cache.dim(),
                " dimensions");
    TORCH_CHECK(v_cache.sizes() == k_cache.sizes(), "v_cache has shape ", v_cache.sizes(), " but k_cache ",
                k_cache.sizes());
    for (const auto& [t, name] : {std::pair<const torch::Tensor*, const char*>{&k_cache, "k_cache"},
                                  {&v_cache, "v_cache"}}) {
        check_contiguous(*t, name);
        check_same_device(query, *t, name);
        TORCH_CHECK(t->scalar_type() == query.scalar_type(), name, " has dtype ", t->scalar_type(),
                    " but query has ", query.scalar_type());
    }
    check_contiguous(query, "query");
    TORCH_CHECK(k_cache.size(3) == query.size(2), "the cache's head size is ", k_cache.size(3), " but the query's ",
                query.size(2));
    TORCH_CHECK(k_cache.size(2) > 0 && query.size(1) % k_cache.size(2) == 0, query.size(1),
                " heads are not a multiple of ", k_cache.size(2), " KV heads");
    check_ints(tables, 2, query, "block_tables");
    check_ints(context, 1, query, "context_lens");
    check_ints(starts, 1, query, "group_starts");
    check_ints(prefix, 1, query, "prefix_lens");
    TORCH_CHECK(tables.size(0) == query.size(0) && context.size(0) == query.size(0),
                "block_tables and context_lens must have a row for each of ", query.size(0), " sequences");
    TORCH_CHECK(starts.size(0) == prefix.size(0) + 1, "group_starts must have one entry more than prefix_lens");
}

torch::Tensor paged_attention_shared_hip(const torch::Tensor& query, const torch::Tensor& k_cache,
                                         const torch::Tensor& v_cache, const torch::Tensor& starts,
                                         const torch::Tensor& prefix, const torch::Tensor& tables,
                                         const torch::Tensor& context, double scale) {
    check_shared(query, k_cache, v_cache, starts, prefix, tables, context);
    const at::DeviceGuard guard(query.device());
    torch::Tensor out = torch::empty_like(query);
    if (query.numel() == 0) return out;
    if (k_cache.size(0) == 0 || k_cache.size(1) == 0 || tables.size(1) == 0) return out.zero_();
    const cf_dtype dtype = to_cf(query, "query");
    const int64_t sequences = query.size(0), heads = query.size(1), dim = query.size(2);
    const int64_t groups = prefix.size(0), kv_heads = k_cache.size(2), block = k_cache.size(1);
    const size_t bytes = cf_paged_attention_shared_workspace_bytes(dtype, sequences, groups, heads, kv_heads, dim,
                                                                   block, tables.size(1));
    const torch::Tensor workspace =
        torch::empty({static_cast<int64_t>(bytes)}, query.options().dtype(torch::kUInt8));
    check_status(cf_paged_attention_shared(
        query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), starts.data_ptr<int32_t>(),
        prefix.data_ptr<int32_t>(), reinterpret_cast<const uint32_t*>(tables.data_ptr<int32_t>()),
        context.data_ptr<int32_t>(), out.data_ptr(), dtype, k_cache.size(0), sequences, groups, heads, kv_heads, dim,
        block, tables.size(1), static_cast<float>(scale), workspace.data_ptr(), bytes, stream_for(query)));
    return out;
}

/// Sequence by sequence over its own table: sharing changes no result.
torch::Tensor paged_attention_shared_cpu(const torch::Tensor& query, const torch::Tensor& k_cache,
                                         const torch::Tensor& v_cache, const torch::Tensor& starts,
                                         const torch::Tensor& prefix, const torch::Tensor& tables,
                                         const torch::Tensor& context, double scale) {
    check_shared(query, k_cache, v_cache, starts, prefix, tables, context);
    torch::Tensor out = torch::zeros_like(query);
    const int64_t pages = k_cache.size(0), block = k_cache.size(1), kv_heads = k_cache.size(2), dim = k_cache.size(3);
    if (query.numel() == 0 || pages == 0 || block == 0 || tables.size(1) == 0) return out;
    const torch::Tensor keys = k_cache.reshape({pages * block, kv_heads, dim});
    const torch::Tensor vals = v_cache.reshape({pages * block, kv_heads, dim});
    for (int64_t s = 0; s < query.size(0); ++s) {
        const int64_t length = std::min<int64_t>(std::max(context[s].item<int32_t>(), 0), tables.size(1) * block);
        const torch::Tensor token = torch::arange(length);
        const torch::Tensor page = tables[s].to(torch::kInt64).index({token.floor_divide(block)});
        const torch::Tensor there = (page >= 0) & (page < pages);
        const torch::Tensor slot = (page * block + token.remainder(block)).index({there});
        if (slot.numel() == 0) continue;
        const torch::Tensor k = keys.index({slot}).to(torch::kFloat32).permute({1, 2, 0});
        const torch::Tensor v = vals.index({slot}).to(torch::kFloat32).permute({1, 0, 2});
        const torch::Tensor q = query[s].to(torch::kFloat32).view({kv_heads, -1, dim});
        const torch::Tensor scores = torch::matmul(q, k) * scale;
        torch::Tensor o = torch::matmul(torch::softmax(scores, -1), v);
        const torch::Tensor none = (scores == -std::numeric_limits<float>::infinity()).all(-1, true);
        o = o.masked_fill(none, 0.0);
        out[s].copy_(o.view({query.size(1), dim}));
    }
    return out;
}

}  // namespace

// ---- direct entry for ordinary GPU calls (the rules: torch_ops_common.hpp) ------

/// The autograd function of cuda_force_amd/autograd.py as a native node: the
/// same saved tensors and kernels, without the interpreter in either direction.
/// Outputs: log probabilities shaped as the tokens, then the entropy, then the
/// likeliest tokens' two, where asked for.
struct TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits,
                                                  const at::Tensor& tokens, double scale, bool entropy, int64_t top) {
        const at::Tensor given = tokens.dim() == 1 ? tokens.unsqueeze(1) : tokens;
        auto [logprobs, stats, h, top_logprobs, top_tokens] =
            logprobs_of(logits, given, tokens.sizes(), scale, entropy, top);
        torch::autograd::variable_list out{logprobs};
        if (entropy) out.push_back(h);
        if (top > 0) {
            out.push_back(top_logprobs);
            out.push_back(top_tokens);
            ctx->mark_non_differentiable({top_logprobs, top_tokens});
        }
        ctx->save_for_backward({logits, given, stats, h});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["entropy"] = entropy;
        ctx->set_materialize_grads(false);
        return out;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &logits = saved[0], &tokens = saved[1], &stats = saved[2], &h = saved[3];
        const double scale = ctx->saved_data["scale"].toDouble();
        std::optional<at::Tensor> g, gh;
        if (grads[0].defined()) g = grads[0].dim() == 1 ? grads[0].unsqueeze(1) : grads[0];
        if (ctx->saved_data["entropy"].toBool() && grads[1].defined()) gh = grads[1];
        at::Tensor grad;
        if (g || gh) {
            // What saved-tensor hooks return, a batched gradient, a mode
            // entered since, and a recorded backward (whose result the
            // dispatcher's entry refuses to differentiate) go through the
            // dispatcher.
            const bool direct = !at::GradMode::is_enabled() && ordinary_context() && plain_gpu(logits) &&
                                plain_gpu(tokens) && plain_gpu(stats) && plain_gpu(h) && (!g || plain_gpu(*g)) &&
                                (!gh || plain_gpu(*gh));
            if (direct) {
                grad = token_logprobs_backward_hip(logits, tokens, scale, stats, h, g, gh);
            } else {
                static const auto op = c10::Dispatcher::singleton()
                                           .findSchemaOrThrow("cudaforge::token_logprobs_backward", "")
                                           .typed<at::Tensor(const at::Tensor&, const at::Tensor&, double,
                                                             const at::Tensor&, const at::Tensor&,
                                                             const std::optional<at::Tensor>&,
                                                             const std::optional<at::Tensor>&)>();
                grad = op.call(logits, tokens, scale, stats, h, g, gh);
            }
        }
        return {grad, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

/// Calls above these go the general way, which names the limit.
constexpr int64_t kLogprobsTokens = 1024;
constexpr int64_t kLogprobsTop = 64;

py::object try_token_logprobs(py::handle logits_, py::handle tokens_, py::handle scale_, py::handle entropy_,
                              py::handle top_) {
    if (!THPVariable_CheckTypeExact(Py_TYPE(logits_.ptr()))) return py::none();
    const at::Tensor& logits = THPVariable_Unpack(logits_.ptr());
    const at::Tensor* tokens = ordinary(tokens_);
    const std::optional<double> scale = plain_double(scale_);
    const std::optional<int64_t> top = plain_int(top_);
    if (!plain_gpu(logits) || tokens == nullptr || !scale || !top || !PyBool_Check(entropy_.ptr()) ||
        !ordinary_context()) {
        return py::none();
    }
    const bool entropy = entropy_.ptr() == Py_True;
    if (!kernel_dtype(logits.scalar_type()) || tokens->scalar_type() != torch::kInt64 ||
        tokens->device() != logits.device() || logits.dim() != 2 || logits.numel() == 0 || logits.stride(1) != 1 ||
        (logits.size(0) > 1 && logits.stride(0) < logits.size(1)) || tokens->dim() < 1 || tokens->dim() > 2 ||
        tokens->size(0) != logits.size(0) || (tokens->dim() == 2 && tokens->size(1) > kLogprobsTokens) ||
        !(*scale > 0 && *scale < 1e29) || *top < 0 || *top > std::min(kLogprobsTop, logits.size(1))) {
        return py::none();
    }
    const bool grad = grad_needed({&logits});
    at::Tensor logprobs, h, top_logprobs, top_tokens;
    {
        py::gil_scoped_release no_gil;
        if (grad) {
            torch::autograd::variable_list out = TokenLogprobs::apply(logits, *tokens, *scale, entropy, *top);
            logprobs = out[0];
            if (entropy) h = out[1];
            if (*top > 0) {
                top_logprobs = out[out.size() - 2];
                top_tokens = out.back();
            }
        } else {
            std::tie(logprobs, std::ignore, h, top_logprobs, top_tokens) = logprobs_of(
                logits, tokens->dim() == 1 ? tokens->unsqueeze(1) : *tokens, tokens->sizes(), *scale, entropy, *top);
        }
    }
    return py::make_tuple(wrap(logprobs), entropy ? wrap(h) : py::none(), *top > 0 ? wrap(top_logprobs) : py::none(),
                          *top > 0 ? wrap(top_tokens) : py::none());
}

/// A list or tuple of ordinary tensors without gradients, or nothing.
std::optional<std::vector<at::Tensor>> ordinary_list(py::handle object) {
    if (!PyList_CheckExact(object.ptr()) && !PyTuple_CheckExact(object.ptr())) return std::nullopt;
    std::vector<at::Tensor> list;
    for (const py::handle item : py::reinterpret_borrow<py::sequence>(object)) {
        const at::Tensor* t = ordinary(item);
        if (t == nullptr || t->requires_grad()) return std::nullopt;
        if (!list.empty() && (t->sizes() != list[0].sizes() || t->scalar_type() != list[0].scalar_type() ||
                              t->device() != list[0].device())) {
            return std::nullopt;
        }
        list.push_back(*t);
    }
    return list.empty() ? std::nullopt : std::make_optional(std::move(list));
}

/// Ordinary int32 tensors of the given dimensions, all on one device.
bool ordinary_ints(std::initializer_list<std::pair<const at::Tensor*, int64_t>> tensors) {
    const at::Tensor* first = tensors.begin()->first;
    for (const auto& [t, dim] : tensors) {
        if (t == nullptr || t->scalar_type() != torch::kInt32 || t->dim() != dim || t->device() != first->device()) {
            return false;
        }
    }
    return true;
}

py::object try_cache_copy(py::handle caches_, py::handle src_, py::handle dst_) {
    const at::Tensor* src = ordinary(src_);
    const at::Tensor* dst = ordinary(dst_);
    if (!ordinary_context() || !ordinary_ints({{src, 1}, {dst, 1}}) || src->size(0) != dst->size(0)) return py::none();
    const auto caches = ordinary_list(caches_);
    if (!caches || (*caches)[0].device() != src->device() || (*caches)[0].dim() < 1) return py::none();
    at::Tensor status;
    {
        py::gil_scoped_release no_gil;
        status = cache_copy_hip(*caches, *src, *dst);
    }
    return wrap(status);
}

py::object try_cache_fork(py::handle caches_, py::handle counts_, py::handle tables_, py::handle context_,
                          py::handle parents_, py::handle children_) {
    const at::Tensor* counts = ordinary(counts_);
    const at::Tensor* tables = ordinary(tables_);
    const at::Tensor* context = ordinary(context_);
    const at::Tensor* parents = ordinary(parents_);
    const at::Tensor* children = ordinary(children_);
    if (!ordinary_context() ||
        !ordinary_ints({{counts, 1}, {tables, 2}, {context, 1}, {parents, 1}, {children, 1}}) ||
        tables->size(0) != context->size(0) || parents->size(0) != children->size(0)) {
        return py::none();
    }
    const auto caches = ordinary_list(caches_);
    if (!caches || (*caches)[0].device() != counts->device() || (*caches)[0].dim() < 2 ||
        (*caches)[0].size(0) != counts->size(0)) {
        return py::none();
    }
    at::Tensor status;
    {
        py::gil_scoped_release no_gil;
        status = cache_fork_hip(*caches, *counts, *tables, *context, *parents, *children);
    }
    return wrap(status);
}

py::object try_cache_extend(py::handle counts_, py::handle tables_, py::handle context_, py::handle sequences_,
                            py::handle block_, py::handle tokens_) {
    const at::Tensor* counts = ordinary(counts_);
    const at::Tensor* tables = ordinary(tables_);
    const at::Tensor* context = ordinary(context_);
    const at::Tensor* sequences = ordinary(sequences_);
    const std::optional<int64_t> block = plain_int(block_);
    const std::optional<int64_t> tokens = plain_int(tokens_);
    if (!ordinary_context() || !ordinary_ints({{counts, 1}, {tables, 2}, {context, 1}, {sequences, 1}}) ||
        tables->size(0) != context->size(0) || !block || !tokens || *block <= 0 || *tokens <= 0) {
        return py::none();
    }
    at::Tensor slots;
    {
        py::gil_scoped_release no_gil;
        slots = cache_extend_hip(*counts, *tables, *context, *sequences, *block, *tokens);
    }
    return wrap(slots);
}

/// True when the call was taken.
bool try_cache_release(py::handle counts_, py::handle tables_, py::handle context_, py::handle sequences_,
                       py::handle block_) {
    const at::Tensor* counts = ordinary(counts_);
    const at::Tensor* tables = ordinary(tables_);
    const at::Tensor* context = ordinary(context_);
    const at::Tensor* sequences = ordinary(sequences_);
    const std::optional<int64_t> block = plain_int(block_);
    if (!ordinary_context() || !ordinary_ints({{counts, 1}, {tables, 2}, {context, 1}, {sequences, 1}}) ||
        tables->size(0) != context->size(0) || !block || *block <= 0) {
        return false;
    }
    py::gil_scoped_release no_gil;
    cache_release_hip(*counts, *tables, *context, *sequences, *block);
    return true;
}

py::object try_cache_compact(py::handle caches_, py::handle counts_, py::handle tables_, py::handle context_) {
    const at::Tensor* counts = ordinary(counts_);
    const at::Tensor* tables = ordinary(tables_);
    const at::Tensor* context = ordinary(context_);
    if (!ordinary_context() || !ordinary_ints({{counts, 1}, {tables, 2}, {context, 1}}) ||
        tables->size(0) != context->size(0)) {
        return py::none();
    }
    const auto caches = ordinary_list(caches_);
    if (!caches || (*caches)[0].device() != counts->device() || (*caches)[0].dim() < 2 ||
        (*caches)[0].size(0) != counts->size(0)) {
        return py::none();
    }
    std::tuple<at::Tensor, at::Tensor, at::Tensor> out;
    {
        py::gil_scoped_release no_gil;
        out = cache_compact_hip(*caches, *counts, *tables, *context);
    }
    return py::make_tuple(wrap(std::get<0>(out)), wrap(std::get<1>(out)), wrap(std::get<2>(out)));
}

py::object try_paged_attention_shared(py::handle query_, py::handle k_, py::handle v_, py::handle starts_,
                                      py::handle prefix_, py::handle tables_, py::handle context_,
                                      py::handle scale_) {
    const at::Tensor* query = ordinary(query_);
    const at::Tensor* k = ordinary(k_);
    const at::Tensor* v = ordinary(v_);
    const at::Tensor* starts = ordinary(starts_);
    const at::Tensor* prefix = ordinary(prefix_);
    const at::Tensor* tables = ordinary(tables_);
    const at::Tensor* context = ordinary(context_);
    const std::optional<double> scale = plain_double(scale_);
    if (starts == nullptr || prefix == nullptr || tables == nullptr || context == nullptr || !scale ||
        !ordinary_context() || !ordinary_set({query, k, v})) {
        return py::none();
    }
    if (query->dim() != 3 || k->dim() != 4 || v->sizes() != k->sizes() || k->size(3) != query->size(2) ||
        query->size(2) > 1024 || query->size(1) % k->size(2) != 0 || starts->dim() != 1 || prefix->dim() != 1 ||
        tables->dim() != 2 || context->dim() != 1 || starts->size(0) != prefix->size(0) + 1 ||
        tables->size(0) != query->size(0) || context->size(0) != query->size(0)) {
        return py::none();
    }
    for (const at::Tensor* t : {starts, prefix, tables, context}) {
        if (t->scalar_type() != torch::kInt32 || t->device() != query->device()) return py::none();
    }
    at::Tensor out;
    {
        py::gil_scoped_release no_gil;
        out = paged_attention_shared_hip(*query, *k, *v, *starts, *prefix, *tables, *context, *scale);
    }
    return wrap(out);
}

void bind_generation(py::module_& m) {
    m.def("try_cache_copy", torch::wrap_pybind_function(&try_cache_copy));
    m.def("try_cache_fork", torch::wrap_pybind_function(&try_cache_fork));
    m.def("try_cache_extend", torch::wrap_pybind_function(&try_cache_extend));
    m.def("try_cache_release", torch::wrap_pybind_function(&try_cache_release));
    m.def("try_cache_compact", torch::wrap_pybind_function(&try_cache_compact));
    m.def("try_paged_attention_shared", torch::wrap_pybind_function(&try_paged_attention_shared));
    m.def("try_token_logprobs", torch::wrap_pybind_function(&try_token_logprobs));
}

}  // namespace cudaforge_amd

TORCH_LIBRARY_FRAGMENT(cudaforge, m) {
    m.def("cache_copy(Tensor(a!)[] caches, Tensor src, Tensor dst) -> Tensor");
    m.def(
        "cache_fork(Tensor(a!)[] caches, Tensor(b!) ref_counts, Tensor(c!) block_tables, Tensor(d!) context_lens, "
        "Tensor parents, Tensor children) -> Tensor");
    m.def(
        "cache_extend(Tensor(a!) ref_counts, Tensor(b!) block_tables, Tensor(c!) context_lens, Tensor sequences, "
        "int block_size, int tokens) -> Tensor");
    m.def(
        "cache_release(Tensor(a!) ref_counts, Tensor block_tables, Tensor(b!) context_lens, Tensor sequences, "
        "int block_size) -> ()");
    m.def(
        "cache_compact(Tensor(a!)[] caches, Tensor ref_counts, Tensor block_tables, Tensor context_lens) "
        "-> (Tensor, Tensor, Tensor)");
    m.def(
        "paged_attention_shared(Tensor query, Tensor k_cache, Tensor v_cache, Tensor group_starts, "
        "Tensor prefix_lens, Tensor block_tables, Tensor context_lens, float scale) -> Tensor");
    m.def(
        "token_logprobs(Tensor logits, Tensor tokens, float scale, bool entropy, int top) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def(
        "token_logprobs_backward(Tensor logits, Tensor tokens, float scale, Tensor stats, Tensor entropy, "
        "Tensor? grad_logprobs, Tensor? grad_entropy) -> Tensor");
}

// As in torch_ops.cpp: differentiating the operators themselves raises;
// the Python layer has the differentiable form.
TORCH_LIBRARY_IMPL(cudaforge, Autograd, m) {
    for (const char* name : {"paged_attention_shared", "token_logprobs", "token_logprobs_backward"}) {
        m.impl(name, torch::autograd::autogradNotImplementedFallback());
    }
}

// The page operators' CPU implementations are the Python layer's
// (paged_cache.py): plain loops over the tables.
TORCH_LIBRARY_IMPL(cudaforge, CPU, m) {
    using namespace cudaforge_amd;
    m.impl("paged_attention_shared", &paged_attention_shared_cpu);
    m.impl("token_logprobs", &token_logprobs_cpu);
    m.impl("token_logprobs_backward", &token_logprobs_backward_cpu);
}

TORCH_LIBRARY_IMPL(cudaforge, CUDA, m) {
    using namespace cudaforge_amd;
    m.impl("cache_copy", &cache_copy_hip);
    m.impl("cache_fork", &cache_fork_hip);
    m.impl("cache_extend", &cache_extend_hip);
    m.impl("cache_release", &cache_release_hip);
    m.impl("cache_compact", &cache_compact_hip);
    m.impl("paged_attention_shared", &paged_attention_shared_hip);
    m.impl("token_logprobs", &token_logprobs_hip);
    m.impl("token_logprobs_backward", &token_logprobs_backward_hip);
}
