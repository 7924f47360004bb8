// Dispatcher registration of the operators of serving in 8 bits: storing into a
// paged cache and reading it back, attention of chunks of new tokens over it,
// and products of 8-bit integers. Same conventions as torch_ops.cpp; the CPU
// implementations are the Python layer's plain forms.
#include "torch_ops_common.hpp"

namespace cudaforge_amd {
namespace {

cf_cache_format format_of(const torch::Tensor& cache, const char* name) {
    switch (cache.scalar_type()) {
        case torch::kInt8:
            return CF_CACHE_INT8;
        case torch::kFloat8_e4m3fn:
            return CF_CACHE_E4M3;
        case torch::kFloat32:
        case torch::kBFloat16:
        case torch::kFloat16:
            return CF_CACHE_PLAIN;
        default:
            TORCH_CHECK(false, name, " has dtype ", cache.scalar_type(),
                        ", which no cache holds (float32, bfloat16, float16, int8 or float8_e4m3fn)");
    }
}

/// The caches and, for 8-bit ones, their scales; `like` names the device.
cf_cache_format check_held(const torch::Tensor& like, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                           const std::optional<torch::Tensor>& k_scales, const std::optional<torch::Tensor>& v_scales) {
    TORCH_CHECK(k_cache.dim() == 4, "k_cache must be [pages, block, kv_heads, head_dim], got ", k_cache.dim(),
                " dimensions");
    TORCH_CHECK(v_cache.sizes() == k_cache.sizes() && v_cache.scalar_type() == k_cache.scalar_type(),
                "v_cache is ", v_cache.sizes(), " of ", v_cache.scalar_type(), " but k_cache ", k_cache.sizes(), " of ",
                k_cache.scalar_type());
    const cf_cache_format format = format_of(k_cache, "k_cache");
    for (const auto& [t, name] :
         {std::pair<const torch::Tensor*, const char*>{&k_cache, "k_cache"}, {&v_cache, "v_cache"}}) {
        check_contiguous(*t, name);
        check_same_device(like, *t, name);
    }
    TORCH_CHECK(k_scales.has_value() == (format != CF_CACHE_PLAIN) && v_scales.has_value() == k_scales.has_value(),
                "k_scales and v_scales are given for 8-bit caches, and for those alone");
    if (format == CF_CACHE_PLAIN) return format;
    for (const auto& [t, name] :
         {std::pair<const torch::Tensor*, const char*>{&*k_scales, "k_scales"}, {&*v_scales, "v_scales"}}) {
        TORCH_CHECK(t->sizes() == k_cache.sizes().slice(0, 3), name, " must be [pages, block, kv_heads], got ",
                    t->sizes());
        TORCH_CHECK(t->scalar_type() == torch::kFloat32, name, " must be float32, got ", t->scalar_type());
        check_contiguous(*t, name);
        check_same_device(like, *t, name);
    }
    return format;
}

float* scales_of(const std::optional<torch::Tensor>& t) { return t ? t->data_ptr<float>() : nullptr; }

void check_slots(const torch::Tensor& slots, const torch::Tensor& like) {
    TORCH_CHECK(slots.dim() == 1, "slots must be [tokens], got ", slots.sizes());
    TORCH_CHECK(slots.scalar_type() == torch::kInt64, "slots must be int64, got ", slots.scalar_type());
    check_contiguous(slots, "slots");
    check_same_device(like, slots, "slots");
}

// ---- storing into a paged cache ------------------------------------------------

/// Whether a tensor of any strides has memory in common with a dense one.
bool shares_memory(const torch::Tensor& x, const torch::Tensor& dense) {
    if (!x.is_alias_of(dense) || x.numel() == 0 || dense.numel() == 0) return false;
    int64_t last = 1;
    for (int64_t d = 0; d < x.dim(); ++d) last += (x.size(d) - 1) * x.stride(d);
    const char* from = static_cast<const char*>(x.data_ptr());
    const char* to = static_cast<const char*>(dense.data_ptr());
    return from < to + dense.nbytes() && to < from + last * x.element_size();
}

void cache_write_hip(const torch::Tensor& keys, const torch::Tensor& values, const torch::Tensor& k_cache,
                     const torch::Tensor& v_cache, const torch::Tensor& slots,
                     const std::optional<torch::Tensor>& k_scales, const std::optional<torch::Tensor>& v_scales) {
    const cf_cache_format format = check_held(keys, k_cache, v_cache, k_scales, v_scales);
    const int64_t kv_heads = k_cache.size(2), dim = k_cache.size(3);
    check_slots(slots, keys);
    for (const auto& [t, name] : {std::pair<const torch::Tensor*, const char*>{&keys, "keys"}, {&values, "values"}}) {
        TORCH_CHECK(t->dim() == 3 && t->size(0) == slots.size(0) && t->size(1) == kv_heads && t->size(2) == dim, name,
                    " must be [", slots.size(0), ", ", kv_heads, ", ", dim, "], got ", t->sizes());
        TORCH_CHECK(dim <= 1 || t->stride(2) == 1, name, " must be dense along head_dim");
        TORCH_CHECK(t->scalar_type() == keys.scalar_type(), "keys and values differ in dtype");
        TORCH_CHECK(format != CF_CACHE_PLAIN || t->scalar_type() == k_cache.scalar_type(), name, " has dtype ",
                    t->scalar_type(), " but the caches ", k_cache.scalar_type());
        check_same_device(keys, *t, name);
    }
    if (keys.numel() == 0 || k_cache.numel() == 0) return;
    const at::DeviceGuard guard(keys.device());
    // Rows of the caches themselves are read before any is written.
    auto apart = [&](const torch::Tensor& x) {
        const bool shares = shares_memory(x, k_cache) || shares_memory(x, v_cache) ||
                            (k_scales && shares_memory(x, *k_scales)) || (v_scales && shares_memory(x, *v_scales));
        return shares ? x.clone(at::MemoryFormat::Contiguous) : x;
    };
    const torch::Tensor k = apart(keys), v = apart(values);
    check_status(cf_cache_write(k.data_ptr(), v.data_ptr(), to_cf(keys, "keys"), keys.size(0), kv_heads, dim,
                                k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                                slots.data_ptr<int64_t>(), k_cache.data_ptr(), v_cache.data_ptr(), format,
                                scales_of(k_scales), scales_of(v_scales), k_cache.size(0) * k_cache.size(1),
                                stream_for(keys)));
    mark_written(k_cache);
    mark_written(v_cache);
    if (k_scales) mark_written(*k_scales);
    if (v_scales) mark_written(*v_scales);
}

std::tuple<torch::Tensor, torch::Tensor> cache_read_hip(const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                                                        const torch::Tensor& slots,
                                                        const std::optional<torch::Tensor>& k_scales,
                                                        const std::optional<torch::Tensor>& v_scales,
                                                        at::ScalarType dtype) {
    const cf_cache_format format = check_held(k_cache, k_cache, v_cache, k_scales, v_scales);
    check_slots(slots, k_cache);
    TORCH_CHECK(format != CF_CACHE_PLAIN || dtype == k_cache.scalar_type(), "a plain cache of ",
                k_cache.scalar_type(), " is read back as that, not as ", dtype);
    const at::DeviceGuard guard(k_cache.device());
    const auto shape = {slots.size(0), k_cache.size(2), k_cache.size(3)};
    torch::Tensor keys = torch::empty(shape, k_cache.options().dtype(dtype));
    torch::Tensor values = torch::empty(shape, k_cache.options().dtype(dtype));
    const cf_dtype type = to_cf(dtype);
    if (keys.numel() == 0) return {keys, values};
    if (k_cache.numel() == 0) return {keys.zero_(), values.zero_()};
    check_status(cf_cache_read(k_cache.data_ptr(), v_cache.data_ptr(), format, scales_of(k_scales),
                               scales_of(v_scales), k_cache.size(0) * k_cache.size(1), slots.data_ptr<int64_t>(),
                               slots.size(0), k_cache.size(2), k_cache.size(3), keys.data_ptr(), values.data_ptr(),
                               type, stream_for(k_cache)));
    return {keys, values};
}

// ---- paged attention of chunks of new tokens -----------------------------------

torch::Tensor paged_attention_chunk_hip(const torch::Tensor& query, const torch::Tensor& k_cache,
                                        const torch::Tensor& v_cache, const torch::Tensor& starts,
                                        const torch::Tensor& tables, const torch::Tensor& context,
                                        const std::optional<torch::Tensor>& k_scales,
                                        const std::optional<torch::Tensor>& v_scales, double scale) {
    TORCH_CHECK(query.dim() == 3, "query must be [tokens, heads, head_dim], got ", query.dim(), " dimensions");
    const cf_cache_format format = check_held(query, k_cache, v_cache, k_scales, v_scales);
    check_contiguous(query, "query");
    TORCH_CHECK(format != CF_CACHE_PLAIN || k_cache.scalar_type() == query.scalar_type(), "the caches have dtype ",
                k_cache.scalar_type(), " but query has ", query.scalar_type());
    TORCH_CHECK(k_cache.size(3) == query.size(2), "the cache's head size is ", k_cache.size(3), " but the query's ",
                query.size(2));
    TORCH_CHECK(k_cache.size(2) > 0 && query.size(1) % k_cache.size(2) == 0, query.size(1),
                " heads are not a multiple of ", k_cache.size(2), " KV heads");
    check_ints(starts, 1, query, "query_starts");
    check_ints(tables, 2, query, "block_tables");
    check_ints(context, 1, query, "context_lens");
    TORCH_CHECK(tables.size(0) == context.size(0) && starts.size(0) == context.size(0) + 1,
                "block_tables must have a row for each of ", context.size(0),
                " sequences, and query_starts one entry more");
    const at::DeviceGuard guard(query.device());
    torch::Tensor out = torch::empty_like(query);
    if (query.numel() == 0) return out;
    if (k_cache.size(0) == 0 || k_cache.size(1) == 0 || tables.numel() == 0) return out.zero_();
    const cf_dtype dtype = to_cf(query, "query");
    const int64_t tokens = query.size(0), heads = query.size(1), dim = query.size(2);
    const int64_t kv_heads = k_cache.size(2), block = k_cache.size(1), sequences = context.size(0);
    const size_t bytes = cf_paged_attention_chunk_workspace_bytes(dtype, format, tokens, sequences, heads, kv_heads,
                                                                  dim, block, tables.size(1));
    torch::Tensor workspace;
    if (bytes > 0) workspace = torch::empty({static_cast<int64_t>(bytes)}, query.options().dtype(torch::kUInt8));
    check_status(cf_paged_attention_chunk(
        query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), scales_of(k_scales), scales_of(v_scales),
        starts.data_ptr<int32_t>(), reinterpret_cast<const uint32_t*>(tables.data_ptr<int32_t>()),
        context.data_ptr<int32_t>(), out.data_ptr(), dtype, format, k_cache.size(0), tokens, sequences, heads,
        kv_heads, dim, block, tables.size(1), static_cast<float>(scale), bytes > 0 ? workspace.data_ptr() : nullptr,
        bytes, stream_for(query)));
    return out;
}

// ---- products of 8-bit integers ------------------------------------------------

std::tuple<torch::Tensor, torch::Tensor> quantize_int8_rows_hip(const torch::Tensor& x) {
    check_2d(x, "x");
    TORCH_CHECK(x.size(1) <= 1 || x.stride(1) == 1, "x must be dense along its rows");
    TORCH_CHECK(x.size(0) <= 1 || x.stride(0) >= x.size(1), "x's rows overlap: call .contiguous() first");
    const at::DeviceGuard guard(x.device());
    torch::Tensor codes = torch::empty(x.sizes(), x.options().dtype(torch::kInt8));
    torch::Tensor scales = torch::empty({x.size(0)}, x.options().dtype(torch::kFloat32));
    const cf_dtype dtype = to_cf(x, "x");
    if (x.size(1) == 0) return {codes, scales.fill_(1.0f)};
    check_status(cf_quantize_int8_rows(x.data_ptr(), dtype, x.size(0), x.size(1),
                                       x.size(0) > 1 ? x.stride(0) : x.size(1), codes.data_ptr<int8_t>(),
                                       scales.data_ptr<float>(), stream_for(x)));
    return {codes, scales};
}

constexpr int64_t kMostProducts = 131071;  // of two codes of -128 each, in 32 bits

torch::Tensor matmul_int8_hip(const torch::Tensor& x, const torch::Tensor& weight, const torch::Tensor& x_scales,
                              const torch::Tensor& w_scales, const std::optional<torch::Tensor>& bias,
                              at::ScalarType dtype) {
    const cf_dtype type = to_cf(dtype);
    check_2d(x, "x");
    check_2d(weight, "weight");
    for (const auto& [t, name] : {std::pair<const torch::Tensor*, const char*>{&x, "x"}, {&weight, "weight"}}) {
        TORCH_CHECK(t->scalar_type() == torch::kInt8, name, " must be int8, got ", t->scalar_type());
        check_contiguous(*t, name);
        check_same_device(x, *t, name);
    }
    TORCH_CHECK(x.size(1) == weight.size(1), "x has ", x.size(1), " columns but weight ", weight.size(1));
    TORCH_CHECK(x.size(1) <= kMostProducts, "rows of ", x.size(1), " products: their sum may leave 32 bits");
    for (const auto& [t, name, n] : {std::tuple<const torch::Tensor*, const char*, int64_t>{&x_scales, "x_scales", x.size(0)},
                                     {&w_scales, "w_scales", weight.size(0)}}) {
        TORCH_CHECK(t->dim() == 1 && t->size(0) == n && t->scalar_type() == torch::kFloat32, name,
                    " must be float32 [", n, "], got ", t->scalar_type(), " ", t->sizes());
        check_contiguous(*t, name);
        check_same_device(x, *t, name);
    }
    if (bias) {
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0) && bias->scalar_type() == dtype,
                    "bias must be ", dtype, " [", weight.size(0), "], got ", bias->scalar_type(), " ", bias->sizes());
        check_contiguous(*bias, "bias");
        check_same_device(x, *bias, "bias");
    }
    const at::DeviceGuard guard(x.device());
    torch::Tensor y = torch::empty({x.size(0), weight.size(0)}, x.options().dtype(dtype));
    if (y.numel() == 0) return y;
    check_status(cf_matmul_int8(x.data_ptr<int8_t>(), weight.data_ptr<int8_t>(), x_scales.data_ptr<float>(),
                                w_scales.data_ptr<float>(), bias ? bias->data_ptr() : nullptr, y.data_ptr(), type,
                                x.size(0), weight.size(0), x.size(1), stream_for(x)));
    return y;
}

// ---- direct entry for ordinary GPU calls (the rules: torch_ops_common.hpp) ------

/// A tensor or None; `good` is cleared for anything else.
std::optional<at::Tensor> ordinary_or_none(py::handle object, bool& good) {
    if (object.is_none()) return std::nullopt;
    const at::Tensor* t = ordinary(object);
    if (t == nullptr || t->requires_grad()) {
        good = false;
        return std::nullopt;
    }
    return *t;
}

bool same_device(const at::Tensor& like, std::initializer_list<const at::Tensor*> tensors) {
    for (const at::Tensor* t : tensors) {
        if (t->device() != like.device()) return false;
    }
    return true;
}

/// 4-D caches of one shape, type and device, with scales where they hold 8 bits.
bool ordinary_held(const at::Tensor* k, const at::Tensor* v, const std::optional<at::Tensor>& k_scales,
                   const std::optional<at::Tensor>& v_scales) {
    if (k == nullptr || v == nullptr || k->dim() != 4 || v->sizes() != k->sizes() ||
        v->scalar_type() != k->scalar_type() || v->device() != k->device() || k->requires_grad() || v->requires_grad()) {
        return false;
    }
    const bool codes = k->scalar_type() == torch::kInt8 || k->scalar_type() == torch::kFloat8_e4m3fn;
    if (!codes && !kernel_dtype(k->scalar_type())) return false;
    if (k_scales.has_value() != codes || v_scales.has_value() != codes) return false;
    for (const auto* s : {&k_scales, &v_scales}) {
        if (codes && ((*s)->sizes() != k->sizes().slice(0, 3) || (*s)->scalar_type() != torch::kFloat32 ||
                      (*s)->device() != k->device())) {
            return false;
        }
    }
    return true;
}

/// Plain, of any layout with a dense last dimension, no gradient needed.
const at::Tensor* ordinary_rows(py::handle object, int64_t dims) {
    if (!THPVariable_CheckTypeExact(Py_TYPE(object.ptr()))) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(object.ptr());
    const bool good = plain_gpu(t) && t.dim() == dims && t.numel() > 0 && !grad_needed({&t}) &&
                      (t.size(dims - 1) == 1 || t.stride(dims - 1) == 1) && kernel_dtype(t.scalar_type());
    return good ? &t : nullptr;
}

/// True when the call was taken.
bool try_cache_write(py::handle keys_, py::handle values_, py::handle k_, py::handle v_, py::handle slots_,
                     py::handle k_scales_, py::handle v_scales_) {
    bool good = ordinary_context();
    const at::Tensor* keys = ordinary_rows(keys_, 3);
    const at::Tensor* values = ordinary_rows(values_, 3);
    const at::Tensor* k = ordinary(k_);
    const at::Tensor* v = ordinary(v_);
    const at::Tensor* slots = ordinary(slots_);
    const auto k_scales = ordinary_or_none(k_scales_, good);
    const auto v_scales = ordinary_or_none(v_scales_, good);
    if (!good || keys == nullptr || values == nullptr || slots == nullptr || !ordinary_held(k, v, k_scales, v_scales) ||
        slots->dim() != 1 || slots->scalar_type() != torch::kInt64 || keys->sizes() != values->sizes() ||
        keys->scalar_type() != values->scalar_type() || keys->size(0) != slots->size(0) ||
        keys->size(1) != k->size(2) || keys->size(2) != k->size(3) ||
        (!k_scales && keys->scalar_type() != k->scalar_type()) || !same_device(*keys, {values, k, slots}) ||
        k_.ptr() == v_.ptr() || (k_scales && k_scales_.ptr() == v_scales_.ptr())) {
        return false;
    }
    py::gil_scoped_release no_gil;
    cache_write_hip(*keys, *values, *k, *v, *slots, k_scales, v_scales);
    return true;
}

py::object try_cache_read(py::handle k_, py::handle v_, py::handle slots_, py::handle k_scales_, py::handle v_scales_,
                          py::handle dtype_) {
    bool good = ordinary_context();
    const at::Tensor* k = ordinary(k_);
    const at::Tensor* v = ordinary(v_);
    const at::Tensor* slots = ordinary(slots_);
    const auto k_scales = ordinary_or_none(k_scales_, good);
    const auto v_scales = ordinary_or_none(v_scales_, good);
    if (!good || slots == nullptr || !ordinary_held(k, v, k_scales, v_scales) || slots->dim() != 1 ||
        slots->scalar_type() != torch::kInt64 || slots->device() != k->device()) {
        return py::none();
    }
    const auto dtype = plain_dtype(dtype_, k_scales ? torch::kFloat32 : k->scalar_type());
    if (!dtype || (!k_scales && *dtype != k->scalar_type())) return py::none();
    std::tuple<at::Tensor, at::Tensor> out;
    {
        py::gil_scoped_release no_gil;
        out = cache_read_hip(*k, *v, *slots, k_scales, v_scales, *dtype);
    }
    return py::make_tuple(wrap(std::get<0>(out)), wrap(std::get<1>(out)));
}

py::object try_paged_attention_chunk(py::handle query_, py::handle k_, py::handle v_, py::handle starts_,
                                     py::handle tables_, py::handle context_, py::handle k_scales_,
                                     py::handle v_scales_, py::handle scale_) {
    bool good = ordinary_context();
    const at::Tensor* query = ordinary(query_);
    const at::Tensor* k = ordinary(k_);
    const at::Tensor* v = ordinary(v_);
    const at::Tensor* starts = ordinary(starts_);
    const at::Tensor* tables = ordinary(tables_);
    const at::Tensor* context = ordinary(context_);
    const auto k_scales = ordinary_or_none(k_scales_, good);
    const auto v_scales = ordinary_or_none(v_scales_, good);
    const std::optional<double> scale = plain_double(scale_);
    if (!good || !scale || query == nullptr || query->dim() != 3 || !kernel_dtype(query->scalar_type()) ||
        grad_needed({query}) || !ordinary_held(k, v, k_scales, v_scales) ||
        !ordinary_ints({{starts, 1}, {tables, 2}, {context, 1}}) || !same_device(*query, {k, starts}) ||
        (!k_scales && query->scalar_type() != k->scalar_type()) || k->size(3) != query->size(2) ||
        query->size(2) > 1024 || query->size(1) % k->size(2) != 0 || tables->size(0) != context->size(0) ||
        starts->size(0) != context->size(0) + 1) {
        return py::none();
    }
    at::Tensor out;
    {
        py::gil_scoped_release no_gil;
        out = paged_attention_chunk_hip(*query, *k, *v, *starts, *tables, *context, k_scales, v_scales, *scale);
    }
    return wrap(out);
}

py::object try_quantize_int8_rows(py::handle x_) {
    const at::Tensor* x = ordinary_rows(x_, 2);
    if (x == nullptr || !ordinary_context() || (x->size(0) > 1 && x->stride(0) < x->size(1))) return py::none();
    std::tuple<at::Tensor, at::Tensor> out;
    {
        py::gil_scoped_release no_gil;
        out = quantize_int8_rows_hip(*x);
    }
    return py::make_tuple(wrap(std::get<0>(out)), wrap(std::get<1>(out)));
}

py::object try_matmul_int8(py::handle x_, py::handle w_, py::handle x_scales_, py::handle w_scales_, py::handle bias_,
                           py::handle dtype_) {
    bool good = ordinary_context();
    const at::Tensor* x = ordinary(x_);
    const at::Tensor* w = ordinary(w_);
    const auto x_scales = ordinary_or_none(x_scales_, good);
    const auto w_scales = ordinary_or_none(w_scales_, good);
    const auto bias = ordinary_or_none(bias_, good);
    const auto dtype = plain_dtype(dtype_, torch::kBFloat16);
    if (!good || dtype_.is_none() || !dtype || x == nullptr || w == nullptr || !x_scales || !w_scales ||
        x->dim() != 2 || w->dim() != 2 || x->scalar_type() != torch::kInt8 || w->scalar_type() != torch::kInt8 ||
        x->size(1) != w->size(1) || x->size(1) > kMostProducts || x_scales->dim() != 1 || w_scales->dim() != 1 ||
        x_scales->size(0) != x->size(0) || w_scales->size(0) != w->size(0) ||
        x_scales->scalar_type() != torch::kFloat32 || w_scales->scalar_type() != torch::kFloat32 ||
        !same_device(*x, {w, &*x_scales, &*w_scales}) ||
        (bias && (bias->dim() != 1 || bias->size(0) != w->size(0) || bias->scalar_type() != *dtype ||
                  bias->device() != x->device()))) {
        return py::none();
    }
    at::Tensor y;
    {
        py::gil_scoped_release no_gil;
        y = matmul_int8_hip(*x, *w, *x_scales, *w_scales, bias, *dtype);
    }
    return wrap(y);
}

}  // namespace

void bind_serving(py::module_& m) {
    m.def("try_cache_write", torch::wrap_pybind_function(&try_cache_write));
    m.def("try_cache_read", torch::wrap_pybind_function(&try_cache_read));
    m.def("try_paged_attention_chunk", torch::wrap_pybind_function(&try_paged_attention_chunk));
    m.def("try_quantize_int8_rows", torch::wrap_pybind_function(&try_quantize_int8_rows));
    m.def("try_matmul_int8", torch::wrap_pybind_function(&try_matmul_int8));
}

}  // namespace cudaforge_amd

TORCH_LIBRARY_FRAGMENT(cudaforge, m) {
    m.def(
        "cache_write(Tensor keys, Tensor values, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, "
        "Tensor(c!)? k_scales, Tensor(d!)? v_scales) -> ()");
    m.def(
        "cache_read(Tensor k_cache, Tensor v_cache, Tensor slots, Tensor? k_scales, Tensor? v_scales, "
        "ScalarType dtype) -> (Tensor, Tensor)");
    m.def(
        "paged_attention_chunk(Tensor query, Tensor k_cache, Tensor v_cache, Tensor query_starts, "
        "Tensor block_tables, Tensor context_lens, Tensor? k_scales, Tensor? v_scales, float scale) -> Tensor");
    m.def("quantize_int8_rows(Tensor x) -> (Tensor, Tensor)");
    m.def(
        "matmul_int8(Tensor x, Tensor weight, Tensor x_scales, Tensor w_scales, Tensor? bias, ScalarType dtype) "
        "-> Tensor");
}

// As in torch_ops.cpp: differentiating the operators themselves raises.
TORCH_LIBRARY_IMPL(cudaforge, Autograd, m) {
    for (const char* name : {"cache_read", "paged_attention_chunk", "quantize_int8_rows", "matmul_int8"}) {
        m.impl(name, torch::autograd::autogradNotImplementedFallback());
    }
}

TORCH_LIBRARY_IMPL(cudaforge, CUDA, m) {
    using namespace cudaforge_amd;
    m.impl("cache_write", &cache_write_hip);
    m.impl("cache_read", &cache_read_hip);
    m.impl("paged_attention_chunk", &paged_attention_chunk_hip);
    m.impl("quantize_int8_rows", &quantize_int8_rows_hip);
    m.impl("matmul_int8", &matmul_int8_hip);
}
