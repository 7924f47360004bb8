// What the files of the dispatcher shim share: argument checks, the current
// stream, and the test for calls that may go straight to the HIP
// implementations.
#pragma once

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/record_function.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <cmath>
#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "cudaforge_hip.h"

namespace cudaforge_amd {

// ---- shared checks ---------------------------------------------------------

inline void check_contiguous(const torch::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous; call .contiguous() first. ",
                "The kernels index rows as `base + row * cols`, which is only "
                "valid for a contiguous row-major layout.");
}

inline void check_2d(const torch::Tensor& t, const char* name) {
    TORCH_CHECK(t.dim() == 2, name, " must be 2-D, got ", t.dim(), " dimensions");
}

inline cf_dtype to_cf(const torch::Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case torch::kFloat32:
            return CF_F32;
        case torch::kBFloat16:
            return CF_BF16;
        case torch::kFloat16:
            return CF_F16;
        default:
            TORCH_CHECK(false, name, " has dtype ", t.scalar_type(),
                        ", which has no HIP kernel (float32, bfloat16 or float16)");
    }
}

inline cf_dtype to_cf(torch::ScalarType type) {
    switch (type) {
        case torch::kFloat32:
            return CF_F32;
        case torch::kBFloat16:
            return CF_BF16;
        case torch::kFloat16:
            return CF_F16;
        default:
            TORCH_CHECK(false, "dtype ", type, " has no HIP kernel (float32, bfloat16 or float16)");
    }
}

inline void check_same_device(const torch::Tensor& a, const torch::Tensor& b, const char* name) {
    TORCH_CHECK(a.device() == b.device(), name, " is on ", b.device(), " but the input is on ",
                a.device());
}

inline void check_ints(const torch::Tensor& t, int64_t dim, const torch::Tensor& like, const char* name) {
    TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimensions, got ", t.dim());
    TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be int32, got ", t.scalar_type());
    check_contiguous(t, name);
    check_same_device(like, t, name);
}

/// Counts a write for autograd's saved-tensor checks, as the mutating
/// operators of torch do.
inline void mark_written(const torch::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

/// PyTorch's current stream on the tensor's device, as the C ABI's void*.
inline void* stream_for(const torch::Tensor& t) {
    return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

inline void check_status(cf_status status) {
    TORCH_CHECK(status == CF_OK, "cudaforge HIP kernel failed: ", cf_last_error());
}

inline bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// ---- direct entry for ordinary GPU calls ---------------------------------------
//
// A call from Python through torch.ops costs 4-5 us of host time (schema
// parsing, boxing, the autograd fallback) on top of the checks in ops.py, more
// than the smallest kernels take. The try_* functions below are what ops.py
// asks first: when a call is an ordinary one they run the HIP implementation
// directly, otherwise they return None and ops.py goes its general way
// (validation messages, copies of non-contiguous inputs, fallbacks, the
// dispatcher). A call is ordinary when every tensor is a plain dense GPU tensor
// (exact type, no dispatch key beyond CUDA and its autograd), nothing is
// tracing, profiling, transforming or overriding it, no gradient is needed,
// and the arguments are ones the general way would pass to the same HIP
// implementation unchanged.

inline bool ordinary_context() {
    // Dispatch keys switched on for the thread: beyond these two, a mode
    // (tracing, functorch, Python dispatch) is active; autocast's key is always
    // on a tensor and excluded for the thread unless autocast is on.
    static const c10::DispatchKeySet usual({c10::DispatchKey::BackendSelect, c10::DispatchKey::ADInplaceOrView});
    const c10::impl::LocalDispatchKeySet local = c10::impl::tls_local_dispatch_key_set();
    return (local.included_.raw_repr() & ~usual.raw_repr()) == 0 &&
           local.excluded_.has(c10::DispatchKey::AutocastCUDA) && !at::impl::torch_function_mode_enabled() && !at::hasCallbacks();
}

/// Dense GPU storage, no dispatch key beyond CUDA and its autograd, and no
/// forward-mode tangent.
inline bool plain_gpu(const at::Tensor& t) {
    static const c10::DispatchKeySet usual(
        {c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::AutocastCUDA,
         c10::DispatchKey::ADInplaceOrView});
    return t.defined() && t.key_set().has(c10::DispatchKey::CUDA) &&
           (t.key_set().raw_repr() & ~usual.raw_repr()) == 0 && !t._fw_grad(0).defined();
}

/// The tensor behind `object`, or null when it is not a plain GPU tensor that
/// is contiguous and not empty.
inline const at::Tensor* ordinary(py::handle object) {
    if (!THPVariable_CheckTypeExact(Py_TYPE(object.ptr()))) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(object.ptr());
    return plain_gpu(t) && t.is_contiguous() && t.numel() > 0 ? &t : nullptr;
}

// The other arguments come as Python objects: a value that is not plainly a
// number or a dtype (a tensor, a NumPy type, a bool, an int out of range) is
// left to the general way, whose conversions and errors stand.

inline std::optional<double> plain_double(py::handle object) {
    if (PyFloat_Check(object.ptr())) return PyFloat_AS_DOUBLE(object.ptr());
    if (!PyLong_CheckExact(object.ptr())) return std::nullopt;
    const double value = PyLong_AsDouble(object.ptr());
    if (value == -1.0 && PyErr_Occurred() != nullptr) {
        PyErr_Clear();
        return std::nullopt;
    }
    return value;
}

inline std::optional<int64_t> plain_int(py::handle object) {
    if (!PyLong_CheckExact(object.ptr())) return std::nullopt;
    int overflow = 0;
    const long long value = PyLong_AsLongLongAndOverflow(object.ptr(), &overflow);
    return overflow == 0 ? std::optional<int64_t>(value) : std::nullopt;
}

/// The dtype given, `otherwise` for None, nothing for any other object or a
/// dtype without kernels.
inline std::optional<at::ScalarType> plain_dtype(py::handle object, at::ScalarType otherwise) {
    if (!object.is_none() && !THPDtype_Check(object.ptr())) return std::nullopt;
    const at::ScalarType t = object.is_none() ? otherwise : reinterpret_cast<THPDtype*>(object.ptr())->scalar_type;
    return t == torch::kFloat32 || t == torch::kBFloat16 || t == torch::kFloat16 ? std::optional<at::ScalarType>(t)
                                                                                 : std::nullopt;
}

inline bool kernel_dtype(at::ScalarType t) {
    return t == torch::kFloat32 || t == torch::kBFloat16 || t == torch::kFloat16;
}

inline bool grad_needed(std::initializer_list<const at::Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor* t : tensors) {
        if (t->requires_grad()) return true;
    }
    return false;
}

/// Plain, same dtype and device, a dtype with kernels, no gradient needed.
inline bool ordinary_set(std::initializer_list<const at::Tensor*> tensors) {
    const at::Tensor* first = *tensors.begin();
    for (const at::Tensor* t : tensors) {
        if (t == nullptr || t->scalar_type() != first->scalar_type() || t->device() != first->device()) return false;
    }
    return kernel_dtype(first->scalar_type()) && !grad_needed(tensors);
}

/// Ordinary int32 tensors of the given dimensions, all on one device.
inline bool ordinary_ints(std::initializer_list<std::pair<const at::Tensor*, int64_t>> tensors) {
    const at::Tensor* first = tensors.begin()->first;
    for (const auto& [t, dim] : tensors) {
        if (t == nullptr || t->scalar_type() != torch::kInt32 || t->dim() != dim || t->device() != first->device()) {
            return false;
        }
    }
    return true;
}

inline py::object wrap(const at::Tensor& t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }

/// Adds the entries of torch_ops_generation.cpp to the extension module.
void bind_generation(py::module_& m);

/// And those of torch_ops_serving.cpp.
void bind_serving(py::module_& m);

}  // namespace cudaforge_amd
