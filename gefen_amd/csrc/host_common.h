// Shared by the host extension's sources: what a call's tensors must be, and the library's errors.
#pragma once

#include <Python.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <ATen/ATen.h>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "gefen_hip.h"

namespace py = pybind11;

namespace gefen_host {

// gefen_last_error of the library that bind_library() was given.
extern decltype(&gefen_last_error) last_error;

inline void need_library() {
    if (!last_error) throw std::runtime_error("bind_library() has not been called");
}

inline void check(int rc) {
    if (rc == GEFEN_OK) return;
    if (rc == GEFEN_EINVAL) throw py::value_error(last_error());
    throw std::runtime_error(last_error());
}

inline int32_t dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return GEFEN_F32;
        case at::kHalf: return GEFEN_F16;
        case at::kBFloat16: return GEFEN_BF16;
        default: return -1;
    }
}

inline gefen_stream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline at::Tensor bytes_on(const at::Tensor& like, size_t n) {
    return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte).requires_grad(false));
}

inline const at::Tensor& tensor_of(py::handle o, const char* name) {
    if (!THPVariable_Check(o.ptr()))
        throw py::type_error(std::string("Expected ") + name + " to be a torch.Tensor, got " + Py_TYPE(o.ptr())->tp_name);
    return THPVariable_Unpack(o.ptr());
}

// Raises for a forward-mode tangent, which a call on addresses would drop.
inline void no_tangent(const at::Tensor& t, const char* name) {
    const auto* meta = torch::autograd::impl::get_autograd_meta(t);
    if (!meta || !meta->fw_grad(/*level=*/0, t).defined()) return;
    PyErr_Format(PyExc_NotImplementedError, "Expected %s without a forward-mode tangent.", name);
    throw py::error_already_set();
}

// A tensor whose memory holds its values: a view that stands for the negative of its memory
// (the imaginary part of a conjugate) is copied.
inline at::Tensor as_stored(const at::Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

inline py::object wrap(const at::Tensor& t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }

inline float* floats(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
inline void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

inline at::Tensor empty_grad(const at::Tensor& like, bool wanted, at::ScalarType type) {
    return wanted ? at::empty(like.sizes(), like.options().dtype(type).requires_grad(false)) : at::Tensor();
}

inline std::string shape_of(c10::IntArrayRef s) {
    std::string out = "(";
    for (size_t i = 0; i < s.size(); ++i) out += (i ? ", " : "") + std::to_string(s[i]);
    return out + ")";
}

// Raises unless a tensor is a plain strided one on the first tensor's device.
inline void plain_on(const at::Tensor& t, const char* name, const at::Tensor& first) {
    if (!t.is_cuda())
        throw py::value_error(std::string("Expected ") + name + " to be on CUDA, got device " + t.device().str() + ".");
    if (t.device() != first.device())
        throw py::value_error(std::string("Expected ") + name + " on " + first.device().str() + ", got " +
                              t.device().str() + ".");
    if (t.unsafeGetTensorImpl()->is_python_dispatch() || t.layout() != at::kStrided)
        throw py::type_error(std::string("Expected ") + name + " to be a plain strided tensor.");
}

}  // namespace gefen_host
