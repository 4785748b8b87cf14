// torch_args.h -- what the torch calls of nflow_block.h and nflow_residual.h
// share: the library's entry points, checks of tensors, errors, allocations.
#pragma once

#include <dlfcn.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>
#include <vector>

#include "nflow_residual.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace nfq_torch {

// The library's entry points.  bind() takes their addresses from the library that
// Python has loaded, which may be another build than the one beside this module:
// linked, the module would bring a second copy into the process.
#define NFLOW_BLOCK_OPS(X) \
    X(nflow_last_error) \
    X(nflow_fp8_block_linear) \
    X(nflow_fp8_block_linear_backward) \
    X(nflow_fp8_block_linear_backward_workspace) \
    X(nflow_fp8_block_linear_workspace) \
    X(nflow_fp8_block_matmul) \
    X(nflow_fp8_block_matmul_workspace) \
    X(nflow_fp8_block_quantise) \
    X(nflow_fp8_block_quantise_weight) \
    X(nflow_layer_norm_backward) \
    X(nflow_layer_norm_backward_workspace) \
    X(nflow_layer_norm_forward) \
    X(nflow_layer_norm_fp8_block)
#define NFLOW_RESIDUAL_OPS(X) \
    X(nflow_dense_linear) \
    X(nflow_dense_linear_backward) \
    X(nflow_dense_linear_backward_workspace) \
    X(nflow_dense_linear_workspace) \
    X(nflow_grad_clip) \
    X(nflow_grad_norm) \
    X(nflow_grad_workspace) \
    X(nflow_rms_norm_backward) \
    X(nflow_rms_norm_backward_workspace) \
    X(nflow_rms_norm_forward) \
    X(nflow_rms_norm_fp8)

struct Api {
#define X(f) decltype(&::f) f = nullptr;
    NFLOW_BLOCK_OPS(X)
    NFLOW_RESIDUAL_OPS(X)
#undef X
};
inline Api api;

#define X(f) #f,
inline std::vector<std::string> entry_points() { return {NFLOW_BLOCK_OPS(X)}; }
inline std::vector<std::string> residual_entry_points() { return {NFLOW_RESIDUAL_OPS(X)}; }
#undef X

inline void bind(const py::function& address) {
#define X(f) api.f = reinterpret_cast<decltype(api.f)>(address(#f).cast<uintptr_t>());
    NFLOW_BLOCK_OPS(X)
    NFLOW_RESIDUAL_OPS(X)
#undef X
}

// The file that the bound entry points are in.
inline std::string library() {
    Dl_info info{};
    return dladdr(reinterpret_cast<void*>(api.nflow_last_error), &info) && info.dli_fname ? info.dli_fname : "";
}

struct Matrix {
    int64_t rows, cols, ld;
};

inline std::string str(const char* name, const std::string& rest) { return std::string(name) + rest; }

inline int dtype_of(const Tensor& t, const char* name) {
    if (!t.defined() || !t.is_cuda()) throw py::type_error(str(name, " must be a CUDA tensor"));
    if (t.scalar_type() == at::kFloat) return NFLOW_DTYPE_F32;
    if (t.scalar_type() == at::kBFloat16) return NFLOW_DTYPE_BF16;
    throw py::type_error(str(name, " must be float32 or bfloat16, got ") + c10::toString(t.scalar_type()));
}

// Rows, columns and row stride: any contiguous tensor, or a 2-D one whose last
// axis is.
inline Matrix matrix(const Tensor& t, const char* name) {
    if (t.dim() == 0) throw py::value_error(str(name, " needs an axis"));
    const int64_t K = t.size(-1);
    if (t.is_contiguous()) {
        int64_t rows = 1;
        for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
        return {rows, K, K};
    }
    if (t.dim() > 2 || t.stride(-1) != 1 || t.dim() == 1 || t.stride(0) < K)
        throw py::value_error(str(name, " must be contiguous, or 2-D with a contiguous last axis"));
    return {t.size(0), K, t.stride(0)};
}

inline void same(const Tensor& t, const char* name, const Tensor& like) {
    dtype_of(t, name);
    if (t.sizes() != like.sizes() || t.scalar_type() != like.scalar_type() || t.device() != like.device())
        throw py::value_error(str(name, " must have the shape, type and device of x"));
}

// An operand's memory has to be on the GPU that the call runs on.
inline void on_device(const Tensor& t, const char* name, const Tensor& like) {
    if (t.device() != like.device())
        throw py::value_error(str(name, " is on ") + t.device().str() + ", the call's other tensors on " +
                              like.device().str());
}

inline float* param(const Maybe& p, int64_t n, const char* name, const Tensor& like, bool required = false) {
    if (!p) {
        if (required) throw py::type_error(str(name, " is required"));
        return nullptr;
    }
    const Tensor& t = *p;
    if (!t.is_cuda()) throw py::type_error(str(name, " must be a CUDA tensor"));
    if (t.scalar_type() != at::kFloat) throw py::type_error(str(name, " must be float32"));
    if (t.numel() != n || !t.is_contiguous())
        throw py::value_error(str(name, " must be ") + std::to_string(n) + " contiguous values");
    on_device(t, name, like);
    return static_cast<float*>(t.data_ptr());
}

inline int64_t blocks(int64_t n) { return (n + 127) / 128; }

// Rows of a block-FP8 matrix, its tensors checked against k and the device of `like`.
inline int64_t block_rows(const Tensor& codes, const Tensor& scales, int64_t k, bool weight, const char* name,
                   const Tensor& like) {
    if (!codes.defined() || !scales.defined() || !codes.is_cuda() || !scales.is_cuda())
        throw py::type_error(str(name, " must hold CUDA tensors"));
    if (codes.scalar_type() != at::kByte || scales.scalar_type() != at::kFloat)
        throw py::type_error(str(name, " must hold uint8 codes and float32 scales"));
    const int64_t kb = blocks(k);
    if (k < 0 || codes.dim() != 2 || codes.size(1) != 128 * kb || !codes.is_contiguous())
        throw py::value_error(str(name, ".codes must be a contiguous (rows, ") + std::to_string(128 * kb) + ") for k = " +
                              std::to_string(k));
    const int64_t R = codes.size(0), cols = weight ? blocks(R) : R;
    if (scales.dim() != 2 || scales.size(0) != kb || scales.size(1) != cols || !scales.is_contiguous())
        throw py::value_error(str(name, ".scales must be a contiguous (") + std::to_string(kb) + ", " +
                              std::to_string(cols) + ")");
    on_device(codes, name, like);
    on_device(scales, name, like);
    return R;
}

template <typename T = void>
T* data(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// The current stream, on t's device, which has to be the current one.
inline void* stream_of(const Tensor& t) {
    const auto here = c10::hip::current_device();
    if (t.device().index() != here)
        throw py::value_error("the tensors are on cuda:" + std::to_string(t.device().index()) +
                              ", the current device is cuda:" + std::to_string(here));
    return c10::hip::getCurrentHIPStream(here).stream();
}

inline void ok(int rc, const char* what) {
    if (rc == NFLOW_OK) return;
    const py::object type = py::module_::import("neuroflow_amd._lib").attr("NflowError");
    const py::object e = type(rc, what, api.nflow_last_error());
    PyErr_SetObject(type.ptr(), e.ptr());
    throw py::error_already_set();
}

inline Tensor empty(at::IntArrayRef size, const Tensor& like, at::ScalarType type) {
    return at::empty(size, like.options().dtype(type));
}
inline Tensor scratch(size_t n, const Tensor& like) {
    return n ? empty({static_cast<int64_t>(n)}, like, at::kByte) : Tensor();
}

}  // namespace nfq_torch
