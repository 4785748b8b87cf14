// block_ops.cpp -- the torch side of include/nflow_block.h: argument checks,
// allocations and the call, in C++.
//
// A call of a few rows takes 3 to 6 us on the GPU, and as many to launch;
// checks, three allocations and a ctypes call in Python add 6 us to that, here
// 1.5 (layer_norm of one token with its statistics: 9.0 -> 6.0 us a call).
// neuroflow_amd/norm.py and block_fp8.py are the public face; the errors raised
// here are theirs (TypeError, ValueError, NflowError).
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

#include "nflow_block.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

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

struct Api {
#define X(f) decltype(&::f) f = nullptr;
    NFLOW_BLOCK_OPS(X)
#undef X
} api;

std::vector<std::string> entry_points() {
#define X(f) #f,
    return {NFLOW_BLOCK_OPS(X)};
#undef X
}

void bind(const py::function& address) {
#define X(f) api.f = reinterpret_cast<decltype(api.f)>(address(#f).cast<uintptr_t>());
    NFLOW_BLOCK_OPS(X)
#undef X
}

// The file that the bound entry points are in.
std::string library() {
    Dl_info info{};
    return dladdr(reinterpret_cast<void*>(api.nflow_last_error), &info) && info.dli_fname ? info.dli_fname : "";
}

struct Matrix {
    int64_t rows, cols, ld;
};

std::string str(const char* name, const std::string& rest) { return std::string(name) + rest; }

int dtype_of(const Tensor& t, const char* name) {
    if (!t.defined() || !t.is_cuda()) throw py::type_error(str(name, " must be a CUDA tensor"));
    if (t.scalar_type() == at::kFloat) return NFLOW_DTYPE_F32;
    if (t.scalar_type() == at::kBFloat16) return NFLOW_DTYPE_BF16;
    throw py::type_error(str(name, " must be float32 or bfloat16, got ") + c10::toString(t.scalar_type()));
}

// Rows, columns and row stride: any contiguous tensor, or a 2-D one whose last
// axis is.
Matrix matrix(const Tensor& t, const char* name) {
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

void same(const Tensor& t, const char* name, const Tensor& like) {
    dtype_of(t, name);
    if (t.sizes() != like.sizes() || t.scalar_type() != like.scalar_type() || t.device() != like.device())
        throw py::value_error(str(name, " must have the shape, type and device of x"));
}

// An operand's memory has to be on the GPU that the call runs on.
void on_device(const Tensor& t, const char* name, const Tensor& like) {
    if (t.device() != like.device())
        throw py::value_error(str(name, " is on ") + t.device().str() + ", the call's other tensors on " +
                              like.device().str());
}

float* param(const Maybe& p, int64_t n, const char* name, const Tensor& like, bool required = false) {
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

int64_t blocks(int64_t n) { return (n + 127) / 128; }

// Rows of a block-FP8 matrix, its tensors checked against k and the device of `like`.
int64_t block_rows(const Tensor& codes, const Tensor& scales, int64_t k, bool weight, const char* name,
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
void* stream_of(const Tensor& t) {
    const auto here = c10::hip::current_device();
    if (t.device().index() != here)
        throw py::value_error("the tensors are on cuda:" + std::to_string(t.device().index()) +
                              ", the current device is cuda:" + std::to_string(here));
    return c10::hip::getCurrentHIPStream(here).stream();
}

void ok(int rc, const char* what) {
    if (rc == NFLOW_OK) return;
    const py::object type = py::module_::import("neuroflow_amd._lib").attr("NflowError");
    const py::object e = type(rc, what, api.nflow_last_error());
    PyErr_SetObject(type.ptr(), e.ptr());
    throw py::error_already_set();
}

Tensor empty(at::IntArrayRef size, const Tensor& like, at::ScalarType type) {
    return at::empty(size, like.options().dtype(type));
}
Tensor scratch(size_t n, const Tensor& like) {
    return n ? empty({static_cast<int64_t>(n)}, like, at::kByte) : Tensor();
}

// ---- layer norm ----

py::object layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps, const Maybe& out,
                      bool stats) {
    const int dt = dtype_of(x, "x");
    const Matrix m = matrix(x, "x");
    const float *w = param(weight, m.cols, "weight", x), *b = param(bias, m.cols, "bias", x);
    Tensor y;
    int64_t ldy = m.cols;
    if (out) {
        y = *out;
        same(y, "out", x);
        ldy = matrix(y, "out").ld;
        if (y.requires_grad() && at::GradMode::is_enabled())
            throw py::value_error("out requires grad: these functions record no autograd graph");
    } else {
        y = empty(x.sizes(), x, x.scalar_type());
    }
    Tensor mean, rstd;
    if (stats) {
        mean = empty({m.rows}, x, at::kFloat);
        rstd = empty({m.rows}, x, at::kFloat);
    }
    ok(api.nflow_layer_norm_forward(data(x), dt, m.rows, m.cols, m.ld, w, b, static_cast<float>(eps), data(y), ldy,
                                data<float>(mean), data<float>(rstd), stream_of(x)), "layer_norm");
    if (out && !y.is_inference()) y.unsafeGetTensorImpl()->bump_version();   // a graph that saved it has to notice
    if (!stats) return py::cast(y);
    return py::make_tuple(y, mean, rstd);
}

py::tuple layer_norm_fp8(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps, bool stats) {
    const int dt = dtype_of(x, "x");
    const Matrix m = matrix(x, "x");
    const float *w = param(weight, m.cols, "weight", x), *b = param(bias, m.cols, "bias", x);
    const Tensor codes = empty({m.rows, 128 * blocks(m.cols)}, x, at::kByte);
    const Tensor scales = empty({blocks(m.cols), m.rows}, x, at::kFloat);
    Tensor mean, rstd;
    if (stats) {
        mean = empty({m.rows}, x, at::kFloat);
        rstd = empty({m.rows}, x, at::kFloat);
    }
    ok(api.nflow_layer_norm_fp8_block(data(x), dt, m.rows, m.cols, m.ld, w, b, static_cast<float>(eps), data<uint8_t>(codes),
                                  data<float>(scales), data<float>(mean), data<float>(rstd), stream_of(x)),
       "layer_norm_fp8");
    return py::make_tuple(codes, scales, m.cols, mean, rstd);
}

py::tuple layer_norm_backward(const Tensor& dy, const Tensor& x, const Maybe& weight, const Maybe& mean,
                              const Maybe& rstd) {
    const int dt = dtype_of(x, "x");
    const Matrix m = matrix(x, "x");
    same(dy, "dy", x);
    const Matrix g = matrix(dy, "dy");
    const float* w = param(weight, m.cols, "weight", x);
    const float *mu = param(mean, m.rows, "mean", x, true), *rs = param(rstd, m.rows, "rstd", x, true);
    const Tensor dx = empty(x.sizes(), x, x.scalar_type());
    const Tensor dw = empty({m.cols}, x, at::kFloat), db = empty({m.cols}, x, at::kFloat);
    size_t n = 0;
    ok(api.nflow_layer_norm_backward_workspace(m.rows, m.cols, &n), "layer_norm_backward");
    const Tensor ws = scratch(n, x);
    ok(api.nflow_layer_norm_backward(data(dy), data(x), dt, m.rows, m.cols, g.ld, m.ld, w, mu, rs, data(dx), m.cols,
                                 data<float>(dw), data<float>(db), data(ws), n, stream_of(x)), "layer_norm_backward");
    return py::make_tuple(dx, dw, db);
}

// ---- block FP8 ----

py::tuple quantise(const Tensor& x, bool rows, bool columns) {
    const int dt = dtype_of(x, "x");
    const Matrix m = matrix(x, "x");
    Tensor c, s, ct, st;
    if (rows) {
        c = empty({m.rows, 128 * blocks(m.cols)}, x, at::kByte);
        s = empty({blocks(m.cols), m.rows}, x, at::kFloat);
    }
    if (columns) {
        ct = empty({m.cols, 128 * blocks(m.rows)}, x, at::kByte);
        st = empty({blocks(m.rows), m.cols}, x, at::kFloat);
    }
    ok(api.nflow_fp8_block_quantise(data(x), dt, m.rows, m.cols, m.ld, data<uint8_t>(c), data<float>(s), data<uint8_t>(ct),
                                data<float>(st), stream_of(x)), "fp8_block_quantise");
    return py::make_tuple(c, s, m.cols, ct, st, m.rows);
}

py::tuple quantise_weight(const Tensor& W, bool transposed) {
    const int dt = dtype_of(W, "W");
    const Matrix m = matrix(W, "W");
    const int64_t nb = blocks(m.rows), kb = blocks(m.cols);
    const Tensor c = empty({m.rows, 128 * kb}, W, at::kByte), s = empty({kb, nb}, W, at::kFloat);
    Tensor ct, st;
    if (transposed) {
        ct = empty({m.cols, 128 * nb}, W, at::kByte);
        st = empty({nb, kb}, W, at::kFloat);
    }
    ok(api.nflow_fp8_block_quantise_weight(data(W), dt, m.rows, m.cols, m.ld, data<uint8_t>(c), data<float>(s),
                                       data<uint8_t>(ct), data<float>(st), stream_of(W)), "fp8_block_quantise_weight");
    return py::make_tuple(c, s, m.cols, ct, st, m.rows);
}

Tensor matmul(const Tensor& ac, const Tensor& as, int64_t ak, const Tensor& wc, const Tensor& wsc, int64_t wk,
              const Maybe& bias, int act, int dt) {
    if (ak != wk)
        throw py::value_error("a has " + std::to_string(ak) + " columns, w has " + std::to_string(wk));
    const int64_t M = block_rows(ac, as, ak, false, "a", ac);
    // One row has one scale a block in either form: taken as a weight's, as linear has it.
    const bool weight = wc.defined() && wsc.defined() && wc.dim() == 2 && wsc.dim() == 2 &&
                        (wsc.size(1) != wc.size(0) || wc.size(0) == 1);
    const int64_t N = block_rows(wc, wsc, wk, weight, "w", ac);
    const float* b = param(bias, N, "bias", ac);
    const Tensor y = empty({M, N}, ac, dt == NFLOW_DTYPE_BF16 ? at::kBFloat16 : at::kFloat);
    size_t n = 0;
    ok(api.nflow_fp8_block_matmul_workspace(M, N, ak, dt, &n), "fp8_block_matmul");
    const Tensor ws = scratch(n, ac);
    ok(api.nflow_fp8_block_matmul(data<uint8_t>(ac), data<float>(as), data<uint8_t>(wc), data<float>(wsc), weight, M, N, ak,
                              b, act, data(y), dt, N, data(ws), n, stream_of(ac)), "fp8_block_matmul");
    return y;
}

Tensor linear(const Tensor& x, const Tensor& wc, const Tensor& wsc, int64_t wk, const Maybe& bias, int act) {
    const int dt = dtype_of(x, "x");
    const Matrix m = matrix(x, "x");
    if (wk != m.cols)
        throw py::value_error("x has " + std::to_string(m.cols) + " columns, w has " + std::to_string(wk));
    const int64_t N = block_rows(wc, wsc, wk, true, "w", x);
    const float* b = param(bias, N, "bias", x);
    c10::SmallVector<int64_t, 6> size(x.sizes().begin(), x.sizes().end());
    size.back() = N;
    const Tensor y = empty(size, x, x.scalar_type());
    size_t n = 0;
    ok(api.nflow_fp8_block_linear_workspace(m.rows, N, wk, dt, &n), "fp8_block_linear");
    const Tensor ws = scratch(n, x);
    ok(api.nflow_fp8_block_linear(data(x), dt, m.rows, m.cols, m.ld, data<uint8_t>(wc), data<float>(wsc), N, b, act, data(y),
                              N, data(ws), n, stream_of(x)), "fp8_block_linear");
    return y;
}

py::tuple linear_backward(const Tensor& dy, const Tensor& xc, const Tensor& xs, int64_t xk, const Tensor& wc,
                          const Tensor& wsc, int64_t wk) {
    const int dt = dtype_of(dy, "dy");
    const Matrix m = matrix(dy, "dy");
    const int64_t K = block_rows(wc, wsc, wk, true, "w_transposed", dy);
    if (wk != m.cols)
        throw py::value_error("dy has " + std::to_string(m.cols) + " columns, w_transposed has " + std::to_string(wk));
    if (xk != m.rows || block_rows(xc, xs, xk, false, "x_columns", dy) != K)
        throw py::value_error("x_columns must be (" + std::to_string(K) + " rows, k = " + std::to_string(m.rows) + ")");
    c10::SmallVector<int64_t, 6> size(dy.sizes().begin(), dy.sizes().end());
    size.back() = K;
    const Tensor dx = empty(size, dy, dy.scalar_type());
    const Tensor dW = empty({m.cols, K}, dy, at::kFloat), db = empty({m.cols}, dy, at::kFloat);
    size_t n = 0;
    ok(api.nflow_fp8_block_linear_backward_workspace(m.rows, m.cols, K, dt, &n), "fp8_block_linear_backward");
    const Tensor ws = scratch(n, dy);
    ok(api.nflow_fp8_block_linear_backward(data(dy), dt, m.rows, m.cols, m.ld, data<uint8_t>(xc), data<float>(xs),
                                       data<uint8_t>(wc), data<float>(wsc), K, data(dx), K, data<float>(dW),
                                       data<float>(db), data(ws), n, stream_of(dy)), "fp8_block_linear_backward");
    return py::make_tuple(dx, dW, db);
}

}  // namespace

PYBIND11_MODULE(block_ops, m) {
    m.doc() = "torch calls of include/nflow_block.h (neuroflow_amd.norm, neuroflow_amd.block_fp8)";
    m.def("bind", &bind);
    m.def("entry_points", &entry_points);
    m.def("library", &library);
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_fp8", &layer_norm_fp8);
    m.def("layer_norm_backward", &layer_norm_backward);
    m.def("quantise", &quantise);
    m.def("quantise_weight", &quantise_weight);
    m.def("matmul", &matmul);
    m.def("linear", &linear);
    m.def("linear_backward", &linear_backward);
}
