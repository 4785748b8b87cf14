// block_ops.cpp -- the torch side of include/nflow_block.h (and, in
// residual_ops.h, of include/nflow_residual.h): argument checks, allocations and
// the call, in C++.
//
// A call of a few rows takes 3 to 6 us on the GPU, and as many to launch;
// checks, three allocations and a ctypes call in Python add 6 us to that, here
// 1.5 (layer_norm of one token with its statistics: 9.0 -> 6.0 us a call).
// neuroflow_amd/norm.py, block_fp8.py, dense.py and grads.py are the public face; the errors raised
// here are theirs (TypeError, ValueError, NflowError).
#include "residual_ops.h"

using namespace nfq_torch;

namespace {

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
    m.doc() = "torch calls of include/nflow_block.h and include/nflow_residual.h";
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
    define_residual_ops(m);
}
