// residual_ops.h -- the torch side of include/nflow_residual.h.
#pragma once

#include "torch_args.h"

namespace nfq_torch {

// A result that the caller gave: of x's type and device, and none that a graph
// would have to record.
inline Matrix result(const Tensor& t, const char* name, at::IntArrayRef size, const Tensor& like) {
    dtype_of(t, name);
    if (t.sizes() != size || t.scalar_type() != like.scalar_type() || t.device() != like.device())
        throw py::value_error(str(name, " must have the shape of the result, and x's type and device"));
    if (t.requires_grad() && at::GradMode::is_enabled())
        throw py::value_error(str(name, " requires grad: these functions record no autograd graph"));
    return matrix(t, name);
}
// A graph that saved what has been written has to notice.
inline void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---- RMS norm ----

struct RmsCall {
    int dt;
    Matrix m, r{0, 0, 0}, s{0, 0, 0};
    const float* w;
    Tensor sum, rstd;
    RmsCall(const Tensor& x, const Maybe& weight, const Maybe& residual, const Maybe& sum_out, bool stats)
        : dt(dtype_of(x, "x")), m(matrix(x, "x")), w(param(weight, m.cols, "weight", x)) {
        if (residual) {
            same(*residual, "residual", x);
            r = matrix(*residual, "residual");
            sum = sum_out ? *sum_out : empty(x.sizes(), x, x.scalar_type());
            s = sum_out ? result(sum, "sum_out", x.sizes(), x) : Matrix{m.rows, m.cols, m.cols};
        } else if (sum_out) {
            throw py::value_error("sum_out without a residual");
        }
        if (stats) rstd = empty({m.rows}, x, at::kFloat);
    }
};

inline py::tuple rms_norm(const Tensor& x, const Maybe& weight, double eps, const Maybe& residual, const Maybe& sum_out,
                          bool stats) {
    const RmsCall c(x, weight, residual, sum_out, stats);
    const Tensor y = empty(x.sizes(), x, x.scalar_type());
    ok(api.nflow_rms_norm_forward(data(x), c.dt, c.m.rows, c.m.cols, c.m.ld, residual ? data(*residual) : nullptr, c.r.ld,
                                  c.w, static_cast<float>(eps), data(y), c.m.cols, data(c.sum), c.s.ld,
                                  data<float>(c.rstd), stream_of(x)), "rms_norm");
    if (sum_out) written(c.sum);
    return py::make_tuple(y, c.sum, c.rstd);
}

inline py::tuple rms_norm_fp8(const Tensor& x, const Maybe& weight, double eps, const Maybe& residual,
                              const Maybe& sum_out, bool stats) {
    const RmsCall c(x, weight, residual, sum_out, stats);
    const Tensor codes = empty({c.m.rows, 128 * blocks(c.m.cols)}, x, at::kByte);
    const Tensor scales = empty({blocks(c.m.cols), c.m.rows}, x, at::kFloat);
    ok(api.nflow_rms_norm_fp8(data(x), c.dt, c.m.rows, c.m.cols, c.m.ld, residual ? data(*residual) : nullptr, c.r.ld, c.w,
                              static_cast<float>(eps), data<uint8_t>(codes), data<float>(scales), data(c.sum), c.s.ld,
                              data<float>(c.rstd), stream_of(x)), "rms_norm_fp8");
    if (sum_out) written(c.sum);
    return py::make_tuple(codes, scales, c.m.cols, c.sum, c.rstd);
}

inline py::tuple rms_norm_backward(const Tensor& dy, const Tensor& x, const Maybe& weight, const Maybe& rstd,
                                   const Maybe& dsum) {
    const int dt = dtype_of(x, "x");
    const Matrix m = matrix(x, "x");
    same(dy, "dy", x);
    const Matrix g = matrix(dy, "dy");
    const float *w = param(weight, m.cols, "weight", x), *rs = param(rstd, m.rows, "rstd", x, true);
    Matrix d{0, 0, 0};
    if (dsum) {
        same(*dsum, "dsum", x);
        d = matrix(*dsum, "dsum");
    }
    const Tensor dx = empty(x.sizes(), x, x.scalar_type()), dw = empty({m.cols}, x, at::kFloat);
    size_t n = 0;
    ok(api.nflow_rms_norm_backward_workspace(m.rows, m.cols, &n), "rms_norm_backward");
    const Tensor ws = scratch(n, x);
    ok(api.nflow_rms_norm_backward(data(dy), data(x), dt, m.rows, m.cols, g.ld, m.ld, w, rs, dsum ? data(*dsum) : nullptr,
                                   d.ld, data(dx), m.cols, data<float>(dw), data(ws), n, stream_of(x)),
       "rms_norm_backward");
    return py::make_tuple(dx, dw);
}

// ---- the linear layer in bf16 or fp32 ----

// `copies` of nflow_dense_linear for a bf16 operand, and for two of them.
inline int odd(const Tensor& t, const Matrix& m) {
    const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
    if ((at & 15) == 0 && m.ld % 8 == 0 && m.cols % 8 == 0 && m.ld < NFLOW_DENSE_MAX_K) return 0;
    return (at & 3) == 0 && m.ld % 2 == 0 ? 2 : 1;
}
inline int odd(int a, int b) { return a == 1 || b == 1 ? 1 : a | b; }

// A weight (N, K) of x's type.
inline Matrix weight_of(const Tensor& W, const Tensor& x, int64_t cols, const char* of) {
    dtype_of(W, "W");
    if (W.dim() != 2) throw py::value_error("W must be (N, K)");
    if (W.scalar_type() != x.scalar_type()) throw py::type_error(str("W must have the type of ", of));
    on_device(W, "W", x);
    const Matrix w = matrix(W, "W");
    if (cols >= 0 && w.cols != cols)
        throw py::value_error(str(of, " has ") + std::to_string(cols) + " columns, W has " + std::to_string(w.cols));
    return w;
}

inline py::tuple dense_linear(const Tensor& x, const Tensor& W, const Maybe& bias, int act, const Maybe& residual,
                              const Maybe& out, bool return_pre) {
    const int dt = dtype_of(x, "x");
    const Matrix m = matrix(x, "x"), w = weight_of(W, x, m.cols, "x");
    const int64_t N = w.rows;
    const float* b = param(bias, N, "bias", x);
    c10::SmallVector<int64_t, 6> size(x.sizes().begin(), x.sizes().end());
    size.back() = N;
    Matrix r{0, 0, 0}, yl{m.rows, N, N};
    if (residual) {
        dtype_of(*residual, "residual");
        if (residual->sizes() != at::IntArrayRef(size) || residual->scalar_type() != x.scalar_type())
            throw py::value_error("residual must have the shape of the result and x's type");
        on_device(*residual, "residual", x);
        r = matrix(*residual, "residual");
    }
    Tensor y, pre;
    if (out) {
        y = *out;
        yl = result(y, "out", size, x);
    } else {
        y = empty(size, x, x.scalar_type());
    }
    if (return_pre) pre = empty(size, x, x.scalar_type());
    size_t n = 0;
    ok(api.nflow_dense_linear_workspace(m.rows, N, m.cols, dt, odd(odd(x, m), odd(W, w)), &n), "dense_linear");
    const Tensor ws = scratch(n, x);
    ok(api.nflow_dense_linear(data(x), dt, m.rows, m.cols, m.ld, data(W), w.ld, N, b, residual ? data(*residual) : nullptr,
                              r.ld, act, data(y), yl.ld, data(pre), N, data(ws), n, stream_of(x)), "dense_linear");
    if (out) written(y);
    return py::make_tuple(y, pre);
}

inline py::tuple dense_linear_backward(const Tensor& dy, const Tensor& x, const Tensor& W, int act, const Maybe& pre) {
    const int dt = dtype_of(dy, "dy");
    const Matrix m = matrix(dy, "dy"), w = weight_of(W, dy, -1, "dy");
    dtype_of(x, "x");
    if (x.scalar_type() != dy.scalar_type()) throw py::type_error("x must have the type of dy");
    on_device(x, "x", dy);
    const Matrix xm = matrix(x, "x");
    const int64_t K = w.cols;
    if (w.rows != m.cols || xm.cols != K || xm.rows != m.rows)
        throw py::value_error("dy (..., N), x (..., K) and W (N, K) do not fit one another");
    Matrix p{0, 0, 0};
    Tensor dz;
    if (act != NFLOW_ACT_NONE) {
        if (!pre) throw py::type_error("pre is required with an activation");
        same(*pre, "pre", dy);
        p = matrix(*pre, "pre");
        dz = empty(dy.sizes(), dy, dy.scalar_type());
    } else if (pre) {
        throw py::value_error("pre without an activation");
    }
    c10::SmallVector<int64_t, 6> size(dy.sizes().begin(), dy.sizes().end());
    size.back() = K;
    const Tensor dx = empty(size, dy, dy.scalar_type()), dW = empty({m.cols, K}, dy, dy.scalar_type());
    const Tensor db = empty({m.cols}, dy, at::kFloat);
    size_t n = 0;
    ok(api.nflow_dense_linear_backward_workspace(m.rows, m.cols, K, dt, odd(dy, m) || odd(x, xm) || odd(W, w), &n), "dense_linear_backward");
    const Tensor ws = scratch(n, dy);
    ok(api.nflow_dense_linear_backward(data(dy), dt, m.rows, m.cols, m.ld, data(x), xm.ld, data(W), w.ld, K, act,
                                       pre ? data(*pre) : nullptr, p.ld, data(dz), m.cols, data(dx), K, data(dW), K,
                                       data<float>(db), data(ws), n, stream_of(dy)), "dense_linear_backward");
    return py::make_tuple(dx, dW, db, dz.defined() ? dz : dy);
}

// ---- gradient clipping ----

struct GradList {
    std::vector<nflow_grad_tensor> t;
    const Tensor* like = nullptr;
};
inline GradList grad_list(const std::vector<Tensor>& grads, const std::vector<Tensor>* out) {
    if (grads.empty()) throw py::value_error("no gradients");
    if (out && out->size() != grads.size()) throw py::value_error("out must hold a tensor for every gradient");
    GradList l;
    l.t.reserve(grads.size());
    l.like = &grads[0];
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor& g = grads[i];
        const int dt = dtype_of(g, "a gradient");
        if (!g.is_contiguous()) throw py::value_error("gradients must be contiguous");
        on_device(g, "a gradient", *l.like);
        const Tensor& o = out ? (*out)[i] : g;
        if (out) {
            dtype_of(o, "out");
            if (o.sizes() != g.sizes() || o.scalar_type() != g.scalar_type() || !o.is_contiguous())
                throw py::value_error("out must have its gradient's shape and type, contiguous");
            on_device(o, "out", *l.like);
        }
        l.t.push_back({g.data_ptr(), o.data_ptr(), g.numel(), dt});
    }
    return l;
}

inline Tensor global_norm(const std::vector<Tensor>& grads) {
    const GradList l = grad_list(grads, nullptr);
    const int count = static_cast<int>(l.t.size());
    const Tensor norm = empty({}, *l.like, at::kFloat);
    size_t n = 0;
    ok(api.nflow_grad_workspace(count, &n), "grad_norm");
    const Tensor ws = scratch(n, *l.like);
    ok(api.nflow_grad_norm(l.t.data(), count, data<float>(norm), data(ws), n, stream_of(*l.like)), "grad_norm");
    return norm;
}

inline Tensor clip_by_global_norm(const std::vector<Tensor>& grads, double max_norm,
                                  const std::optional<std::vector<Tensor>>& out) {
    const GradList l = grad_list(grads, out ? &*out : nullptr);
    const std::vector<Tensor>& to = out ? *out : grads;
    for (const Tensor& t : to)
        if (t.requires_grad() && at::GradMode::is_enabled())
            throw py::value_error("a tensor to write to requires grad: these functions record no autograd graph");
    const int count = static_cast<int>(l.t.size());
    const Tensor norm = empty({}, *l.like, at::kFloat);
    size_t n = 0;
    ok(api.nflow_grad_workspace(count, &n), "grad_clip");
    const Tensor ws = scratch(n, *l.like);
    ok(api.nflow_grad_clip(l.t.data(), count, static_cast<float>(max_norm), data<float>(norm), data(ws), n,
                           stream_of(*l.like)), "grad_clip");
    for (const Tensor& t : to) written(t);
    return norm;
}

inline void define_residual_ops(py::module_& m) {
    m.def("residual_entry_points", &residual_entry_points);
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_fp8", &rms_norm_fp8);
    m.def("rms_norm_backward", &rms_norm_backward);
    m.def("dense_linear", &dense_linear);
    m.def("dense_linear_backward", &dense_linear_backward);
    m.def("global_norm", &global_norm);
    m.def("clip_by_global_norm", &clip_by_global_norm);
}

}  // namespace nfq_torch
