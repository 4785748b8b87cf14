/*
 * nflow_residual.h -- C-ABI of what stands around the quantised layers of a
 * residual block: RMS norm with the residual's addition (also straight to
 * 128-block FP8), the linear layer in bf16 or fp32 with bias, residual and
 * activation in its epilogue, the backward pass of each, and the clipping of
 * gradients by their global norm.
 *
 * The conventions are those of nflow_block.h: status codes and
 * nflow_last_error(), DEVICE pointers, kernels enqueued on `stream`, no
 * synchronisation and no allocation; `workspace` is 16-byte aligned device
 * memory of at least the bytes that the _workspace function names, one per call
 * in flight, its contents of no matter before and after.  Every entry point may
 * be recorded into a HIP graph.  The same call on the same device gives the same
 * bits.  Activations are NFLOW_DTYPE_F32 or NFLOW_DTYPE_BF16; rows are
 * contiguous, ld* the elements from one row to the next, and rows need no
 * alignment beyond that of their elements.  Matrices that are columns of one buffer,
 * at one row stride, share no memory; those of different strides are taken to where
 * the memory that they span does.  There is no counterpart in the
 * reference, whose norm is a layer norm (cpp/src/fno.cpp:1418-1438) and whose
 * linear layers run on a CPU.
 */
#ifndef NFLOW_RESIDUAL_H
#define NFLOW_RESIDUAL_H

#include <stddef.h>
#include <stdint.h>

#include "nflow_block.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- RMS norm ---- */

/* t = x + residual (fp32; residual NULL: t = x), rstd = 1 / sqrt(mean_D(t^2) +
 * eps), y = t * rstd * weight over the D columns of each of M rows.  The norm is
 * of t before its rounding; its squares are summed in fp32, so a row whose sum of
 * them is past fp32's range (values from 1.8e19 on) has rstd 0.  sum, of x's type,
 * takes the rounded t; it is wanted only with a residual and may be NULL, as weight
 * (ones) and rstd (M) may.  sum and y may each be x or residual at the same row
 * stride, but not one another; memory that a result shares in any other way is
 * refused. */
int nflow_rms_norm_forward(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const void* residual,
                           int64_t ldr, const float* weight, float eps, void* y, int64_t ldy, void* sum,
                           int64_t ldsum, float* rstd, void* stream);

/* The same y as block-FP8 codes and scales (ceil(D / 128), M), as
 * nflow_layer_norm_fp8_block's: quantised from its fp32 value. */
int nflow_rms_norm_fp8(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const void* residual,
                       int64_t ldr, const float* weight, float eps, uint8_t* codes, float* scales, void* sum,
                       int64_t ldsum, float* rstd, void* stream);

/* With t what was normed (sum, or x), g = dy * weight and h = t * rstd:
 *   dt = rstd * (g - h * mean_D(g * h)) + dsum,   dweight = sum_M(dy * h).
 * dt is the gradient of x and of residual alike; dsum (NULL: 0) is what t has
 * from its other use, the residual stream.  weight may be NULL (ones), dweight
 * (D) NULL (not wanted).  dt may be dy, t or dsum at the same row stride; dt and
 * dweight share no other memory with an input or one another.  M = 0 gives zero
 * dweight. */
int nflow_rms_norm_backward(const void* dy, const void* t, int dtype, int64_t M, int64_t D, int64_t lddy,
                            int64_t ldt, const float* weight, const float* rstd, const void* dsum, int64_t lddsum,
                            void* dt, int64_t lddt, float* dweight, void* workspace, size_t workspace_bytes,
                            void* stream);
int nflow_rms_norm_backward_workspace(int64_t M, int64_t D, size_t* bytes);

/* ---- the linear layer in bf16 or fp32 ---- */

/* Columns a product may sum over. */
#define NFLOW_DENSE_MAX_K ((int64_t)1 << 21)

/* z = x W^T + bias + residual, y = act(z): x (M, K), W (N, K), residual, y and
 * pre (M, N) of one type, bias (N) fp32.  The residual joins ahead of the
 * activation, as in nflow_layer_forward_residual.  pre takes z, which the
 * backward pass of an activation needs.  bias, residual and pre may be NULL.
 * Sums are fp32; bf16 products are exact.  fp32 products are formed from three
 * bf16 parts of each operand, which hold it exactly (below 2^-110 to 2^-134, half
 * a step of bf16's subnormals), without the three smallest of nine (at most 2^-24 of
 * a product, half a step of fp32); an infinite operand gives NaN there, as a NaN
 * does, with ReLU too.  y may be residual at the same row stride; y and pre may
 * share no other memory with an input or one another.  A bf16 operand x or W whose
 * address, row stride and row are not whole 16-byte groups, or whose stride is
 * NFLOW_DENSE_MAX_K or more, is copied into the workspace first, but for a call of few
 * rows that is faster without.  `copies` asks for the room: 0 where neither is such, 2
 * where those that are lie at addresses and strides of whole 4-byte words, else 1. */
int nflow_dense_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* W, int64_t ldw,
                       int64_t N, const float* bias, const void* residual, int64_t ldr, int activation, void* y,
                       int64_t ldy, void* pre, int64_t ldpre, void* workspace, size_t workspace_bytes,
                       void* stream);
int nflow_dense_linear_workspace(int64_t M, int64_t N, int64_t K, int dtype, int copies, size_t* bytes);

/* The gradients of nflow_dense_linear from dy (M, N):
 *   dz = dy * act'(pre) (M, N), the gradient of residual too,
 *   dx (M, K) = dz W,  dW (N, K) = dz^T x,  dbias (N, fp32) = the sum of dz's rows.
 * dz, dx and dW are of dy's type, and the products take dz as it is returned;
 * dbias sums it ahead of its rounding.  In fp32 the products, and with no activation
 * dbias too, are of three parts of each operand, as above.  With no activation dz is
 * dy and both dz and pre are NULL; with one both are required (for ReLU pre may be
 * y).  dx, dW and dbias may each be NULL (not wanted).  M = 0 gives zero dW and
 * dbias, N = 0 zero dx.
 * dz may be dy or pre at the same row stride; results share no other memory
 * with an input or one another.  `copies` as above, for dz (or dy), x and W. */
int nflow_dense_linear_backward(const void* dy, int dtype, int64_t M, int64_t N, int64_t lddy, const void* x,
                                int64_t ldx, const void* W, int64_t ldw, int64_t K, int activation, const void* pre,
                                int64_t ldpre, void* dz, int64_t lddz, void* dx, int64_t lddx, void* dW,
                                int64_t lddw, float* dbias, void* workspace, size_t workspace_bytes, void* stream);
int nflow_dense_linear_backward_workspace(int64_t M, int64_t N, int64_t K, int dtype, int copies, size_t* bytes);

/* ---- gradient clipping ---- */

/* A gradient of `count` contiguous elements; out: where the clipped one goes
 * (grad itself to clip in place). */
typedef struct nflow_grad_tensor {
    const void* grad;
    void* out;
    int64_t count;
    int dtype;
} nflow_grad_tensor;

/* *norm (device, fp32) = the root of the sum of squares over all tensors, taken
 * in 64 bits (no square over- or underflows) and rounded once.  out is not
 * read.  The table is host memory, read before the call returns. */
int nflow_grad_norm(const nflow_grad_tensor* tensors, int count, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream);

/* The same norm, and each gradient times min(1, max_norm / norm), the factor
 * rounded to fp32.  Where that is 1, gradients clipped in place are not touched.
 * A NaN in any gradient makes all of them NaN, an infinity makes finite ones 0
 * and itself NaN (their norm says so); with an infinite max_norm and no NaN all are
 * left as they are.  An out that is not its own grad, and norm, share no memory with
 * any gradient or other out. */
int nflow_grad_clip(const nflow_grad_tensor* tensors, int count, float max_norm, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream);

/* For both, of `count` tensors. */
int nflow_grad_workspace(int count, size_t* bytes);

/* ---- for tests: which kernel a size takes (no GPU needed: 256 CUs without one) ---- */

/* The kernel of the linear layer's product at this size, of operands in whole 16-byte
 * groups: 0 the few-row one, else
 * tiles of 64 x 64 (1), 128 x 64 (2, bf16), 128 x 128 (3; 4 the same with its loads
 * further ahead, bf16) or 256 x 256 (5; fp32 256 x 128); and the workgroups that
 * tiles' K steps are dealt out to, or 0 where tiles stay whole.  form: 0 forward,
 * 1 dx (M, K, N of the layer as M, N, K), 2 dW (N, K, M), 3 both in one launch (the
 * layer's M, N, K; groups 0: they are not). */
int nflow_debug_dense_cut(int form, int64_t M, int64_t N, int64_t K, int dtype, int* kernel, int* groups);

#ifdef __cplusplus
}
#endif
#endif /* NFLOW_RESIDUAL_H */
