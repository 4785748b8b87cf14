/*
 * nflow_block.h -- C-ABI of layer norm and of the linear layer in 128-block
 * FP8: the norm in front of a projection, its output or any activation as
 * E4M3 codes with a scale for every 128 values, the product of such codes,
 * and the backward pass of each.
 *
 * The conventions are those of nflow_quant.h: status codes and
 * nflow_last_error(), DEVICE pointers, kernels enqueued on `stream`, no
 * synchronisation.  Nothing here allocates: an entry point that needs scratch
 * takes `workspace` (16-byte aligned device memory, its contents of no matter
 * before and after) of at least the bytes its _workspace function names, and
 * NULL where that is 0.  Calls that may overlap in time need a workspace
 * each.  Every entry point may be recorded into a HIP graph.  Results do not
 * depend on timing: the same call on the same device gives the same bits.
 *
 * Types: NFLOW_DTYPE_F32 and NFLOW_DTYPE_BF16 for activations and their
 * gradients; parameters (weight, bias of the norm, bias of the layer) and
 * their gradients are fp32.  Rows are contiguous; ldx, ldy, ... are the
 * elements from one row to the next (at least the row's length), and rows
 * need no alignment beyond that of their elements.
 *
 * Block FP8.  A matrix of R rows and K columns is held as
 *   codes   R rows of 128 * ceil(K / 128) E4M3 bytes, the bytes past K zero,
 *           16-byte aligned;
 *   scales  fp32, ceil(K / 128) rows of R (a scale for every 128 values of a
 *           row), or of ceil(R / 128) (a weight: for every 128 x 128 block).
 * A value is its code's times the scale.  The scale of a block is absmax / 448,
 * or 1 where absmax < 448 * 2^-126 (an all-zero block among them); its codes
 * are fp32_to_e4m3_bits(clamp(x * (1 / scale), -448, 448)) as
 * nflow_fp8_quantise_per_token's (cpp/include/neuroflow/fp8_e4m3.h:106-215,
 * 319-327).  A NaN takes the NaN code and leaves the scale to the others; an
 * infinity makes its block's scale infinite, and so all of the block NaN.
 * There is no counterpart in the reference, whose scales are per tensor,
 * channel or token (cpp/include/neuroflow/int8_gemm.h:45-65).
 */
#ifndef NFLOW_BLOCK_H
#define NFLOW_BLOCK_H

#include <stddef.h>
#include <stdint.h>

#include "nflow_quant.h"

#ifdef __cplusplus
extern "C" {
#endif

enum nflow_dtype {
    NFLOW_DTYPE_F32 = 0,
    NFLOW_DTYPE_BF16 = 1
};

/* Columns a block-FP8 matrix may have (the length a product sums over). */
#define NFLOW_BLOCK_MAX_K ((int64_t)1 << 22)

/* ---- layer norm (the norm of cpp/src/fno.cpp:1418-1438, and its gradient) ---- */

/* y = (x - mean) * rstd * weight + bias over the D columns of each of M rows,
 * mean and rstd = 1 / sqrt(var + eps) in fp32 (var the mean of squares about
 * the mean).  weight, bias (D) may be NULL (ones, zeros); mean, rstd (M) may
 * be NULL (not wanted).  y may be x, at the same row stride; rows that overlap
 * x's in any other way are refused. */
int nflow_layer_norm_forward(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const float* weight,
                             const float* bias, float eps, void* y, int64_t ldy, float* mean, float* rstd,
                             void* stream);

/* The same y as block-FP8 codes and scales (ceil(D / 128), M), quantised from
 * its fp32 value: y itself is never rounded to x's type or written. */
int nflow_layer_norm_fp8_block(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const float* weight,
                               const float* bias, float eps, uint8_t* codes, float* scales, float* mean,
                               float* rstd, void* stream);

/* With g = dy * weight and h = (x - mean) * rstd:
 *   dx = rstd * (g - mean_D(g) - h * mean_D(g * h)),
 *   dweight = sum_M(dy * h), dbias = sum_M(dy)
 * from the mean and rstd of the forward pass.  weight may be NULL (ones);
 * dweight and dbias (D) may each be NULL (not wanted).  dx may be dy or x,
 * as y may be x above.
 * M = 0 gives zero dweight and dbias. */
int nflow_layer_norm_backward(const void* dy, const void* x, int dtype, int64_t M, int64_t D, int64_t lddy,
                              int64_t ldx, const float* weight, const float* mean, const float* rstd, void* dx,
                              int64_t lddx, float* dweight, float* dbias, void* workspace, size_t workspace_bytes,
                              void* stream);
int nflow_layer_norm_backward_workspace(int64_t M, int64_t D, size_t* bytes);

/* ---- 128-block FP8 ---- */

/* x (M, K) to codes and scales along its rows (codes, scales) and / or along
 * its columns (codes_t (K rows of 128 * ceil(M / 128)), scales_t
 * (ceil(M / 128), K)): the form the transpose of x takes in a product.  A pair
 * that is not wanted is NULL.  Both come from one read of x. */
int nflow_fp8_block_quantise(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* codes,
                             float* scales, uint8_t* codes_t, float* scales_t, void* stream);

/* A weight W (N, K) with a scale for every 128 x 128 block: codes, scales
 * (ceil(K / 128), ceil(N / 128)), and, unless codes_t is NULL, the same codes
 * and scales transposed (codes_t: K rows of 128 * ceil(N / 128); scales_t:
 * (ceil(N / 128), ceil(K / 128))), which the backward pass multiplies by. */
int nflow_fp8_block_quantise_weight(const void* W, int dtype, int64_t N, int64_t K, int64_t ldw, uint8_t* codes,
                                    float* scales, uint8_t* codes_t, float* scales_t, void* stream);

/* C = act(A W^T + bias): A (M, K) with scales (ceil(K / 128), M), W (N, K) with
 * scales (ceil(K / 128), N), or with w_blocks != 0 (ceil(K / 128), ceil(N /
 * 128)).  Each 128 columns' products are summed by the matrix cores, scaled
 * in fp32 and summed in fp32; C is rounded once, to c_dtype.  An fp32 C comes
 * from bf16 matrix instructions on the codes' exact values (products and sums
 * to fp32 accuracy).  A bf16 C comes from FP8 ones, which drop low bits of what
 * they sum: 128 products' sum is off by at most 2^-12 of the sum of their
 * magnitudes.  On normal data the error is 1.3e-5 of C (2-norm) where rounding
 * C to bf16 is 1.7e-3; but it goes by the magnitudes and not by the result,
 * and where products cancel it can pass bf16's rounding of what is left (the
 * bound does from |C| < 1/8 of the magnitudes on).  c_dtype fp32 has neither;
 * linear and linear_backward follow x's and dy's type (dW is always fp32).
 * The product of two blocks' scales has to lie in fp32's normal range.
 * bias (N) may be NULL. */
int nflow_fp8_block_matmul(const uint8_t* A, const float* scale_A, const uint8_t* W, const float* scale_W,
                           int w_blocks, int64_t M, int64_t N, int64_t K, const float* bias, int activation,
                           void* C, int c_dtype, int64_t ldc, void* workspace, size_t workspace_bytes,
                           void* stream);
int nflow_fp8_block_matmul_workspace(int64_t M, int64_t N, int64_t K, int c_dtype, size_t* bytes);

/* y = act(q(x) W^T + bias), q the quantise above: x (M, K) and y (M, N) of
 * one type, W a weight in 128 x 128 blocks.  A few rows, and many rows of up to
 * 512 columns where that is faster, are one launch; the workspace has room for
 * x's codes past a few rows either way. */
int nflow_fp8_block_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* W,
                           const float* scale_W, int64_t N, const float* bias, int activation, void* y,
                           int64_t ldy, void* workspace, size_t workspace_bytes, void* stream);
int nflow_fp8_block_linear_workspace(int64_t M, int64_t N, int64_t K, int dtype, size_t* bytes);

/* The gradients of y = q(x) W^T + bias (no activation) from dy (M, N):
 *   dx (M, K), of dy's type = q(dy) W, W as quantise_weight's transposed
 *     (W_t: K rows of 128 * ceil(N / 128) codes, scale_W_t);
 *   dW (N, K), fp32 = q(dy^T) q(x^T)^T, x as quantise's column pair (x_t: K
 *     rows of 128 * ceil(M / 128) codes, scale_x_t);
 *   dbias (N) = the sum of dy's rows, before any quantise.
 * The quantise passes its gradient straight through.  dx, dW and dbias may
 * each be NULL (not wanted; their inputs may then be NULL too).  M = 0 gives
 * zero dW and dbias. */
int nflow_fp8_block_linear_backward(const void* dy, int dtype, int64_t M, int64_t N, int64_t lddy,
                                    const uint8_t* x_t, const float* scale_x_t, const uint8_t* W_t,
                                    const float* scale_W_t, int64_t K, void* dx, int64_t lddx, float* dW,
                                    float* dbias, void* workspace, size_t workspace_bytes, void* stream);
int nflow_fp8_block_linear_backward_workspace(int64_t M, int64_t N, int64_t K, int dtype, size_t* bytes);

/* ---- for tests: which kernel a size takes (no GPU needed: 256 CUs without one) ---- */

/* The tile edge of matmul's kernel at this size, 64, 128 or 256, or 0 for the
 * few-row kernel; and the runs that the K blocks are split into. */
int nflow_debug_fp8_block_cut(int64_t M, int64_t N, int64_t K, int c_dtype, int* edge, int* splits);
/* What linear runs: 0 the few-row kernel on x's values, 1 the kernel of many
 * rows on x's values, with its workgroups, 2 the quantise and matmul's kernel. */
int nflow_debug_fp8_block_linear_kernel(int64_t M, int64_t N, int64_t K, int dtype, int* kernel, int* workgroups);

#ifdef __cplusplus
}
#endif
#endif /* NFLOW_BLOCK_H */
