// dense.h -- arguments of the bf16 / fp32 product, and the launchers its
// translation units share.
#pragma once

#include "block_dev.h"
#include "nflow_residual.h"

namespace nfq {

// C (M, N) = act(sum_k a(m, k) b(n, k) + bias + R), the operands of C's type.
// An operand lies along k (element (m, k) at m ld + k), or across it (k ld + m).
struct DenseArgs {
    const void* A;
    const void* B;
    int64_t lda, ldb;
    int64_t M, N, K;
    const float* bias;
    const void* R;
    int64_t ldr;
    int act;
    void* C;
    int64_t ldc;
    void* Z;            // the sum ahead of the activation, or null
    int64_t ldz;
    float* sums;        // of a(m, .) for every m, or null (of the dW form)
};

// Which operands lie across k: the layer's three products.
enum DenseForm { DENSE_FORWARD = 0, DENSE_DX = 1, DENSE_DW = 2 };

// How a product is cut: the kernel or tile, and, unless 0, the workgroups that
// the tiles and the K steps of what is left of them are dealt out to.
enum DenseKind { DENSE_FEW, DENSE_SMALL, DENSE_TALL, DENSE_MID, DENSE_DEEP, DENSE_BIG };
struct DensePlan {
    DenseKind kind;
    int groups;
    size_t bytes;       // of the shared tiles' partial results
    double us;          // estimated
};

// The tiled product, one translation unit per type.
void launch_dense_bf16(const DenseArgs& a, DenseForm form, const DensePlan& p, float* part, hipStream_t st);
void launch_dense_f32(const DenseArgs& a, DenseForm form, const DensePlan& p, float* part, hipStream_t st);
// dx and dW by one launch, their K steps dealt out to p.groups workgroups.
void launch_dense_pair_f32(const DenseArgs& dx, const DenseArgs& dw, const DensePlan& p, float* part, hipStream_t st);

// A bf16 operand as the tiled product can fetch it: whole 16-byte groups at
// 16-byte places, and a tile's rows within a buffer's range.
inline bool dense_fetchable(const void* p, int64_t ld, int64_t cols) {
    return aligned(p, 16) && ld % 8 == 0 && cols % 8 == 0 && ld < NFLOW_DENSE_MAX_K;
}
// Others are copied into rows of this many values.
__host__ __device__ inline int64_t dense_pitch(int64_t cols) { return (cols + 7) / 8 * 8; }
struct DensePack {
    const void* from;
    void* to;
    int64_t rows, cols, ld;
};
void launch_dense_pack(const DensePack (&m)[3], hipStream_t st);

// The product for few rows, operands along k (dense_few.hip).
constexpr int64_t kDenseFewRows = 32;
template <typename T>
void launch_dense_few(const DenseArgs& a, hipStream_t st);

}  // namespace nfq
