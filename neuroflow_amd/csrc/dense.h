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
};

// Which operands lie across k: the layer's three products.
enum DenseForm { DENSE_FORWARD = 0, DENSE_DX = 1, DENSE_DW = 2 };

// How a product is cut: the kernel or tile, and the runs that K is split into
// (joined by a second launch).
enum DenseKind { DENSE_FEW, DENSE_SMALL, DENSE_MID, DENSE_BIG };
struct DensePlan {
    DenseKind kind;
    int splits;
    size_t bytes;       // of the partial results
};

// The tiled product, one translation unit per type.
template <typename T>
void launch_dense(const DenseArgs& a, DenseForm form, const DensePlan& p, float* part, hipStream_t st);

// The product for few rows, operands along k (dense_few.hip).
constexpr int64_t kDenseFewRows = 64;
template <typename T>
void launch_dense_few(const DenseArgs& a, hipStream_t st);

}  // namespace nfq
