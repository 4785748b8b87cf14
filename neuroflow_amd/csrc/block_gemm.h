// block_gemm.h -- arguments of the block-FP8 product, and the launchers its
// translation units share.
#pragma once

#include "block_dev.h"

namespace nfq {

// C = act(A W^T + bias); codes in rows of 128 * blk_count(K) bytes, scales
// (blk_count(K), M) and (blk_count(K), w_blocks ? blk_count(N) : N).
struct BlockGemmArgs {
    const uint8_t* A;
    const float* sA;
    const uint8_t* W;
    const float* sW;
    bool w_blocks;
    int64_t M, N, K;
    const float* bias;
    int act;
    void* C;
    int out;            // nflow_dtype of C
    int64_t ldc;
};

// x along its rows and / or columns (block_quantise.hip); arguments checked by
// the caller, M, K > 0.  col_sums (blk_count(M), K): also the sums of each 128
// rows of every column.
int block_quantise(const char* what, const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* codes,
                   float* scales, uint8_t* codes_t, float* scales_t, float* col_sums, hipStream_t st);

// The product for few rows (block_few.hip): from codes, and from the values of
// x (of C's type, row stride ldx) quantised on the way, W in 128 x 128 blocks.
void launch_block_few(const BlockGemmArgs& a, hipStream_t st);
bool few_values(int64_t M, int64_t K);
void launch_block_few_values(const BlockGemmArgs& a, const void* x, int64_t ldx, hipStream_t st);

// And for many rows of few K blocks, from the values (block_rows.hip).
bool many_rows_values(int64_t M, int64_t N, int64_t K, int dtype);
void launch_block_rows(const BlockGemmArgs& a, const void* x, int64_t ldx, hipStream_t st);
unsigned block_rows_grid(int64_t M, int64_t N);      // its workgroups

}  // namespace nfq
