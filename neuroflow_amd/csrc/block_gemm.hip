// block_gemm.hip -- the product of 128-block FP8 codes and the linear layer
// around it, forward and backward (include/nflow_block.h).
#include "block_gemm.h"

namespace nfq {
namespace {

// 64 x 64 outputs per block of 256 threads, 4 x 4 a thread; the codes of 32
// columns at a time decoded into LDS.
template <typename TO>
__global__ __launch_bounds__(256) void k_block_matmul(BlockGemmArgs a) {
    constexpr int BT = 64, BK = 32;
    __shared__ float As[BK][BT + 1], Ws[BK][BT + 1];
    const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;
    const int64_t tn = (a.N + BT - 1) / BT;
    const int64_t m0 = blockIdx.x / tn * BT, n0 = blockIdx.x % tn * BT;
    const int64_t kb = blk_count(a.K), ld = kb * kBlk, nb = blk_count(a.N);
    float acc[4][4] = {};
    for (int64_t b = 0; b < kb; ++b) {
        float sum[4][4] = {};
        for (int k0 = 0; k0 < kBlk; k0 += BK) {
            __syncthreads();
            for (int i = tid; i < BT * BK; i += 256) {
                const int r = i / BK, k = i % BK;
                As[k][r] = m0 + r < a.M ? e4m3_decode(a.A[(m0 + r) * ld + b * kBlk + k0 + k]) : 0.0f;
                Ws[k][r] = n0 + r < a.N ? e4m3_decode(a.W[(n0 + r) * ld + b * kBlk + k0 + k]) : 0.0f;
            }
            __syncthreads();
            for (int k = 0; k < BK; ++k)
                for (int i = 0; i < 4; ++i)
                    for (int j = 0; j < 4; ++j)
                        sum[i][j] = __builtin_fmaf(As[k][tr * 4 + i], Ws[k][tc * 4 + j], sum[i][j]);
        }
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const int64_t m = m0 + tr * 4 + i, n = n0 + tc * 4 + j;
                if (m >= a.M || n >= a.N) continue;
                const float sw = a.w_blocks ? a.sW[b * nb + n / kBlk] : a.sW[b * a.N + n];
                acc[i][j] = __builtin_fmaf(sum[i][j], a.sA[b * a.M + m] * sw, acc[i][j]);
            }
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + tr * 4 + i, n = n0 + tc * 4 + j;
            if (m >= a.M || n >= a.N) continue;
            const float z = acc[i][j] + (a.bias ? a.bias[n] : 0.0f);
            static_cast<TO*>(a.C)[m * a.ldc + n] = from_f32<TO>(activate_rt(z, a.act));
        }
}

// Sum of the rows of x, a thread per column.
template <typename T>
__global__ __launch_bounds__(256) void k_column_sums(const T* __restrict__ x, int64_t M, int64_t N, int64_t ld,
                                                     float* __restrict__ out) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (n >= N) return;
    float s = 0.0f;
    for (int64_t m0 = 0; m0 < M; m0 += 256) {       // sums of 256 rows, then their sum
        float p = 0.0f;
        for (int64_t m = m0; m < m0 + 256 && m < M; ++m) p += to_f32(x[m * ld + n]);
        s += p;
    }
    out[n] = s;
}

int block_gemm(const char* what, const BlockGemmArgs& a, hipStream_t st) {
    if (a.M == 0 || a.N == 0) return NFLOW_OK;
    const int64_t tiles = ((a.M + 63) / 64) * ((a.N + 63) / 64);
    if (tiles > INT32_MAX) return bad_arg(what, "more than 2^31 - 1 tiles");
    const dim3 grid(static_cast<unsigned>(tiles)), block(256);
    if (a.out == NFLOW_DTYPE_BF16) hipLaunchKernelGGL((k_block_matmul<bf16>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_block_matmul<float>), grid, block, 0, st, a);
    return launch_status(what);
}

int check_gemm(const char* what, const BlockGemmArgs& a) {
    if (!dtype_ok(a.out)) return bad_arg(what, "unknown dtype");
    if (a.M < 0 || a.N < 0 || a.K < 0) return bad_arg(what, "bad dims");
    if (a.K > NFLOW_BLOCK_MAX_K) return bad_arg(what, "a product over more than NFLOW_BLOCK_MAX_K columns");
    if (a.act != NFLOW_ACT_NONE && a.act != NFLOW_ACT_RELU && a.act != NFLOW_ACT_GELU_TANH)
        return bad_arg(what, "unknown activation");
    if (a.ldc < a.N) return bad_arg(what, "row stride smaller than a row");
    if (a.M == 0 || a.N == 0) return NFLOW_OK;
    if (!a.C) return bad_arg(what, "null output");
    if (a.K > 0 && (!a.A || !a.sA || !a.W || !a.sW)) return bad_arg(what, "null codes or scales");
    if (!aligned(a.A, 16) || !aligned(a.W, 16)) return bad_arg(what, "codes must be 16-byte aligned");
    return NFLOW_OK;
}

// The codes and scales of a (rows, cols) matrix in a workspace.
struct BlockSpace {
    size_t codes, scales;
    BlockSpace(int64_t rows, int64_t cols)
        : codes(static_cast<size_t>(rows) * blk_count(cols) * kBlk),
          scales(round16(static_cast<size_t>(rows) * blk_count(cols) * sizeof(float))) {}
    size_t bytes() const { return codes + scales; }
};

}  // namespace
}  // namespace nfq

using namespace nfq;

extern "C" {

int nflow_fp8_block_matmul_workspace(int64_t M, int64_t N, int64_t K, int c_dtype, size_t* bytes) {
    clear_error();
    if (!bytes) return bad_arg("fp8_block_matmul_workspace", "null output");
    *bytes = 0;
    if (M < 0 || N < 0 || K < 0) return bad_arg("fp8_block_matmul_workspace", "bad dims");
    if (!dtype_ok(c_dtype)) return bad_arg("fp8_block_matmul_workspace", "unknown dtype");
    return NFLOW_OK;
}

int nflow_fp8_block_matmul(const uint8_t* A, const float* scale_A, const uint8_t* W, const float* scale_W,
                           int w_blocks, int64_t M, int64_t N, int64_t K, const float* bias, int activation,
                           void* C, int c_dtype, int64_t ldc, void* workspace, size_t workspace_bytes,
                           void* stream) {
    clear_error();
    const char* what = "fp8_block_matmul";
    const BlockGemmArgs a{A, scale_A, W, scale_W, w_blocks != 0, M, N, K, bias, activation, C, c_dtype, ldc};
    if (int rc = check_gemm(what, a)) return rc;
    size_t need = 0;
    if (int rc = nflow_fp8_block_matmul_workspace(M, N, K, c_dtype, &need)) return rc;
    if (int rc = check_workspace(what, workspace, workspace_bytes, need)) return rc;
    return block_gemm(what, a, as_stream(stream));
}

int nflow_fp8_block_linear_workspace(int64_t M, int64_t N, int64_t K, int dtype, size_t* bytes) {
    clear_error();
    if (!bytes) return bad_arg("fp8_block_linear_workspace", "null output");
    *bytes = 0;
    if (int rc = nflow_fp8_block_matmul_workspace(M, N, K, dtype, bytes)) return rc;
    *bytes = round16(*bytes) + BlockSpace(M, K).bytes();
    return NFLOW_OK;
}

int nflow_fp8_block_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* W,
                           const float* scale_W, int64_t N, const float* bias, int activation, void* y,
                           int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "fp8_block_linear";
    size_t need = 0;
    if (int rc = nflow_fp8_block_linear_workspace(M, N, K, dtype, &need)) return rc;
    if (int rc = check_workspace(what, workspace, workspace_bytes, need)) return rc;
    if (ldx < K) return bad_arg(what, "row stride smaller than a row");
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    const BlockSpace xs(M, K);
    float* scales = reinterpret_cast<float*>(codes + xs.codes);
    const BlockGemmArgs a{codes, scales, W, scale_W, true, M, N, K, bias, activation, y, dtype, ldy};
    if (int rc = check_gemm(what, a)) return rc;
    if (M == 0 || N == 0) return NFLOW_OK;
    if (K > 0) {
        if (!x) return bad_arg(what, "null x");
        if (int rc = block_quantise(what, x, dtype, M, K, ldx, codes, scales, nullptr, nullptr, as_stream(stream)))
            return rc;
    }
    return block_gemm(what, a, as_stream(stream));
}

int nflow_fp8_block_linear_backward_workspace(int64_t M, int64_t N, int64_t K, int dtype, size_t* bytes) {
    clear_error();
    if (!bytes) return bad_arg("fp8_block_linear_backward_workspace", "null output");
    *bytes = 0;
    size_t dx = 0, dw = 0;
    if (int rc = nflow_fp8_block_matmul_workspace(M, K, N, dtype, &dx)) return rc;
    if (int rc = nflow_fp8_block_matmul_workspace(N, K, M, NFLOW_DTYPE_F32, &dw)) return rc;
    *bytes = round16(std::max(dx, dw)) + BlockSpace(M, N).bytes() + BlockSpace(N, M).bytes();
    return NFLOW_OK;
}

int nflow_fp8_block_linear_backward(const void* dy, int dtype, int64_t M, int64_t N, int64_t lddy,
                                    const uint8_t* x_t, const float* scale_x_t, const uint8_t* W_t,
                                    const float* scale_W_t, int64_t K, void* dx, int64_t lddx, float* dW,
                                    float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "fp8_block_linear_backward";
    size_t need = 0;
    if (int rc = nflow_fp8_block_linear_backward_workspace(M, N, K, dtype, &need)) return rc;
    if (int rc = check_workspace(what, workspace, workspace_bytes, need)) return rc;
    if (lddy < N) return bad_arg(what, "row stride smaller than a row");
    if (M > 0 && N > 0 && !dy) return bad_arg(what, "null dy");
    hipStream_t st = as_stream(stream);
    uint8_t* q = static_cast<uint8_t*>(workspace);
    const BlockSpace rows(M, N), cols(N, M);
    float* sq = reinterpret_cast<float*>(q + rows.codes);
    uint8_t* t = q + rows.bytes();
    float* stt = reinterpret_cast<float*>(t + cols.codes);
    const BlockGemmArgs ax{q, sq, W_t, scale_W_t, true, M, K, N, nullptr, NFLOW_ACT_NONE, dx, dtype, lddx};
    const BlockGemmArgs aw{t, stt, x_t, scale_x_t, false, N, K, M, nullptr, NFLOW_ACT_NONE, dW, NFLOW_DTYPE_F32, K};
    if (dx)
        if (int rc = check_gemm(what, ax)) return rc;
    if (dW)
        if (int rc = check_gemm(what, aw)) return rc;
    if (M > 0 && N > 0 && (dx || dW))
        if (int rc = block_quantise(what, dy, dtype, M, N, lddy, dx ? q : nullptr, dx ? sq : nullptr,
                                    dW ? t : nullptr, dW ? stt : nullptr, st))
            return rc;
    if (dbias && N > 0) {
        const dim3 grid(static_cast<unsigned>((N + 255) / 256)), block(256);
        if (dtype == NFLOW_DTYPE_BF16)
            hipLaunchKernelGGL((k_column_sums<bf16>), grid, block, 0, st, static_cast<const bf16*>(dy), M, N, lddy, dbias);
        else
            hipLaunchKernelGGL((k_column_sums<float>), grid, block, 0, st, static_cast<const float*>(dy), M, N, lddy, dbias);
        if (int rc = launch_status(what)) return rc;
    }
    if (dx)
        if (int rc = block_gemm(what, ax, st)) return rc;
    if (dW)
        if (int rc = block_gemm(what, aw, st)) return rc;
    return NFLOW_OK;
}

}  // extern "C"
