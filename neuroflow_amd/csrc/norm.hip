// norm.hip -- layer norm, forward (to the activation's type or straight to
// 128-block FP8) and backward (include/nflow_block.h).
#include "block_dev.h"

namespace nfq {
namespace {

constexpr int kNormThreads = 256;

// Sum over the block; every thread gets it.  `part` holds a value per wave.
__device__ __forceinline__ float block_sum(float v, float* part) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kNormThreads / 64; ++w) s += part[w];
    return s;
}

struct NormArgs {
    const void* x;
    int64_t M, D, ldx;
    const float* weight;
    const float* bias;
    float eps;
    void* y;
    int64_t ldy;
    uint8_t* codes;
    float* scales;
    float* mean;
    float* rstd;
};

// One block per row, three passes over it: the sum, the squares about the
// mean, the result.
template <typename T, bool FP8>
__global__ __launch_bounds__(kNormThreads) void k_norm_rows(NormArgs a) {
    __shared__ float part[kNormThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
        float s = 0.0f;
        for (int64_t c = tid; c < a.D; c += kNormThreads) s += to_f32(x[c]);
        const float mean = block_sum(s, part) / static_cast<float>(a.D);
        float q = 0.0f;
        for (int64_t c = tid; c < a.D; c += kNormThreads) {
            const float d = to_f32(x[c]) - mean;
            q += d * d;
        }
        const float rstd = 1.0f / sqrtf(block_sum(q, part) / static_cast<float>(a.D) + a.eps);
        if (tid == 0) {
            if (a.mean) a.mean[m] = mean;
            if (a.rstd) a.rstd[m] = rstd;
        }
        auto value = [&](int64_t c) {
            const float h = (to_f32(x[c]) - mean) * rstd;
            return h * (a.weight ? a.weight[c] : 1.0f) + (a.bias ? a.bias[c] : 0.0f);
        };
        if constexpr (!FP8) {
            T* y = static_cast<T*>(a.y) + m * a.ldy;
            for (int64_t c = tid; c < a.D; c += kNormThreads) y[c] = from_f32<T>(value(c));
        } else {
            const int64_t kb = blk_count(a.D);
            for (int64_t b = wave; b < kb; b += kNormThreads / 64) {
                const int64_t c = b * kBlk + 2 * lane;
                const float v0 = c < a.D ? value(c) : 0.0f, v1 = c + 1 < a.D ? value(c + 1) : 0.0f;
                const float sc = blk_scale(wave_max(amax_of(amax_of(0.0f, v0), v1)));
                const float inv = 1.0f / sc;
                const uint32_t w = fp8_quant(v0, inv) | fp8_quant(v1, inv) << 8;
                *reinterpret_cast<uint16_t*>(a.codes + m * kb * kBlk + c) =
                    static_cast<uint16_t>(c + 1 < a.D ? w : (c < a.D ? w & 0xFFu : 0u));
                if (lane == 0) a.scales[b * a.M + m] = sc;
            }
        }
    }
}

struct NormGradArgs {
    const void* dy;
    const void* x;
    int64_t M, D, lddy, ldx;
    const float* weight;
    const float* mean;
    const float* rstd;
    void* dx;
    int64_t lddx;
    float* part;        // (blocks, 2, D) partial dweight, dbias
    int64_t rows_per;   // rows of a block's share
    float* dweight;
    float* dbias;
};

// dx, one block per row.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void k_norm_grad_rows(NormGradArgs a) {
    __shared__ float part[kNormThreads / 64];
    const int tid = threadIdx.x;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
        const T* dy = static_cast<const T*>(a.dy) + m * a.lddy;
        T* dx = static_cast<T*>(a.dx) + m * a.lddx;
        const float mean = a.mean[m], rstd = a.rstd[m];
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t c = tid; c < a.D; c += kNormThreads) {
            const float g = to_f32(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            s1 += g;
            s2 += g * ((to_f32(x[c]) - mean) * rstd);
        }
        const float c1 = block_sum(s1, part) / static_cast<float>(a.D);
        const float c2 = block_sum(s2, part) / static_cast<float>(a.D);
        for (int64_t c = tid; c < a.D; c += kNormThreads) {
            const float g = to_f32(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            const float h = (to_f32(x[c]) - mean) * rstd;
            dx[c] = from_f32<T>(rstd * (g - c1 - h * c2));
        }
    }
}

// Partial sums of dy * h and dy over a block's rows, a thread per column.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void k_norm_grad_params(NormGradArgs a) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x;
    if (c >= a.D) return;
    const int64_t m0 = blockIdx.y * a.rows_per, m1 = m0 + a.rows_per < a.M ? m0 + a.rows_per : a.M;
    float dw = 0.0f, db = 0.0f;
    for (int64_t m = m0; m < m1; ++m) {
        const float g = to_f32(static_cast<const T*>(a.dy)[m * a.lddy + c]);
        dw += g * ((to_f32(static_cast<const T*>(a.x)[m * a.ldx + c]) - a.mean[m]) * a.rstd[m]);
        db += g;
    }
    a.part[blockIdx.y * 2 * a.D + c] = dw;
    a.part[(blockIdx.y * 2 + 1) * a.D + c] = db;
}

// Sum of the blocks' partials, in their order.
__global__ __launch_bounds__(kNormThreads) void k_norm_grad_join(NormGradArgs a, int64_t blocks) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x;
    if (c >= a.D) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t b = 0; b < blocks; ++b) {
        dw += a.part[b * 2 * a.D + c];
        db += a.part[(b * 2 + 1) * a.D + c];
    }
    if (a.dweight) a.dweight[c] = dw;
    if (a.dbias) a.dbias[c] = db;
}

int64_t grad_blocks(int64_t M) { return std::min<int64_t>(M, 256); }

unsigned row_grid(int64_t M) { return static_cast<unsigned>(std::min<int64_t>(M, 8 * num_cus())); }

int check_norm(const char* what, const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, float eps) {
    if (!dtype_ok(dtype)) return bad_arg(what, "unknown dtype");
    if (M < 0 || D <= 0) return bad_arg(what, "bad dims");
    if (ldx < D) return bad_arg(what, "row stride smaller than a row");
    if (!(eps >= 0.0f)) return bad_arg(what, "eps must not be negative or NaN");
    if (M > 0 && !x) return bad_arg(what, "null x");
    return NFLOW_OK;
}

template <bool FP8>
int norm_forward(const char* what, const NormArgs& a, int dtype, void* stream) {
    hipStream_t st = as_stream(stream);
    if (dtype == NFLOW_DTYPE_BF16)
        hipLaunchKernelGGL((k_norm_rows<bf16, FP8>), dim3(row_grid(a.M)), dim3(kNormThreads), 0, st, a);
    else
        hipLaunchKernelGGL((k_norm_rows<float, FP8>), dim3(row_grid(a.M)), dim3(kNormThreads), 0, st, a);
    return launch_status(what);
}

}  // namespace
}  // namespace nfq

using namespace nfq;

extern "C" {

int nflow_layer_norm_forward(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const float* weight,
                             const float* bias, float eps, void* y, int64_t ldy, float* mean, float* rstd,
                             void* stream) {
    clear_error();
    const char* what = "layer_norm_forward";
    if (int rc = check_norm(what, x, dtype, M, D, ldx, eps)) return rc;
    if (ldy < D) return bad_arg(what, "row stride smaller than a row");
    if (M == 0) return NFLOW_OK;
    if (!y) return bad_arg(what, "null y");
    return norm_forward<false>(what, NormArgs{x, M, D, ldx, weight, bias, eps, y, ldy, nullptr, nullptr, mean, rstd},
                               dtype, stream);
}

int nflow_layer_norm_fp8_block(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const float* weight,
                               const float* bias, float eps, uint8_t* codes, float* scales, float* mean,
                               float* rstd, void* stream) {
    clear_error();
    const char* what = "layer_norm_fp8_block";
    if (int rc = check_norm(what, x, dtype, M, D, ldx, eps)) return rc;
    if (M == 0) return NFLOW_OK;
    if (!codes || !scales) return bad_arg(what, "null codes or scales");
    if (!aligned(codes, 16)) return bad_arg(what, "codes must be 16-byte aligned");
    return norm_forward<true>(what, NormArgs{x, M, D, ldx, weight, bias, eps, nullptr, 0, codes, scales, mean, rstd},
                              dtype, stream);
}

int nflow_layer_norm_backward_workspace(int64_t M, int64_t D, size_t* bytes) {
    clear_error();
    if (!bytes) return bad_arg("layer_norm_backward_workspace", "null output");
    *bytes = 0;
    if (M < 0 || D <= 0) return bad_arg("layer_norm_backward_workspace", "bad dims");
    *bytes = static_cast<size_t>(grad_blocks(M)) * 2 * static_cast<size_t>(D) * sizeof(float);
    return NFLOW_OK;
}

int nflow_layer_norm_backward(const void* dy, const void* x, int dtype, int64_t M, int64_t D, int64_t lddy,
                              int64_t ldx, const float* weight, const float* mean, const float* rstd, void* dx,
                              int64_t lddx, float* dweight, float* dbias, void* workspace, size_t workspace_bytes,
                              void* stream) {
    clear_error();
    const char* what = "layer_norm_backward";
    if (int rc = check_norm(what, x, dtype, M, D, ldx, 0.0f)) return rc;
    if (lddy < D || lddx < D) return bad_arg(what, "row stride smaller than a row");
    if (M > 0 && (!dy || !mean || !rstd || !dx)) return bad_arg(what, "null dy, mean, rstd or dx");
    size_t need = 0;
    if (int rc = nflow_layer_norm_backward_workspace(M, D, &need)) return rc;
    if (int rc = check_workspace(what, workspace, workspace_bytes, need)) return rc;
    hipStream_t st = as_stream(stream);
    const int64_t nb = grad_blocks(M);
    NormGradArgs a{dy, x, M, D, lddy, ldx, weight, mean, rstd, dx, lddx, static_cast<float*>(workspace),
                   nb ? (M + nb - 1) / nb : 0, dweight, dbias};
    const unsigned gc = static_cast<unsigned>((D + kNormThreads - 1) / kNormThreads);
    if (M > 0) {
        const dim3 grid(row_grid(M)), gp(gc, static_cast<unsigned>(nb)), block(kNormThreads);
        if (dtype == NFLOW_DTYPE_BF16) {
            if (dweight || dbias) hipLaunchKernelGGL((k_norm_grad_params<bf16>), gp, block, 0, st, a);
            hipLaunchKernelGGL((k_norm_grad_rows<bf16>), grid, block, 0, st, a);
        } else {
            if (dweight || dbias) hipLaunchKernelGGL((k_norm_grad_params<float>), gp, block, 0, st, a);
            hipLaunchKernelGGL((k_norm_grad_rows<float>), grid, block, 0, st, a);
        }
    }
    if (dweight || dbias) hipLaunchKernelGGL(k_norm_grad_join, dim3(gc), dim3(kNormThreads), 0, st, a, nb);
    return launch_status(what);
}

}  // extern "C"
