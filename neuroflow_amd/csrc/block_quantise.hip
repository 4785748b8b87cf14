// block_quantise.hip -- activations and weights to 128-block FP8
// (include/nflow_block.h).
#include "block_dev.h"

namespace nfq {
namespace {

// One wave per 128 values of a line: element e of line r at x[r * rs + e * cs],
// so rows (rs = ld, cs = 1) and columns (rs = 1, cs = ld) are the same kernel.
template <typename T>
__global__ __launch_bounds__(256) void k_block_quantise(const T* __restrict__ x, int64_t R, int64_t L, int64_t rs,
                                                        int64_t cs, uint8_t* __restrict__ codes,
                                                        float* __restrict__ scales) {
    const int lane = threadIdx.x & 63;
    const int64_t kb = blk_count(L), n = R * kb;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 4;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); i < n; i += step) {
        const int64_t r = i / kb, b = i % kb, e = b * kBlk + 2 * lane;
        const float v0 = e < L ? to_f32(x[r * rs + e * cs]) : 0.0f;
        const float v1 = e + 1 < L ? to_f32(x[r * rs + (e + 1) * cs]) : 0.0f;
        const float sc = blk_scale(wave_max(amax_of(amax_of(0.0f, v0), v1)));
        const float inv = 1.0f / sc;
        // Past the line's end the byte is 0 whatever the scale.
        const uint32_t w0 = e < L ? fp8_quant(v0, inv) : 0u, w1 = e + 1 < L ? fp8_quant(v1, inv) : 0u;
        *reinterpret_cast<uint16_t*>(codes + r * kb * kBlk + e) = static_cast<uint16_t>(w0 | w1 << 8);
        if (lane == 0) scales[b * R + r] = sc;
    }
}

// One block of 256 threads per 128 x 128 block of a weight.
template <typename T>
__global__ __launch_bounds__(256) void k_block_quantise_weight(const T* __restrict__ W, int64_t N, int64_t K,
                                                               int64_t ldw, uint8_t* __restrict__ codes,
                                                               float* __restrict__ scales,
                                                               uint8_t* __restrict__ codes_t,
                                                               float* __restrict__ scales_t) {
    __shared__ float part[4];
    const int64_t nb = blk_count(N), kb = blk_count(K);
    const int64_t n0 = blockIdx.x / kb * kBlk, k0 = blockIdx.x % kb * kBlk;
    float amax = 0.0f;
    for (int i = threadIdx.x; i < kBlk * kBlk; i += 256) {
        const int64_t n = n0 + i / kBlk, k = k0 + i % kBlk;
        if (n < N && k < K) amax = amax_of(amax, to_f32(W[n * ldw + k]));
    }
    amax = wave_max(amax);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
    __syncthreads();
    const float sc = blk_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
    const float inv = 1.0f / sc;
    for (int i = threadIdx.x; i < kBlk * kBlk; i += 256) {
        const int64_t n = n0 + i / kBlk, k = k0 + i % kBlk;
        const uint32_t q = n < N && k < K ? fp8_quant(to_f32(W[n * ldw + k]), inv) : 0u;
        if (n < N) codes[n * kb * kBlk + k] = static_cast<uint8_t>(q);
        if (codes_t && k < K) codes_t[k * nb * kBlk + n] = static_cast<uint8_t>(q);
    }
    if (threadIdx.x == 0) {
        scales[(k0 / kBlk) * nb + n0 / kBlk] = sc;
        if (scales_t) scales_t[(n0 / kBlk) * kb + k0 / kBlk] = sc;
    }
}

template <typename T>
void launch_lines(const T* x, int64_t R, int64_t L, int64_t rs, int64_t cs, uint8_t* codes, float* scales,
                  hipStream_t st) {
    hipLaunchKernelGGL((k_block_quantise<T>), dim3(grid_for(R * blk_count(L), 4, 8)), dim3(256), 0, st, x, R, L, rs,
                       cs, codes, scales);
}

int check_matrix(const char* what, const void* x, int dtype, int64_t M, int64_t K, int64_t ldx) {
    if (!dtype_ok(dtype)) return bad_arg(what, "unknown dtype");
    if (M < 0 || K < 0) return bad_arg(what, "bad dims");
    if (ldx < K) return bad_arg(what, "row stride smaller than a row");
    if (M > 0 && K > 0 && !x) return bad_arg(what, "null input");
    return NFLOW_OK;
}

}  // namespace

int block_quantise(const char* what, const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* codes,
                   float* scales, uint8_t* codes_t, float* scales_t, hipStream_t st) {
    auto run = [&](auto* p) {
        if (codes) launch_lines(p, M, K, ldx, int64_t{1}, codes, scales, st);
        if (codes_t) launch_lines(p, K, M, int64_t{1}, ldx, codes_t, scales_t, st);
    };
    if (dtype == NFLOW_DTYPE_BF16) run(static_cast<const bf16*>(x));
    else run(static_cast<const float*>(x));
    return launch_status(what);
}

}  // namespace nfq

using namespace nfq;

extern "C" {

int nflow_fp8_block_quantise(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* codes,
                             float* scales, uint8_t* codes_t, float* scales_t, void* stream) {
    clear_error();
    const char* what = "fp8_block_quantise";
    if (int rc = check_matrix(what, x, dtype, M, K, ldx)) return rc;
    if (M == 0 || K == 0) return NFLOW_OK;
    if (!codes && !codes_t) return bad_arg(what, "no output asked for");
    if (!codes != !scales || !codes_t != !scales_t) return bad_arg(what, "codes and scales come in pairs");
    if (!aligned(codes, 16) || !aligned(codes_t, 16)) return bad_arg(what, "codes must be 16-byte aligned");
    return block_quantise(what, x, dtype, M, K, ldx, codes, scales, codes_t, scales_t, as_stream(stream));
}

int nflow_fp8_block_quantise_weight(const void* W, int dtype, int64_t N, int64_t K, int64_t ldw, uint8_t* codes,
                                    float* scales, uint8_t* codes_t, float* scales_t, void* stream) {
    clear_error();
    const char* what = "fp8_block_quantise_weight";
    if (int rc = check_matrix(what, W, dtype, N, K, ldw)) return rc;
    if (N == 0 || K == 0) return NFLOW_OK;
    if (!codes || !scales) return bad_arg(what, "null codes or scales");
    if (!codes_t != !scales_t) return bad_arg(what, "codes and scales come in pairs");
    if (!aligned(codes, 16) || !aligned(codes_t, 16)) return bad_arg(what, "codes must be 16-byte aligned");
    const int64_t blocks = blk_count(N) * blk_count(K);
    if (blocks > INT32_MAX) return bad_arg(what, "more than 2^31 - 1 blocks");
    const dim3 grid(static_cast<unsigned>(blocks)), block(256);
    if (dtype == NFLOW_DTYPE_BF16)
        hipLaunchKernelGGL((k_block_quantise_weight<bf16>), grid, block, 0, as_stream(stream),
                           static_cast<const bf16*>(W), N, K, ldw, codes, scales, codes_t, scales_t);
    else
        hipLaunchKernelGGL((k_block_quantise_weight<float>), grid, block, 0, as_stream(stream),
                           static_cast<const float*>(W), N, K, ldw, codes, scales, codes_t, scales_t);
    return launch_status(what);
}

}  // extern "C"
