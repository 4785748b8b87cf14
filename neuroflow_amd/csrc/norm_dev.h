// norm_dev.h -- what the layer norm and the RMS norm share: a row's sums, its
// 1 / sqrt, and how many workgroups run at once.
#pragma once

#include "block_dev.h"

namespace nfq {

constexpr int kNormThreads = 256;

// Widest row the register kernels hold (1024 threads, 16 values each).
constexpr int64_t kNormRegMax = 16384;

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

// 1 / sqrt(v), correctly rounded but for a hundredth of an ulp: the hardware's
// estimate r (an ulp) and a Newton step from its remainder 1 - v r r, taken
// exactly (v r as a rounded product and what that leaves; without the latter the
// result is up to 1.9 ulp off, with a square root and a division 1.5).  The
// division at the ends of the range, where the estimate or the step would leave it.
__device__ __forceinline__ float norm_rstd(float v) {
    const float r = __builtin_amdgcn_rsqf(v);
    const float p = v * r, left = __builtin_fmaf(v, r, -p);
    const float e = __builtin_fmaf(-left, r, __builtin_fmaf(-p, r, 1.0f));
    const float s = __builtin_fmaf(0.5f * r, e, r);
    return v > 0x1p-100f && v < 0x1p100f ? s : 1.0f / sqrtf(v);
}

// L = 16 (four rows a wave), 64, or a whole workgroup of 256 or 1024.
template <int L>
constexpr int row_threads() { return L <= 64 ? 256 : L; }

// Sum over the L threads of a row; part: two sets of a value per wave, used in turn.
template <int L>
__device__ __forceinline__ float row_sum(float v, float (*part)[L <= 64 ? 1 : L / 64], int set) {
    if constexpr (L <= 64) {
        return lanes_reduce<L, SumOp>(v);
    } else {
        v = wave_sum(v);
        if ((threadIdx.x & 63) == 0) part[set][threadIdx.x >> 6] = v;
        __syncthreads();
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < L / 64; ++w) s += part[set][w];
        return s;
    }
}

// The sum of n values, n a power of two, by halves: as many additions as in a
// row, and the mean's error is that of log2 D of them (7.6e-8 of it at 256
// columns where sixteen in a row gave 9.7e-8).
template <int n>
__device__ __forceinline__ float pair_sum(const float* v) {
    if constexpr (n == 1) return v[0];
    else return pair_sum<n / 2>(v) + pair_sum<n / 2>(v + n / 2);
}

// Eight values of a parameter from column c on; `none` where there is no parameter.
__device__ __forceinline__ void load_param(const float* p, int c, int D, float none, float (&v)[8]) {
    if (p) {
        load8(p + c, D - c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = none;
    }
}

inline unsigned row_grid(int64_t M) { return static_cast<unsigned>(std::min<int64_t>(M, 8 * num_cus())); }

// Workgroups of `threads` that run at once, from the kernel's registers and LDS.
template <typename Kernel>
inline int64_t resident(Kernel k, int threads) {
    int n = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, threads, 0) != hipSuccess || n < 1) n = 1;
    return static_cast<int64_t>(n) * num_cus();
}

inline constexpr const char* kOverlap = "the result overlaps an input, and not row for row";

}  // namespace nfq
