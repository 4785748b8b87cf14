// block_dev.h -- device and host helpers shared by the layer norm, the
// 128-block quantise and the block-FP8 product (include/nflow_block.h).
#pragma once

#include <cmath>
#include <string>

#include "common.h"
#include "launch.h"
#include "nflow_block.h"
#include "status.h"

namespace nfq {

constexpr int kBlk = 128;   // values per scale

__host__ __device__ constexpr int64_t blk_count(int64_t n) { return (n + kBlk - 1) / kBlk; }

// ---- element types ----------------------------------------------------------

typedef __bf16 bf16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return static_cast<T>(v); }   // bf16: nearest, ties to even

// ---- 128-block scale ----------------------------------------------------------

// Below this a block's codes would need a subnormal scale, whose inverse
// overflows: such a block is all zero codes under scale 1.
constexpr float kBlkTiny = 448.0f * 0x1p-126f;

__device__ __forceinline__ float blk_scale(float amax) { return amax < kBlkTiny ? 1.0f : amax / 448.0f; }

// max that ignores a NaN in v (amax itself is never one).
__device__ __forceinline__ float amax_of(float amax, float v) { return fmaxf(amax, fabsf(v)); }

// ---- reductions over a wave -------------------------------------------------------

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

// ---- checks of the entry points ----------------------------------------------------

inline bool dtype_ok(int dtype) { return dtype == NFLOW_DTYPE_F32 || dtype == NFLOW_DTYPE_BF16; }
inline size_t dtype_size(int dtype) { return dtype == NFLOW_DTYPE_BF16 ? 2 : 4; }

inline int bad_arg(const char* what, const char* why) {
    return set_error(NFLOW_INVALID_ARG, std::string(what) + ": " + why);
}

inline int launch_status(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(NFLOW_INTERNAL, std::string(what) + ": " + hipGetErrorString(e));
    return NFLOW_OK;
}

// The workspace an entry point was given against the bytes it needs.
inline int check_workspace(const char* what, const void* ws, size_t have, size_t need) {
    if (need == 0) return NFLOW_OK;
    if (!ws || have < need) return bad_arg(what, "workspace missing or smaller than its _workspace function says");
    if (!aligned(ws, 16)) return bad_arg(what, "workspace must be 16-byte aligned");
    return NFLOW_OK;
}

inline size_t round16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

}  // namespace nfq
