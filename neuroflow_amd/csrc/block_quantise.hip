// block_quantise.hip -- activations and weights to 128-block FP8
// (include/nflow_block.h).
#include <type_traits>

#include "block_gemm.h"

namespace nfq {
namespace {

// ---- rows ------------------------------------------------------------------
// 16 lanes take a block of 128 values, 8 adjacent ones a lane: the largest
// magnitude is a DPP reduction within the 16, the codes are 8 bytes a lane.
// Sixteen neighbouring groups take the same blocks of neighbouring rows, so a
// workgroup's scales (rows of the (blocks, M) array) leave as runs.  HBM
// bound: each group has kRun blocks of its row in flight.  16384 x 4096 bf16:
// 45.5 us, 4.5 TB/s.
constexpr int kRun = 4;

template <typename T>
__global__ __launch_bounds__(256) void k_quantise_rows_blk(const T* __restrict__ x, int64_t M, int64_t K, int64_t ldx,
                                                           uint8_t* __restrict__ codes, float* __restrict__ scales) {
    const int cl = threadIdx.x & 15;
    const int64_t kb = blk_count(K), runs = (kb + kRun - 1) / kRun, n = M * runs;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
    if (i >= n) return;
    const int64_t b0 = i / M * kRun, m = i % M;
    const T* row = x + m * ldx;
    float v[kRun][8];
#pragma unroll
    for (int u = 0; u < kRun; ++u) {
        const int64_t c = (b0 + u) * kBlk + 8 * cl;
        load8(row + c, K - c, v[u]);
    }
    float amax[kRun], inv[kRun], sc;
#pragma unroll
    for (int u = 0; u < kRun; ++u) {
        amax[u] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax[u] = amax_of(amax[u], v[u][e]);
        amax[u] = max16(amax[u]);
    }
    blk_scales<kRun>(amax, sc, inv);
    if (cl < kRun && b0 + cl < kb) scales[(b0 + cl) * M + m] = sc;
#pragma unroll
    for (int u = 0; u < kRun; ++u) {
        const int64_t b = b0 + u;
        if (b >= kb) break;
        *reinterpret_cast<v2u*>(codes + m * kb * kBlk + b * kBlk + 8 * cl) =
            blk_codes8(v[u], inv[u]);
    }
}

// ---- both axes, and weights ----------------------------------------------------
// A workgroup takes 128 x 128 values, one read: 16 lanes cover a row, and
// thread (rg, cl) holds the 8 x 8 values of rows 8 rg .. and columns 8 cl ...
// Row maxima are a DPP reduction, column maxima a shuffle over the wave's four
// row groups and LDS over the four waves.  The column codes are 8 bytes of a
// column per thread and column; they cross to rows of the transposed array in
// LDS (8-byte slot s of line c at s ^ (c / 8), which spreads the 16 lanes of
// a write over the banks) and leave as whole 128-byte lines.  HBM bound, with the
// VALU half busy (17.6 instructions a value): 16384 x 4096 bf16 57.5 us, 4.7 TB/s.
struct TileOut {
    uint8_t* codes;       // along rows, or null
    float* scales;
    uint8_t* codes_t;     // along columns, or null
    float* scales_t;
    float* col_sums;      // (row tiles, K) sums of 128 rows, or null
};

template <typename T, bool WEIGHT>
__global__ __launch_bounds__(256) void k_quantise_tile(const T* __restrict__ x, int64_t M, int64_t K, int64_t ldx,
                                                       TileOut o) {
    __shared__ __attribute__((aligned(16))) uint8_t lt[kBlk * kBlk];
    __shared__ __attribute__((aligned(16))) float cmax[4][kBlk];
    __shared__ __attribute__((aligned(16))) float csum[4][kBlk];
    __shared__ __attribute__((aligned(16))) float colinv[kBlk];
    const int tid = threadIdx.x, cl = tid & 15, rg = tid >> 4, wave = tid >> 6, lane = tid & 63;
    const int64_t kb = blk_count(K), mb = blk_count(M);
    const int64_t tm = blockIdx.x / kb, tk = blockIdx.x % kb;
    const int64_t m0 = tm * kBlk + 8 * rg, c0 = tk * kBlk + 8 * cl;
    Raw8<T> v[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) v[p].load(x + (m0 + p) * ldx + c0, m0 + p < M ? K - c0 : 0);
    // bf16 values stay packed, two to a register, and are converted at each of
    // their uses: held as floats they would take 64 registers, and six
    // workgroups a CU would be four (16384 x 4096: 60.1 against 63.8 us then).
    auto keep = [&] {
#pragma unroll
        for (int p = 0; p < 8; ++p) asm volatile("" : "+v"(v[p].q));
    };

    float ca[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        ca[e] = 0.0f;
#pragma unroll
        for (int p = 0; p < 8; ++p) ca[e] = amax_of(ca[e], v[p][e]);
        ca[e] = fmaxf(ca[e], __shfl_xor(ca[e], 16));
        ca[e] = fmaxf(ca[e], __shfl_xor(ca[e], 32));
    }
    if (lane < 16) {
        *reinterpret_cast<v4f*>(&cmax[wave][8 * cl]) = v4f{ca[0], ca[1], ca[2], ca[3]};
        *reinterpret_cast<v4f*>(&cmax[wave][8 * cl + 4]) = v4f{ca[4], ca[5], ca[6], ca[7]};
    }
    if (!WEIGHT && o.col_sums) {
        float cs[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            cs[e] = 0.0f;
#pragma unroll
            for (int p = 0; p < 8; ++p) cs[e] += v[p][e];
            cs[e] += __shfl_xor(cs[e], 16);
            cs[e] += __shfl_xor(cs[e], 32);
        }
        if (lane < 16) {
            *reinterpret_cast<v4f*>(&csum[wave][8 * cl]) = v4f{cs[0], cs[1], cs[2], cs[3]};
            *reinterpret_cast<v4f*>(&csum[wave][8 * cl + 4]) = v4f{cs[4], cs[5], cs[6], cs[7]};
        }
    }
    __syncthreads();
    float cinv[8];
    if constexpr (WEIGHT) {
        float w = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) w = fmaxf(w, cmax[q >> 1][64 * (q & 1) + lane]);
        const float sblk = blk_scale(wave_max(w)), inv = blk_inverse(sblk);
#pragma unroll
        for (int e = 0; e < 8; ++e) cinv[e] = inv;
        if (tid == 0) {
            o.scales[tk * mb + tm] = sblk;
            if (o.scales_t) o.scales_t[tm * kb + tk] = sblk;
        }
    } else {
        // A thread per column divides; all read the inverses past the rows' part.
        if (tid < kBlk) {
            const float m4 = fmaxf(fmaxf(cmax[0][tid], cmax[1][tid]), fmaxf(cmax[2][tid], cmax[3][tid]));
            const float sc = blk_scale(m4);
            if (o.codes_t) {
                colinv[tid] = blk_inverse(sc);
                if (tk * kBlk + tid < K) o.scales_t[tm * K + tk * kBlk + tid] = sc;
            }
            if (o.col_sums && tk * kBlk + tid < K)
                o.col_sums[tm * K + tk * kBlk + tid] = (csum[0][tid] + csum[1][tid]) + (csum[2][tid] + csum[3][tid]);
        }
    }

    keep();
    if (o.codes) {
        float rinv[8];
        if constexpr (WEIGHT) {
#pragma unroll
            for (int p = 0; p < 8; ++p) rinv[p] = cinv[0];
        } else {
            float ra[8], sc;
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                ra[p] = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ra[p] = amax_of(ra[p], v[p][e]);
                ra[p] = max16(ra[p]);
            }
            keep();
            blk_scales<8>(ra, sc, rinv);
            if (cl < 8 && m0 + cl < M) o.scales[tk * M + m0 + cl] = sc;
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            float r[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) r[e] = v[p][e];
            const v2u q8 = blk_codes8(r, rinv[p]);
            if (m0 + p < M) *reinterpret_cast<v2u*>(o.codes + (m0 + p) * kb * kBlk + c0) = q8;
        }
    }
    keep();
    if (!WEIGHT && o.codes_t) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) cinv[e] = colinv[8 * cl + e];
    }
    if (o.codes_t) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float r[8];
#pragma unroll
            for (int p = 0; p < 8; ++p) r[p] = v[p][e];
            *reinterpret_cast<v2u*>(lt + (8 * cl + e) * kBlk + 8 * (rg ^ cl)) = blk_codes8(r, cinv[e]);
        }
        __syncthreads();
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int c = 32 * it + (tid >> 3), s = 2 * (tid & 7), x = c >> 3;
            const v2u lo = *reinterpret_cast<const v2u*>(lt + c * kBlk + 8 * (s ^ x));
            const v2u hi = *reinterpret_cast<const v2u*>(lt + c * kBlk + 8 * ((s + 1) ^ x));
            if (tk * kBlk + c < K)
                *reinterpret_cast<v4u*>(o.codes_t + (tk * kBlk + c) * mb * kBlk + tm * kBlk + 8 * s) =
                    v4u{lo[0], lo[1], hi[0], hi[1]};
        }
    }
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
                   float* scales, uint8_t* codes_t, float* scales_t, float* col_sums, hipStream_t st) {
    const int64_t kb = blk_count(K);
    const bool tile = codes_t || col_sums;
    const int64_t blocks = tile ? blk_count(M) * kb : (M * ((kb + kRun - 1) / kRun) + 15) / 16;
    if (blocks > INT32_MAX) return bad_arg(what, "more than 2^31 - 1 blocks");
    const dim3 grid(static_cast<unsigned>(blocks)), block(256);
    auto run = [&](auto* p) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
        if (tile)
            hipLaunchKernelGGL((k_quantise_tile<T, false>), grid, block, 0, st, p, M, K, ldx,
                               TileOut{codes, scales, codes_t, scales_t, col_sums});
        else
            hipLaunchKernelGGL((k_quantise_rows_blk<T>), grid, block, 0, st, p, M, K, ldx, codes, scales);
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
    return block_quantise(what, x, dtype, M, K, ldx, codes, scales, codes_t, scales_t, nullptr, as_stream(stream));
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
    const TileOut o{codes, scales, codes_t, scales_t, nullptr};
    if (dtype == NFLOW_DTYPE_BF16)
        hipLaunchKernelGGL((k_quantise_tile<bf16, true>), grid, block, 0, as_stream(stream),
                           static_cast<const bf16*>(W), N, K, ldw, o);
    else
        hipLaunchKernelGGL((k_quantise_tile<float, true>), grid, block, 0, as_stream(stream),
                           static_cast<const float*>(W), N, K, ldw, o);
    return launch_status(what);
}

}  // extern "C"
