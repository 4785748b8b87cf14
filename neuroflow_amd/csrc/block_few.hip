// block_few.hip -- the block-FP8 product for few rows: one new token, or a
// small batch of them, against a weight that is read once.
//
// A workgroup owns 16 CT columns and all the rows; its waves deal the K blocks
// out among them (wave w takes blocks w, w + W, ...), so that the workgroup has
// its whole share of the weight in flight at once, straight from HBM to the
// MFMA operand registers: nothing is shared between waves, and a byte of the
// weight is used by one of them.  Each wave keeps fp32 sums of its blocks, and
// the workgroup joins them in LDS in the waves' order.  Bound by reading the
// weight: N K bytes, plus the launch and one load's latency (1 row, 4096 x 4096
// bf16: 5.7 us).
//
// Rows come as codes, or as values, which every workgroup then quantises by
// itself into LDS while its first weight loads are in flight: 16 lanes a block
// of 128 values, as in block_quantise.hip. That spares a launch and repeats the
// quantise in each workgroup, so it is for few values (few_values).
#include "block_gemm_kernel.h"

namespace nfq {
namespace {

// X: uint8_t (codes and scales), float or bf16 (values, quantised here).
template <typename TO, typename X, bool BLOCKS, int RT, int CT, int W>
__global__ __launch_bounds__(64 * W) void k_block_few(BlockGemmArgs a, const X* __restrict__ x, int64_t ldx) {
    constexpr bool FP8 = std::is_same_v<TO, bf16>;
    constexpr bool CODES = std::is_same_v<X, uint8_t>;
    __shared__ __attribute__((aligned(16))) v4f red[W > 1 ? W : 1][RT * CT][64];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16 * CT;
    const int kb = static_cast<int>(blk_count(a.K));
    const int64_t ld = static_cast<int64_t>(kb) * kBlk, nb = blk_count(a.N);

    v4f acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    // Rows past the last (of W or of x) read row 0: their products are never stored.
    const uint8_t* wrow[CT];
#pragma unroll
    for (int j = 0; j < CT; ++j) {
        const int64_t n = n0 + 16 * j + r;
        wrow[j] = a.W + (n < a.N ? n : 0) * ld + 16 * g;
    }
    auto load_codes = [&](const uint8_t* p) {
        const v4i lo = *reinterpret_cast<const v4i*>(p);
        const v4i hi = *reinterpret_cast<const v4i*>(p + 64);
        return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };

    v8i wn[2][CT];
    auto fetch_w = [&](int k, v8i (&w)[CT]) {
        const int64_t at = static_cast<int64_t>(k < kb ? k : 0) * kBlk;      // past the last: any, never used
#pragma unroll
        for (int j = 0; j < CT; ++j) w[j] = load_codes(wrow[j] + at);
    };
    if (kb > 0) {
        fetch_w(wid, wn[0]);
        fetch_w(wid + W, wn[1]);
    }
    // Values to codes and scales in LDS, rows of ldx_lds bytes (16 more than the
    // codes, against bank conflicts between rows).
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int ldl = static_cast<int>(ld) + 16;
    float* lds_scale = reinterpret_cast<float*>(lds + (CODES ? 0 : a.M * ldl));
    if constexpr (!CODES) {
        const int items = static_cast<int>(a.M) * kb, cl = threadIdx.x & 15;
        for (int i = threadIdx.x >> 4; i < items; i += 4 * W) {
            const int m = i / kb, b = i - m * kb, c = b * kBlk + 8 * cl;
            float v[8], amax = 0.0f;
            load8(x + m * ldx + c, a.K - c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = amax_of(amax, v[e]);
            const float sc = blk_scale(max16(amax));
            *reinterpret_cast<v2u*>(lds + m * ldl + c) = blk_codes8(v, blk_inverse(sc));
            if (cl == 0) lds_scale[i] = sc;
        }
        __syncthreads();
    }
    auto step = [&](int k, const v8i (&wf)[CT]) {
        v4f sw[CT];
#pragma unroll
        for (int j = 0; j < CT; ++j) {
            const int64_t n = n0 + 16 * j + 4 * g;
            if constexpr (BLOCKS) {
                const float s = a.sW[k * nb + (n0 + 16 * j < a.N ? (n0 + 16 * j) / kBlk : 0)];
                sw[j] = v4f{s, s, s, s};
            } else {
#pragma unroll
                for (int v = 0; v < 4; ++v) sw[j][v] = n + v < a.N ? a.sW[k * a.N + n + v] : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int64_t m = 16 * i + r, mm = m < a.M ? m : 0;
            v8i xf;
            float sa;
            if constexpr (CODES) {
                xf = load_codes(x + mm * ld + static_cast<int64_t>(k) * kBlk + 16 * g);
                sa = a.sA[k * a.M + mm];
            } else {
                xf = load_codes(lds + mm * ldl + k * kBlk + 16 * g);
                sa = lds_scale[mm * kb + k];
            }
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                v4f d{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (FP8) {
                    d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], xf, d, 0, 0, 0, 0, 0, 0);
                } else {
                    const Bf16x32 wb = to_bf16(wf[j]), xb = to_bf16(xf);
#pragma unroll
                    for (int q = 0; q < 4; ++q) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb.q[q], xb.q[q], d, 0, 0, 0);
                }
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    acc[i][j][v] = __builtin_fmaf(BLOCKS ? d[v] : d[v] * sw[j][v], BLOCKS ? sa * sw[j][v] : sa, acc[i][j][v]);
            }
        }
    };
    // Blocks in pairs, each pair's codes asked for two of the wave's turns ahead.
    for (int k = wid; k < kb; k += 2 * W) {
        step(k, wn[0]);
        fetch_w(k + 2 * W, wn[0]);
        if (k + W < kb) {
            step(k + W, wn[1]);
            fetch_w(k + 3 * W, wn[1]);
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) red[wid][i * CT + j][lane] = acc[i][j];
    __syncthreads();
    const bool vec = a.ldc % 4 == 0 && (reinterpret_cast<uintptr_t>(a.C) & (4 * sizeof(TO) - 1)) == 0;
    for (int t = wid; t < RT * CT; t += W) {
        v4f z = red[0][t][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) z += red[w][t][lane];
        store4<TO>(a, 16 * (t / CT) + r, n0 + 16 * (t % CT) + 4 * g, z, vec);
    }
}

// LDS of the quantised rows.
size_t few_lds(int64_t M, int64_t K) {
    return static_cast<size_t>(M * (blk_count(K) * kBlk + 16) + 4 * M * blk_count(K));
}

template <typename TO, typename X, bool BLOCKS, int RT, int CT, int W>
void launch_w(const BlockGemmArgs& a, const X* x, int64_t ldx, hipStream_t st) {
    const unsigned grid = static_cast<unsigned>((a.N + 16 * CT - 1) / (16 * CT));
    const size_t lds = std::is_same_v<X, uint8_t> ? 0 : few_lds(a.M, a.K);
    hipLaunchKernelGGL((k_block_few<TO, X, BLOCKS, RT, CT, W>), dim3(grid), dim3(64 * W), lds, st, a, x, ldx);
}

// Waves per workgroup: 16 while that is at most 16 waves a CU, fewer for wide
// N, where there are workgroups enough, or where K has fewer blocks.
template <typename TO, typename X, bool BLOCKS, int RT, int CT>
void launch_few(const BlockGemmArgs& a, const X* x, int64_t ldx, hipStream_t st) {
    const int64_t groups = (a.N + 16 * CT - 1) / (16 * CT), kb = blk_count(a.K);
    const int64_t want = std::min<int64_t>(kb, 16 * num_cus() / std::max<int64_t>(groups, 1));
    if (want > 8) launch_w<TO, X, BLOCKS, RT, CT, 16>(a, x, ldx, st);
    else if (want > 4) launch_w<TO, X, BLOCKS, RT, CT, 8>(a, x, ldx, st);
    else launch_w<TO, X, BLOCKS, RT, CT, 4>(a, x, ldx, st);
}

template <typename TO, bool BLOCKS>
void launch_codes(const BlockGemmArgs& a, hipStream_t st) {
    if (a.M <= 16) launch_few<TO, uint8_t, BLOCKS, 1, 1>(a, a.A, 0, st);
    else if (a.M <= 32) launch_few<TO, uint8_t, BLOCKS, 2, 1>(a, a.A, 0, st);
    else launch_few<TO, uint8_t, BLOCKS, 4, 1>(a, a.A, 0, st);
}

}  // namespace

void launch_block_few(const BlockGemmArgs& a, hipStream_t st) {
    if (a.out == NFLOW_DTYPE_BF16) {
        if (a.w_blocks) launch_codes<bf16, true>(a, st);
        else launch_codes<bf16, false>(a, st);
    } else {
        if (a.w_blocks) launch_codes<float, true>(a, st);
        else launch_codes<float, false>(a, st);
    }
}

// Up to 32768 values a workgroup quantises them faster than a launch of its own
// would (us, in the kernel / two launches: 4096 x 4096 1 row 7.5 / 12, 8 rows 9.8
// / 12, 16 rows 12.7 / 12.9; 8192 x 8192 1 row 16.3 / 20.7, 4 rows 21.2 / 20.9).
bool few_values(int64_t M, int64_t K) { return M <= 16 && M * blk_count(K) * kBlk <= 32768; }

void launch_block_few_values(const BlockGemmArgs& a, const void* x, int64_t ldx, hipStream_t st) {
    if (a.out == NFLOW_DTYPE_BF16) launch_few<bf16, bf16, true, 1, 1>(a, static_cast<const bf16*>(x), ldx, st);
    else launch_few<float, float, true, 1, 1>(a, static_cast<const float*>(x), ldx, st);
}

}  // namespace nfq
