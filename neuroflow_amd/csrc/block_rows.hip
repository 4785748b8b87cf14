// block_rows.hip -- the linear layer of many rows and few K blocks, from values:
// the rows are quantised on their way into the product.
//
// A wave owns 16 rows for all of their columns.  It reads its rows once, the 32
// values of a K block that lane (r, g) = (l % 16, l / 16) multiplies: groups g
// and g + 4 of 16 of row r, so a block's largest magnitude is a lane's own and
// two permlane swaps, and the codes (or their exact bf16 values) stay in the
// operand registers while the weight passes by: K blocks of 128 columns, 16 KB,
// in a ring of three LDS stages that the workgroup's four waves share.  No codes
// of the rows are stored, and the result is the tiled product's bit for bit: the
// same instructions over the same bytes in the same order.
//
// Bound by HBM, x once and y once, and by reading all of x ahead of the first
// store: 32768 x 256 -> 768 fp32 33.0 us, 4.1 TB/s.
#include <algorithm>
#include <cmath>

#include "block_gemm_kernel.h"

namespace nfq {
namespace {

constexpr int kRowsMaxBlocks = 4;

struct RowsTile {
    static constexpr int WAVES = 4, BM = 16 * WAVES, BN = kBlk, NS = 3;
    static constexpr int STAGE = BN * kBlk, NL = STAGE / 1024 / WAVES;      // 1 KB code loads per wave and step
    static constexpr int COLS = 64;                                        // of a strip
    static constexpr int STRIP_ROW = COLS + 4, STRIP = 16 * STRIP_ROW;
    static constexpr int BYTES = NS * STAGE + WAVES * STRIP * 4;
};

template <typename T, int KB>
__global__ __launch_bounds__(64 * RowsTile::WAVES, 2) void k_block_rows(BlockGemmArgs a, const T* __restrict__ x,
                                                                        int64_t ldx, int groups, int per) {
    using R = RowsTile;
    constexpr bool FP8 = std::is_same_v<T, bf16>;
    constexpr int TJ = R::BN / 16, HALF = R::COLS / 16, ROWS = 8 * R::WAVES;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t m0 = static_cast<int64_t>(blockIdx.x % groups) * R::BM + 16 * wid;
    const int tiles = static_cast<int>((a.N + R::BN - 1) / R::BN);          // also the weight's columns of scales
    const int t0 = blockIdx.x / groups * per, t1 = t0 + per < tiles ? t0 + per : tiles;
    constexpr int ld = KB * kBlk;

    // K block b of the weight's tile t into a stage, rows swizzled as the tiled
    // product has them; past the workgroup's last tile the range is empty.
    const uint32_t lds0 = wide_lds_addr(lds);
    const int lrow = 8 * wid + (lane >> 3);
    const int voff = lrow * ld + 16 * ((lane & 7) ^ ((lrow >> 1) & 7));
    auto load = [&](int t, int b, int s) {
#pragma unroll
        for (int c = 0; c < R::NL; ++c) {
            const int64_t row = static_cast<int64_t>(t) * R::BN + ROWS * c;
            wide_dma(wide_desc(a.W + row * ld, t < t1 ? (a.N - row < ROWS ? a.N - row : ROWS) * ld : 0),
                     lds0 + s * R::STAGE + 1024 * (wid + R::WAVES * c), voff, kBlk * b);
        }
    };
    load(t0, 0, 0);
    load(t0 + 1 / KB, 1 % KB, 1);

    // The rows' codes and scales.
    v8i xf[KB];
    float sx[KB];
    const T* row = x + (m0 + r) * ldx;
    const bool on = m0 + r < a.M;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        float v[4][8], amax = 0.0f;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int c = b * kBlk + 16 * g + 64 * (h >> 1) + 8 * (h & 1);
            load8(row + c, on ? a.K - c : 0, v[h]);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = amax_of(amax, v[h][e]);
        sx[b] = blk_scale(cross_rows<MaxOp>(amax));
        const float inv = blk_inverse(sx[b]);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const v2u q = blk_codes8(v[h], inv);
            xf[b][2 * h] = static_cast<int>(q[0]);
            xf[b][2 * h + 1] = static_cast<int>(q[1]);
        }
    }
    Bf16x32 xb[FP8 ? 1 : KB];
    if constexpr (!FP8) {
#pragma unroll
        for (int b = 0; b < KB; ++b) xb[b] = to_bf16(xf[b]);
    }

    const int flo = r * kBlk + 16 * (g ^ ((r >> 1) & 7)), fhi = flo ^ 64;
    float* strip = reinterpret_cast<float*>(lds + R::NS * R::STAGE) + wid * R::STRIP;
    int stage = 0;
    for (int t = t0; t < t1; ++t) {
        v4f acc[2][1][HALF];
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[j / HALF][0][j % HALF] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            // A tile's first block waits for the last tile's stores as well
            // (counting past them instead is no faster).
            if (b == 0) wait_barrier<0>();
            else wait_barrier<R::NL>();
            const int ns = stage >= 1 ? stage - 1 : stage + 2;              // two steps on, of three
            load(t + (b + 2) / KB, (b + 2) % KB, ns);
            const uint8_t* st = lds + stage * R::STAGE;
            stage = stage == R::NS - 1 ? 0 : stage + 1;
            const float s = sx[b] * a.sW[static_cast<int64_t>(b) * tiles + t];
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                const v4i lo = *reinterpret_cast<const v4i*>(st + flo + 16 * kBlk * j);
                const v4i hi = *reinterpret_cast<const v4i*>(st + fhi + 16 * kBlk * j);
                const v8i wf{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                v4f d{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (FP8) {
                    d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf[b], d, 0, 0, 0, 0, 0, 0);
                } else {
                    const Bf16x32 wb = to_bf16(wf);
#pragma unroll
                    for (int q = 0; q < 4; ++q) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb.q[q], xb[b].q[q], d, 0, 0, 0);
                }
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    acc[j / HALF][0][j % HALF][v] = __builtin_fmaf(d[v], s, acc[j / HALF][0][j % HALF][v]);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            store_tiles<T, R, true>(acc[h], strip, static_cast<T*>(a.C), a.M, a.N, a.ldc, a.bias, a.act, m0,
                                    static_cast<int64_t>(t) * R::BN + R::COLS * h);
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");   // the empty loads past the last tile
}

// How the columns are dealt out: `per` tiles a workgroup, `n` workgroups on the
// fullest CU, and the share of the n * per tile slots of all CUs that have work.
// More shares of the columns fill and balance the CUs, and each quantises its
// rows again, about one and a half tiles' time; n workgroups of a CU take 0.8 n
// times as long as one.
struct RowsCut {
    int per, n;
    double filled;
};
RowsCut rows_cut(int64_t M, int64_t N) {
    const int64_t groups = (M + RowsTile::BM - 1) / RowsTile::BM, tiles = blk_count(N), cus = num_cus();
    RowsCut best{};
    double least = HUGE_VAL;
    // From a workgroup for every CU (fewer shares than that are no faster) to a tile each.
    const int64_t shares = std::max<int64_t>(1, cus / groups);
    for (int64_t per = (tiles + shares - 1) / shares; per > 0; --per) {
        const int64_t n = (groups * ((tiles + per - 1) / per) + cus - 1) / cus;
        const double t = (static_cast<double>(per) + 1.5) * std::max(1.0, 0.8 * static_cast<double>(n));
        if (t < least) {
            least = t;
            best = RowsCut{static_cast<int>(per), static_cast<int>(n),
                           static_cast<double>(groups * tiles) / static_cast<double>(cus * n * per)};
        }
    }
    return best;
}

unsigned rows_grid(int64_t M, int64_t N, int per) {
    return static_cast<unsigned>((M + RowsTile::BM - 1) / RowsTile::BM * ((blk_count(N) + per - 1) / per));
}

template <typename T, int KB>
void launch_rows(const BlockGemmArgs& a, const void* x, int64_t ldx, hipStream_t st) {
    static const hipError_t once = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_block_rows<T, KB>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, RowsTile::BYTES);
    (void)once;
    const int groups = static_cast<int>((a.M + RowsTile::BM - 1) / RowsTile::BM);
    const int per = rows_cut(a.M, a.N).per;
    hipLaunchKernelGGL((k_block_rows<T, KB>), dim3(rows_grid(a.M, a.N, per)), dim3(64 * RowsTile::WAVES), RowsTile::BYTES,
                       st, a, static_cast<const T*>(x), ldx, groups, per);
}

template <typename T>
void launch_rows_kb(const BlockGemmArgs& a, const void* x, int64_t ldx, hipStream_t st) {
    switch (blk_count(a.K)) {
    case 1: return launch_rows<T, 1>(a, x, ldx, st);
    case 2: return launch_rows<T, 2>(a, x, ldx, st);
    case 3: return launch_rows<T, 3>(a, x, ldx, st);
    default: return launch_rows<T, 4>(a, x, ldx, st);
    }
}

}  // namespace

// Where this is the faster of the two.  Of 600 sizes (17 to 32768 rows, 64 to 4096
// columns, K of 100 to 512) it holds at 301, which take 0.77 of the time of the
// quantise and the product (geometric mean; 0.52 to 1.035).  At 17 to 2000 rows of
// 2048 to 200000 columns, in replayed graphs, where a launch costs least, it takes
// 0.67 to 1.08 of it (fp32 results of two K blocks are the ones over 1: 96 x 256 ->
// 32768 11.6 / 10.8, 100 x 256 -> 256 7.7 / 7.2).  Here / there in us, call by call:
// fp32 100 x 256 -> 256 7.4 / 8.7, 32768 x 128 -> 768 24.6 / 30.3, 32768 x 256 ->
// 768 32.1 / 34.7; bf16 4096 x 256 -> 768 8.6 / 10.7, 32768 x 256 -> 256 10.4 / 18.7.
// - A wave converts or reads the whole weight for 16 rows, which the tiled
//   product does for 64: past two K blocks, and past a width, that costs more
//   than the rows' codes save, for fp32 results (whose codes are converted)
//   sooner (fp32 16384 x 128 -> 2048 42 / 35).
// - A large result has to leave in whole 128-byte lines (bf16 20000 x 256 -> 1000
//   41 / 31), from CUs with equal work (313 groups of rows, bf16 20000 x 512 ->
//   768 35 / 28); in a small one the launch saved is more than either.
// - Past 32768 columns a second group of rows makes a CU pass three tiles and more
//   of the weight one after the other (65 x 256 -> 64000 bf16 15.6 / 11.6, fp32
//   18.8 / 13.3); one group does not (17 x 128 -> 200000 bf16 15.7 / 21.9).
// - Up to 64 rows the product of the codes is the few-row kernel, which sums
//   several K blocks in another order; elsewhere both give the same bits.
bool many_rows_values(int64_t M, int64_t N, int64_t K, int dtype) {
    const int64_t kb = blk_count(K);
    if (kb == 0 || kb > kRowsMaxBlocks || M <= (kb == 1 ? 16 : 64)) return false;
    const bool bf = dtype == NFLOW_DTYPE_BF16, small = M * N <= (1 << 22);
    if (M > 64 && N > 32768) return false;
    if (kb > 2 && (bf ? M < 2048 || N > 1024 : M < 8192 || N > 256)) return false;
    if (small || N <= 256) return true;
    if (N > (bf ? 2048 : 1024) || N * (bf ? 2 : 4) % 128 != 0) return false;
    const RowsCut c = rows_cut(M, N);
    return c.n == 1 || c.filled >= 0.9;
}

unsigned block_rows_grid(int64_t M, int64_t N) { return rows_grid(M, N, rows_cut(M, N).per); }

void launch_block_rows(const BlockGemmArgs& a, const void* x, int64_t ldx, hipStream_t st) {
    if (a.out == NFLOW_DTYPE_BF16) launch_rows_kb<bf16>(a, x, ldx, st);
    else launch_rows_kb<float>(a, x, ldx, st);
}

}  // namespace nfq
