// block_gemm_kernel.h -- the tiled product of 128-block FP8 codes on the
// matrix cores.
//
//   C[m][n] = act(sum_b sA[b][m] sW[b][n] (sum over block b of a[m][k] w[n][k]) + bias[n])
//
// A scale covers 128 values of k, and one step of the K loop is such a block:
// 128 bytes of every row of the tile, which is also one
// v_mfma_f32_16x16x128_f8f6f4 (or four v_mfma_f32_16x16x32_bf16) deep.  The
// instruction starts from zero, and its sum joins the fp32 accumulators by one
// FMA per output with sA * sW: 4 VALU instructions (16 cycles) beside 32
// cycles of matrix core, so they fit under it.
//
// bf16 outputs take the FP8 instruction.  It drops low bits of the products
// it sums: measured against the exact sum on normal and uniform codes, 1.3e-5
// and 6e-6 of the result in the 2-norm, at worst 2^-12.6 of the block's sum
// of magnitudes over all finite codes, whatever K; a bf16 result keeps 2^-9.
// fp32 outputs take the bf16 instruction on the codes' values, which are exact
// in bf16 (1e-8 to 1e-7 of the result), at half the rate.
//
// The weight is the A operand, so a lane holds four adjacent columns of one
// row: lane (r, g) = (l % 16, l / 16) of tile (i, j) has row 16 i + r and
// columns 16 j + 4 g .. + 3, and its row scale is one register per i.  Both
// operands take the bytes of 16-byte groups g and g + 4 of the row for lane
// group g: the same k on both sides, in an order of its own.
#pragma once

#include <type_traits>

#include "block_gemm.h"
#include "gemm_kernel.h"
#include "wide_kernel.h"

namespace nfq {

typedef int v8i __attribute__((ext_vector_type(8)));

// 4 bytes per lane from the buffer at voff + soff into LDS at lds + 4 lane.
__device__ __forceinline__ void dma_dword(v4u desc, uint32_t lds, int voff, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(voff), "s"(desc), "s"(soff)
                 : "memory", "m0");
}

// All but the last N vector memory operations and every LDS read of this
// wave are done, and every wave of the block has got here.
template <int N>
__device__ __forceinline__ void wait_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

template <int WM_, int WN_, int TI_, int TJ_, int NS_>
struct BlockTile {
    static constexpr int WM = WM_, WN = WN_, TI = TI_, TJ = TJ_, NS = NS_;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int BM = 16 * TI * WM, BN = 16 * TJ * WN;
    static constexpr int CODES = (BM + BN) * kBlk;                 // bytes of a stage's codes
    static constexpr int STAGE = CODES + 256 * WAVES;              // and of its scales, 64 a wave
    static constexpr int NL = (BM + BN) / 8 / WAVES;               // 1 KB code loads per wave and step
    static constexpr int LOADS = NL + 1;                           // and one 64-scale load
    static_assert((BM + BN) / 8 % WAVES == 0, "code loads spread evenly");
    static_assert((BM + BN) / 64 <= WAVES && BM % 64 == 0 && BN % 64 == 0, "one scale load per wave covers the tile");
    static_assert(kBlk % (16 * TJ) == 0, "a wave's columns lie in one 128-block");
    static_assert((NS - 1) * LOADS < 64, "vmcnt field");
};

// Where block `bid` of the grid works: blocks go round-robin to the XCDs, and
// each XCD takes a contiguous run of tiles, in groups of `gm` tile rows walked
// column by column, so the tiles an XCD's CUs hold at once form a patch that
// shares its rows and columns behind one L2.
struct TilePos {
    int64_t tm;
    int64_t tn;
};
__device__ __forceinline__ TilePos tile_pos(int64_t t, int64_t tiles_m, int64_t tiles_n, int gm) {
    const int64_t per = gm * tiles_n, grp = t / per, in = t - grp * per;
    const int64_t rows = tiles_m - grp * gm < gm ? tiles_m - grp * gm : gm;
    return TilePos{grp * gm + in % rows, in / rows};
}

// Four outputs of a row from column n on: bias, activation, one rounding.
template <typename TO>
__device__ __forceinline__ void store4(const BlockGemmArgs& a, int64_t m, int64_t n, v4f z, bool vec) {
    if (m >= a.M || n >= a.N) return;
    TO* c = static_cast<TO*>(a.C) + m * a.ldc + n;
    float y[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const float b = a.bias && n + v < a.N ? a.bias[n + v] : 0.0f;
        y[v] = activate_rt(z[v] + b, a.act);
    }
    if (vec && n + 3 < a.N) {
        typedef TO v4t __attribute__((ext_vector_type(4)));
        *reinterpret_cast<v4t*>(c) = v4t{from_f32<TO>(y[0]), from_f32<TO>(y[1]), from_f32<TO>(y[2]), from_f32<TO>(y[3])};
        return;
    }
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (n + v < a.N) c[v] = from_f32<TO>(y[v]);
}

// 32 codes per lane as the bf16 operands of four 16x16x32 products.
struct Bf16x32 {
    v8bf q[4];
};
__device__ __forceinline__ Bf16x32 to_bf16(v8i c) {
    Bf16x32 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.q[i] = fp8x8_to_bf16(c[2 * i], c[2 * i + 1]);
    return o;
}

// TO: type of C, and with it the instruction.  BLOCKS: a weight's scales (one
// per 128 x 128), else one per row of W.  With splits > 1 the K blocks are
// dealt out in runs of `per`, and split s writes its fp32 sums, unscaled by
// anything further, to part[s] (M, N).
template <typename TO, bool BLOCKS, typename T>
__global__ __launch_bounds__(T::THREADS, 2) void k_block_gemm(BlockGemmArgs a, int64_t tiles_m, int64_t tiles_n,
                                                              int splits, int per, float* part) {
    constexpr bool FP8 = std::is_same_v<TO, bf16>;
    constexpr int TI = T::TI, TJ = T::TJ, BM = T::BM, BN = T::BN, LEAD = T::NS - 1;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wid / T::WN, wn = wid % T::WN;
    const int r = lane & 15, g = lane >> 4;
    const int64_t t = gemm_tile_of_block(blockIdx.x, gridDim.x, 8);
    const int split = splits > 1 ? static_cast<int>(t % splits) : 0;
    const TilePos pos = tile_pos(splits > 1 ? t / splits : t, tiles_m, tiles_n, 4);
    const int64_t m0 = pos.tm * BM, n0 = pos.tn * BN;
    const int kb = static_cast<int>(blk_count(a.K));
    const int k0 = split * per, k1 = k0 + per < kb ? k0 + per : kb;
    const int64_t ld = static_cast<int64_t>(kb) * kBlk;
    const int64_t nb = blk_count(a.N);
    const int64_t rows_a = a.M - m0 < BM ? a.M - m0 : BM, rows_w = a.N - n0 < BN ? a.N - n0 : BN;

    // Loads of K block k into a stage.  1 KB load c of this wave fills rows
    // 8 q .. 8 q + 7 (q = wid + WAVES c; A's rows, then W's): lane l fills slot
    // l % 8 of row 8 q + l / 8, which holds 16-byte group (l % 8) ^ ((row >> 1) & 7),
    // so that the 16 rows a fragment read takes at once lie in different banks.
    // A block past the last gets an empty range: it fetches nothing, and every
    // step issues the same number of loads.
    const uint32_t lds0 = wide_lds_addr(lds);
    int voff[T::NL];
#pragma unroll
    for (int c = 0; c < T::NL; ++c) {
        const int row = 8 * (wid + T::WAVES * c) + (lane >> 3);
        const int grp = (lane & 7) ^ ((row >> 1) & 7);
        voff[c] = static_cast<int>((row < BM ? row : row - BM) * ld) + 16 * grp;
    }
    const uint8_t* baseA = a.A + m0 * ld;
    const uint8_t* baseW = a.W + n0 * ld;
    auto load = [&](int k, int s) {
        const bool on = k < k1;
        const v4u dA = wide_desc(baseA, on ? rows_a * ld : 0);
        const v4u dW = wide_desc(baseW, on ? rows_w * ld : 0);
        const uint32_t st = lds0 + s * T::STAGE;
#pragma unroll
        for (int c = 0; c < T::NL; ++c) {
            const int q = wid + T::WAVES * c;
            wide_dma(q < BM / 8 ? dA : dW, st + 1024 * q, voff[c], kBlk * k);
        }
        // Scales: wave w takes 64 of them, A's rows first, then W's (with BLOCKS
        // those of the tile's 128-blocks of columns, all by one wave); a wave with
        // none left fills its 256 bytes with zeros.
        const bool of_a = wid < BM / 64;
        const int w = of_a ? wid : wid - BM / 64;
        const int64_t left = of_a ? rows_a - 64 * w : BLOCKS ? (w == 0 ? nb - n0 / kBlk : 0) : rows_w - 64 * w;
        const float* src = of_a ? a.sA + k * a.M + m0 + 64 * w
                                : BLOCKS ? a.sW + k * nb + n0 / kBlk : a.sW + k * a.N + n0 + 64 * w;
        dma_dword(wide_desc(src, on ? (left < 64 ? left : 64) * 4 : 0), st + T::CODES + 256 * wid, 4 * lane, 0);
    };

    v4f acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    const int64_t ncol = n0 + 16 * TJ * wn;

    auto fragment = [&](const uint8_t* st, int row) {
        const uint8_t* p = st + row * kBlk;
        const int x = (row >> 1) & 7;
        const v4i lo = *reinterpret_cast<const v4i*>(p + 16 * (g ^ x));
        const v4i hi = *reinterpret_cast<const v4i*>(p + 16 * ((g + 4) ^ x));
        return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };

#pragma unroll
    for (int s = 0; s < LEAD; ++s) load(k0 + s, s);
    int stage = 0;
    // One K block: row tile i's products are issued while row tile i - 1's sums
    // join the accumulators (four FMAs behind each product) and row tile i + 1's
    // codes come from LDS.  With a weight's scales the last row tile's sums wait
    // in registers for the next block, past the barrier and its LDS latency.
    v4f d[2][TJ];
    float pend = 0.0f;
#pragma unroll
    for (int j = 0; j < TJ; ++j) d[1][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = k0; k < k1; ++k) {
        wait_barrier<(LEAD - 1) * T::LOADS>();
        {
            const int ns = stage + LEAD;
            load(k + LEAD, ns >= T::NS ? ns - T::NS : ns);
        }
        const uint8_t* st = lds + stage * T::STAGE;
        const float* sc = reinterpret_cast<const float*>(st + T::CODES);
        stage = stage + 1 == T::NS ? 0 : stage + 1;

        // Fragments run ahead of the products: one row tile for the FP8
        // instruction, two for the bf16 one, whose operands are converted a row
        // tile ahead.
        constexpr int AHEAD = FP8 ? 1 : 2;
        v8i wf[TJ], xf[2];
        v4f swv[TJ];
        float sa[TI];
        auto xfrag = [&](int i) { return fragment(st, 16 * TI * wm + 16 * i + r); };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) xf[i] = xfrag(i);
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            wf[j] = fragment(st + BM * kBlk, 16 * TJ * wn + 16 * j + r);
            if constexpr (!BLOCKS) swv[j] = *reinterpret_cast<const v4f*>(sc + BM + 16 * TJ * wn + 16 * j + 4 * g);
        }
        const float sw = BLOCKS ? sc[BM + 16 * TJ * wn / kBlk] : 1.0f;
#pragma unroll
        for (int i = 0; i < TI; ++i) sa[i] = sc[16 * TI * wm + 16 * i + r];
        auto join = [&](int i, const v4f (&dd)[TJ], int j, float s) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
                acc[i][j][v] = __builtin_fmaf(BLOCKS ? dd[j][v] : dd[j][v] * swv[j][v], s, acc[i][j][v]);
        };
        Bf16x32 wb[FP8 ? 1 : TJ], xb[FP8 ? 1 : 2];
        if constexpr (!FP8) {
#pragma unroll
            for (int j = 0; j < TJ; ++j) wb[j] = to_bf16(wf[j]);
            xb[0] = to_bf16(xf[0]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TI; ++i) {
            const int pi = (i + TI - 1) % TI;
            const bool joins = i > 0 || BLOCKS, reads = i + AHEAD < TI;
            if constexpr (FP8) {
                if (reads) xf[(i + 1) & 1] = xfrag(i + 1);
#pragma unroll
                for (int j = 0; j < TJ; ++j) {
                    d[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        wf[j], xf[i & 1], v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
                    if (joins) join(pi, d[(i + 1) & 1], j, pend);
                }
                if (reads) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);     // LDS reads
#pragma unroll
                for (int j = 0; j < TJ; ++j) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);            // a product
                    if (joins) __builtin_amdgcn_sched_group_barrier(0x002, BLOCKS ? 4 : 8, 0);
                }
            } else {
                if (i + 1 < TI) xb[(i + 1) & 1] = to_bf16(xf[(i + 1) & 1]);
                if (reads) xf[i & 1] = xfrag(i + 2);
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int j = 0; j < TJ; ++j)
                        d[i & 1][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            wb[j].q[q], xb[i & 1].q[q], q ? d[i & 1][j] : v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
                if (joins) {
#pragma unroll
                    for (int j = 0; j < TJ; ++j) join(pi, d[(i + 1) & 1], j, pend);
                }
                if (reads) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
                for (int j = 0; j < 4 * TJ; ++j) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (i + 1 < TI) __builtin_amdgcn_sched_group_barrier(0x002, 4 / TJ, 0);   // a conversion
                    if (joins) __builtin_amdgcn_sched_group_barrier(0x002, BLOCKS ? 1 : 2, 0);
                }
            }
            pend = sa[i] * sw;
            __builtin_amdgcn_sched_barrier(0);
        }
        static_assert(TI % 2 == 0, "the pending sums are those of an odd row tile");
        if constexpr (!BLOCKS) {
#pragma unroll
            for (int j = 0; j < TJ; ++j) join(TI - 1, d[1], j, pend);
        }
    }
    if constexpr (BLOCKS) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[TI - 1][j][v] = __builtin_fmaf(d[1][j][v], pend, acc[TI - 1][j][v]);
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");   // the empty loads past the last block

    if (splits > 1) {
        BlockGemmArgs p = a;
        p.C = part + split * a.M * a.N;
        p.ldc = a.N;
        p.bias = nullptr;
        p.act = NFLOW_ACT_NONE;
        const bool vec = a.N % 4 == 0;
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j)
                store4<float>(p, m0 + 16 * TI * wm + 16 * i + r, ncol + 16 * j + 4 * g, acc[i][j], vec);
        return;
    }
    const bool vec = a.ldc % 4 == 0 && (reinterpret_cast<uintptr_t>(a.C) & (4 * sizeof(TO) - 1)) == 0;
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
            store4<TO>(a, m0 + 16 * TI * wm + 16 * i + r, ncol + 16 * j + 4 * g, acc[i][j], vec);
}

}  // namespace nfq
