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
// of magnitudes over all finite codes, whatever K.  Rounding to bf16 costs
// 1.7e-3 in the 2-norm, so as a whole a result is no less exact; one whose
// products cancel to under an eighth of their magnitudes may lose more here than
// in its rounding.  That is the price of twice the bf16 instruction's rate
// (8192 x 8192 x 8192: 473 us against 876), and the type of the result chooses.
// fp32 outputs take the bf16 instruction on the codes' values, which are exact
// in bf16 (1e-8 to 1e-7 of the result), at half the rate.
//
// The weight is the A operand, so a lane holds four adjacent columns of one
// row: lane (r, g) = (l % 16, l / 16) of tile (i, j) has row 16 i + r and
// columns 16 j + 4 g .. + 3, and its row scale is one register per i.  Both
// operands take the bytes of 16-byte groups g and g + 4 of the row for lane
// group g: the same k on both sides, in an order of its own.
//
// Large products are bound by the matrix cores with the joins beside them, at the
// clock that such a load leaves: 8192 x 8192 x 8192 bf16 473 us, 2.3 PFLOP/s, the
// matrix cores busy 55% of the time and the VALU 42% (without the joins 457 us
// against 504 in one run); fp32 876 us with a weight's scales, 973 with a scale per
// row of both.  Few K blocks are bound by what a tile does outside its loop:
// 65536 x 1024 x 1024 bf16 82 us, 1.7 PFLOP/s.
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
    static constexpr int STRIP_ROW = 16 * TJ + 4, STRIP = 16 * STRIP_ROW;   // floats of a wave's 16 rows on their way out
    static_assert(WAVES * STRIP * 4 <= NS * STAGE, "the strips fit the stages");
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
        const v4t q{from_f32<TO>(y[0]), from_f32<TO>(y[1]), from_f32<TO>(y[2]), from_f32<TO>(y[3])};
        *reinterpret_cast<v4t*>(c) = q;
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

// A wave's TI x TJ tiles of sums to rows m0 .., columns n0 .. of C, with bias
// and activation, through its strip of LDS.
// STREAM: non-temporal stores, for results that the caller's next launch reads,
// if at all, from beyond the L2 (65536 x 1024 x 1024: bf16 95 -> 88 us, fp32 172
// -> 156 us; 8192 x 8192 x 8192 515 -> 504 us).
template <typename TO, typename T, bool STREAM, int TI, int TJ>
__device__ __forceinline__ void store_tiles(const v4f (&acc)[TI][TJ], float* strip, TO* C, int64_t M, int64_t N,
                                            int64_t ldc, const float* bias, int act, int64_t m0, int64_t n0) {
    constexpr int V = 16 / sizeof(TO), LPR = 16 * TJ / V, RPI = 64 / LPR;   // values a lane, lanes a row, rows a store
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int row = lane / LPR, col = V * (lane % LPR);
    const int64_t n = n0 + col;
    const bool vec = n + V <= N && ldc % V == 0 && (reinterpret_cast<uintptr_t>(C) & 15) == 0;
    float b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) b[v] = bias && n + v < N ? bias[n + v] : 0.0f;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
#pragma unroll
        for (int j = 0; j < TJ; ++j) *reinterpret_cast<v4f*>(strip + r * T::STRIP_ROW + 16 * j + 4 * g) = acc[i][j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int q = 0; q < 16 / RPI; ++q) {
            const int64_t m = m0 + 16 * i + RPI * q + row;
            const float* p = strip + (RPI * q + row) * T::STRIP_ROW + col;
            float y[V];
#pragma unroll
            for (int v = 0; v < V; v += 4) {
                const v4f z = *reinterpret_cast<const v4f*>(p + v);
#pragma unroll
                for (int u = 0; u < 4; ++u) y[v + u] = z[u] + b[v + u];
            }
            if (act == NFLOW_ACT_RELU) {
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = activate<ACT_RELU>(y[v]);
            } else if (act == NFLOW_ACT_GELU_TANH) {
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = activate<ACT_GELU_TANH>(y[v]);
            }
            if (m >= M) continue;
            TO* c = C + m * ldc + n;
            if (vec) {
                typedef TO vt __attribute__((ext_vector_type(V)));
                vt o;
#pragma unroll
                for (int v = 0; v < V; ++v) o[v] = from_f32<TO>(y[v]);
                if constexpr (STREAM) __builtin_nontemporal_store(o, reinterpret_cast<vt*>(c));
                else *reinterpret_cast<vt*>(c) = o;
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (n + v < N) c[v] = from_f32<TO>(y[v]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// TO: type of C, and with it the instruction.  BLOCKS: a weight's scales (one
// per 128 x 128), else one per row of W.  With splits > 1 the K blocks are
// dealt out in runs of `per`, and split s writes its fp32 sums, unscaled by
// anything further, to part[s] (M, N).
struct GemmShare {
    int64_t tiles_m, tiles_n;
    int splits, per;
    float* part;
    int blocks;         // workgroups of the product
};
template <typename TO, bool BLOCKS, typename T>
__device__ __forceinline__ void gemm_tile(const BlockGemmArgs& a, const GemmShare& sh, int bid) {
    constexpr bool FP8 = std::is_same_v<TO, bf16>;
    constexpr int TI = T::TI, TJ = T::TJ, BM = T::BM, BN = T::BN, LEAD = T::NS - 1;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wid / T::WN, wn = wid % T::WN;
    const int r = lane & 15, g = lane >> 4;
    const int64_t t = gemm_tile_of_block(bid, sh.blocks, 8);
    const int splits = sh.splits, per = sh.per;
    const int split = splits > 1 ? static_cast<int>(t % splits) : 0;
    const TilePos pos = tile_pos(splits > 1 ? t / splits : t, sh.tiles_m, sh.tiles_n, 4);
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
    // A load's rows are in its range's base, so one offset register serves all.
    // A block past the last gets empty ranges: it fetches nothing, and every
    // step issues the same number of loads.
    const uint32_t lds0 = wide_lds_addr(lds);
    constexpr int ROWS = 8 * T::WAVES, NLA = BM / ROWS;      // rows per round of loads, rounds of A's
    static_assert(BM % ROWS == 0 && BN % ROWS == 0 && ROWS % 16 == 0, "rounds of A's and of W's rows");
    const int lrow = 8 * wid + (lane >> 3);
    const int voff = static_cast<int>(lrow * ld) + 16 * ((lane & 7) ^ ((lrow >> 1) & 7));
    const uint8_t* baseA = a.A + m0 * ld;
    const uint8_t* baseW = a.W + n0 * ld;
    auto load_codes = [&](int k, int s, int c) {
        const int64_t left = c < NLA ? rows_a - ROWS * c : rows_w - ROWS * (c - NLA);
        const uint8_t* base = c < NLA ? baseA + ROWS * c * ld : baseW + ROWS * (c - NLA) * ld;
        wide_dma(wide_desc(base, k < k1 ? left * ld : 0), lds0 + s * T::STAGE + 1024 * (wid + T::WAVES * c), voff,
                 kBlk * k);
    };
    // Scales: wave w takes 64 of them, A's rows first, then W's (with BLOCKS
    // those of the tile's 128-blocks of columns, all by one wave); a wave with
    // none left fills its 256 bytes with zeros.
    const bool of_a = wid < BM / 64;
    const int sw_at = of_a ? wid : wid - BM / 64;
    const int64_t s_left = of_a ? rows_a - 64 * sw_at
                                : BLOCKS ? (sw_at == 0 ? nb - n0 / kBlk : 0) : rows_w - 64 * sw_at;
    const int64_t s_bytes = (s_left < 64 ? s_left : 64) * 4, s_step = of_a ? a.M : BLOCKS ? nb : a.N;
    const float* s_src = of_a ? a.sA + m0 + 64 * sw_at : BLOCKS ? a.sW + n0 / kBlk : a.sW + n0 + 64 * sw_at;
    s_src += k0 * s_step;                                    // of the block whose turn is next
    auto load_scales = [&](int k, int s) {
        dma_dword(wide_desc(s_src, k < k1 ? s_bytes : 0), lds0 + s * T::STAGE + T::CODES + 256 * wid, 4 * lane, 0);
        s_src += s_step;
    };
    auto load = [&](int k, int s) {
#pragma unroll
        for (int c = 0; c < T::NL; ++c) load_codes(k, s, c);
        load_scales(k, s);
    };

    v4f acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    const int64_t ncol = n0 + 16 * TJ * wn;

    // Fragments of 16-row tile i (of A) or j (of W) of a stage: two reads at an
    // immediate offset from a lane's place in the first tile, whose swizzle is
    // that of every tile (16 rows on).
    const int flo = r * kBlk + 16 * (g ^ ((r >> 1) & 7)), fhi = flo ^ 64;
    const int xat = 16 * TI * wm, wat = BM + 16 * TJ * wn;   // first rows in the stage
    auto fragment = [&](const uint8_t* st, int row0, int i) {
        const v4i lo = *reinterpret_cast<const v4i*>(st + (row0 * kBlk + flo) + 16 * kBlk * i);
        const v4i hi = *reinterpret_cast<const v4i*>(st + (row0 * kBlk + fhi) + 16 * kBlk * i);
        return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    auto xscale_of = [&](const uint8_t* st, int i) {
        return reinterpret_cast<const float*>(st + T::CODES + 4 * (xat + r))[16 * i];
    };

    v4f d[2][TJ];
    float pend = 0.0f;
#pragma unroll
    for (int j = 0; j < TJ; ++j) d[1][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    static_assert(TI % 2 == 0, "the pending sums are those of an odd row tile");

    if constexpr (FP8 && BLOCKS && T::NS == 2) {
        // One K block: row tile i's products are issued while row tile i - 1's sums
        // join the accumulators (four FMAs behind each product) and row tile i + 1's
        // codes come from LDS.  The block's barrier stands before its last row
        // tile, whose codes are in registers by then: past it the stage is free
        // for the block after next, the next block's stage is complete, and its
        // first fragments arrive under the last row tile's products.  The last
        // sums join in the next block.
        load(k0, 0);
        load(k0 + 1, 1);
        wait_barrier<T::LOADS>();
        const uint8_t* st = lds;
        auto xfrag = [&](int i) { return fragment(st, xat, i); };
        auto wfrag = [&](int j) { return fragment(st, wat, j); };
        auto xscale = [&](int i) { return xscale_of(st, i); };
        auto wscale = [&] { return reinterpret_cast<const float*>(st + T::CODES)[BM + 16 * TJ * wn / kBlk]; };
        v8i wf[TJ], xf[2];
#pragma unroll
        for (int j = 0; j < TJ; ++j) wf[j] = wfrag(j);
        xf[0] = xfrag(0);
        float sx = xscale(0), sw = wscale();
        auto product = [&](int i, int j) {
            d[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], xf[i & 1], v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0,
                                                                          0, 0, 0, 0, 0);
            const int pi = (i + TI - 1) % TI;
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[pi][j][v] = __builtin_fmaf(d[(i + 1) & 1][j][v], pend, acc[pi][j][v]);
        };
        int s = 0;
        for (int k = k0; k < k1; ++k) {
#pragma unroll
            for (int i = 0; i < TI - 1; ++i) {
                xf[(i + 1) & 1] = xfrag(i + 1);
                const float sn = xscale(i + 1);
#pragma unroll
                for (int j = 0; j < TJ; ++j) product(i, j);
                __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);            // LDS reads
#pragma unroll
                for (int j = 0; j < TJ; ++j) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);        // a product
                    __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);        // four FMAs
                }
                pend = sx * sw;
                sx = sn;
                __builtin_amdgcn_sched_barrier(0);
            }
            wait_barrier<0>();
            st = lds + (s ^ 1) * T::STAGE;
            __builtin_amdgcn_sched_barrier(0);
            xf[0] = xfrag(0);
            const float sn = xscale(0), swn = wscale();
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                product(TI - 1, j);
                wf[j] = wfrag(j);
#pragma unroll
                for (int c = j; c < T::NL; c += TJ) load_codes(k + 2, s, c);
                if (j == TJ - 1) load_scales(k + 2, s);
                __builtin_amdgcn_sched_barrier(0);
            }
            pend = sx * sw;
            sx = sn;
            sw = swn;
            s ^= 1;
        }
    } else {
#pragma unroll
    for (int s = 0; s < LEAD; ++s) load(k0 + s, s);
    int stage = 0;
    // As above, with one barrier at the block's start, and the sums of the last
    // row tile joined at its end.
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
        auto xfrag = [&](int i) { return fragment(st, xat, i); };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) xf[i] = xfrag(i);
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            wf[j] = fragment(st, wat, j);
            if constexpr (!BLOCKS) swv[j] = *reinterpret_cast<const v4f*>(sc + BM + 16 * TJ * wn + 16 * j + 4 * g);
        }
        const float sw = BLOCKS ? sc[BM + 16 * TJ * wn / kBlk] : 1.0f;
#pragma unroll
        for (int i = 0; i < TI; ++i) sa[i] = xscale_of(st, i);
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
                    if (i + 1 < TI) __builtin_amdgcn_sched_group_barrier(0x002, TJ >= 4 ? 1 : 4 / TJ, 0);   // conversions
                    if (joins) __builtin_amdgcn_sched_group_barrier(0x002, BLOCKS ? 1 : 2, 0);
                }
            }
            pend = sa[i] * sw;
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!BLOCKS) {
#pragma unroll
            for (int j = 0; j < TJ; ++j) join(TI - 1, d[1], j, pend);
        }
    }
    }
    if constexpr (BLOCKS) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[TI - 1][j][v] = __builtin_fmaf(d[1][j][v], pend, acc[TI - 1][j][v]);
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");   // the empty loads past the last block

    // Results leave through LDS (the stages' memory), a row tile at a time: a
    // wave writes its 16 rows as the products hold them and reads them back along
    // the rows, so that its stores are whole 128-byte lines.
    __syncthreads();
    float* strip = reinterpret_cast<float*>(lds) + wid * T::STRIP;
    if (splits > 1)
        store_tiles<float, T, false>(acc, strip, sh.part + split * a.M * a.N, a.M, a.N, a.N, nullptr, NFLOW_ACT_NONE,
                              m0 + xat, ncol);
    else
        store_tiles<TO, T, true>(acc, strip, static_cast<TO*>(a.C), a.M, a.N, a.ldc, a.bias, a.act, m0 + xat, ncol);
}

template <typename TO, bool BLOCKS, typename T>
__global__ __launch_bounds__(T::THREADS, 2) void k_block_gemm(BlockGemmArgs a, GemmShare sh) {
    gemm_tile<TO, BLOCKS, T>(a, sh, blockIdx.x);
}

// Two independent fp32 products in one launch, a's workgroups first: where
// neither fills the chip evenly by itself, one's workgroups run in the CUs that
// the other leaves idle at its end.
template <typename T>
__global__ __launch_bounds__(T::THREADS, 2) void k_block_gemm_pair(BlockGemmArgs a, GemmShare sa, BlockGemmArgs b,
                                                                   GemmShare sb) {
    if (static_cast<int>(blockIdx.x) < sa.blocks) gemm_tile<float, false, T>(a, sa, blockIdx.x);
    else gemm_tile<float, true, T>(b, sb, blockIdx.x - sa.blocks);
}

}  // namespace nfq
