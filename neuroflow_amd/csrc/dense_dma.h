// dense_dma.h -- the tiled product of bf16 operands that the LDS-DMA can fetch:
// 16-byte aligned, a whole number of 8 values in every row.
//
// Bound by the matrix cores and the clock they run at under load: 8192 x 8192 x
// 8192 with bias and GELU 777 us (1415 TFLOP/s, MFMA 74% of the SIMD-cycles, VALU 28%,
// LDS conflicts under 1%), a library product alone 685 to 718.  Over few K steps a
// tile's start and stores weigh: dx of 65536 x 1024 x 1024, 16 steps, MFMA 41%; dW of
// it, whose 16 tiles 16 workgroups share each, 52%.
#pragma once

#include "dense_kernel.h"

namespace nfq {

// The byte ranges and offsets of an operand's loads.  One 1 KB load of a wave
// fills rows of the stage in LDS: along k 8 rows of 128 bytes, across k 1 KB /
// (2 R) rows.  Load c of wave w is region w + WAVES c; the permutation of a row's groups
// repeats every 16 rows, so a lane has one offset for even and one for odd loads.
template <bool ACROSS, int R, int WAVES>
struct DenseFetch {
    static constexpr int KB = 64;
    static constexpr int ROWS = ACROSS ? 512 / R : 8;            // rows of the stage in 1 KB
    static constexpr int N = (ACROSS ? KB : R) / (ROWS * WAVES);  // loads of a wave
    static_assert((ACROSS ? KB : R) % (ROWS * WAVES) == 0 && ROWS * WAVES % 8 == 0, "loads spread evenly");
    const uint8_t* base;
    int64_t ld2, row0, rows, K;      // bytes of a row in memory; first row, rows, k's in all
    int voff[2];                     // this lane's offset within its region's rows, of even and of odd loads
    int tail[2];                     // the same in the stage where k runs out
    int tail_k;                      // which that is
    __device__ __forceinline__ DenseFetch(const void* p, int64_t ld, int64_t row0_, int64_t rows_, int64_t K_, int wid)
        : ld2(2 * ld), row0(row0_), rows(rows_), K(K_) {
        const int lane = threadIdx.x & 63;
        base = static_cast<const uint8_t*>(p);
        if constexpr (!ACROSS) {
            base += row0 * ld2;
            tail_k = static_cast<int>(K / KB);
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                const int i = ROWS * wid + (lane >> 3), c = (lane & 7) ^ (((i + ROWS * WAVES * odd) >> 1) & 7);
                voff[odd] = static_cast<int>(i * ld2) + 16 * c;
                tail[odd] = tail_k * KB + 8 * c < K ? voff[odd] : INT32_MIN;   // past every range
            }
        } else {
            constexpr int L = R / 8;                             // lanes of a row
            base += 2 * row0;
            tail_k = -1;
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                const int i = ROWS * wid + lane / L, k = i + ROWS * WAVES * odd, p8 = lane % L;
                const int f = ((k & 3) | ((k >> 1) & 4)) & (R / 16 - 1);
                voff[odd] = static_cast<int>(i * ld2) + 16 * ((((p8 >> 1) ^ f) << 1) | (p8 & 1));
            }
        }
    }
    // The memory of stage k (none of it where `on` is not): base and bytes.
    __device__ __forceinline__ v4u range(int k, bool on) const {
        if constexpr (!ACROSS) {
            const int64_t left = rows - row0 < R ? rows - row0 : R;
            return wide_desc(base, on ? (left - 1) * ld2 + 2 * dense_pitch(K) : 0);
        } else {
            const int64_t at = static_cast<int64_t>(k) * KB, left = K - at < KB ? K - at : KB;
            return wide_desc(base + at * ld2, on ? (left - 1) * ld2 + 2 * (dense_pitch(rows) - row0) : 0);
        }
    }
    // Load c of stage k to `lds`, this operand's region.
    __device__ __forceinline__ void load(v4u desc, int k, uint32_t lds, int wid, int c) const {
        const int at = ROWS * WAVES * c * static_cast<int>(ld2) + (ACROSS ? 0 : 128 * k);   // the round's first row, the stage
        const int v = !ACROSS && k == tail_k ? tail[c & 1] : voff[c & 1];
        wide_dma(desc, lds + 1024 * (wid + WAVES * c), v + at, 0);
    }
};

// A stage, 64 k's, is computed in two halves of 32.  While one half is
// multiplied, the other's fragments come from LDS, and the block's one barrier a
// stage stands between the halves: by then all of the stage is in registers, so
// its memory takes the loads of the stage NS on, and the next stage, whose loads
// are waited for there, gives its first fragments.  Reads and loads are spread
// evenly, a few ahead of every row tile's products.
// SUMS: with the sums of a's rows.
template <bool AX, bool BX, bool SUMS, typename Tile>
__device__ __forceinline__ void dense_dma_tile(const DenseArgs& a, const DenseSlots& sl, const TilePos& pos, int k0, int k1,
                                               int slot) {
    constexpr int TI = Tile::TI, TJ = Tile::TJ, NS = Tile::NS;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wid / Tile::WN, wn = wid % Tile::WN;
    const uint32_t lds0 = wide_lds_addr(lds);
    const int64_t m0 = pos.tm * Tile::BM, n0 = pos.tn * Tile::BN;
    const DenseFetch<AX, Tile::BM, Tile::WAVES> fa(a.A, a.lda, m0, a.M, a.K, wid);
    const DenseFetch<BX, Tile::BN, Tile::WAVES> fb(a.B, a.ldb, n0, a.N, a.K, wid);
    constexpr int NA = fa.N, LOADS = fa.N + fb.N;                  // loads of a wave: A's, of a stage
    static_assert((NS - 1) * LOADS < 64, "vmcnt field");
    // Load c of stage k, whose ranges are da and db, into the memory of stage s.
    auto load = [&](v4u da, v4u db, int k, int s, int c) {
        if (c < NA) fa.load(da, k, lds0 + s * Tile::STAGE, wid, c);
        else fb.load(db, k, lds0 + s * Tile::STAGE + Tile::PLANE_A, wid, c - NA);
    };

    v4f acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    DenseSums<Tile> sums(SUMS && pos.tn == 0, wn);
    const int arow = 16 * TI * wm, brow = 16 * TJ * wn;
    v8bf xa[2][TI], xb[2][TJ];
    // Fragment e of half h of a stage: the TJ of B, then the TI of A, in the order of need.
    auto read = [&](const uint8_t* st, int h, int e) {
        if (e < TJ) xb[h][e] = dense_fragment<BX, Tile::BN, 64>(st + Tile::PLANE_A, brow + 16 * e, 32 * h);
        else xa[h][e - TJ] = dense_fragment<AX, Tile::BM, 64>(st, arow + 16 * (e - TJ), 32 * h);
    };
    auto products = [&](int h, int i) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[h][j], xa[h][i], acc[i][j], 0, 0, 0);
        if constexpr (SUMS) {
            const v8bf one[1] = {xa[h][i]};
            sums.add(i, one);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int F = TI + TJ, EACH = (F + TI - 1) / TI, LEACH = (LOADS + TI - 1) / TI;

#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int c = 0; c < LOADS; ++c)
            load(fa.range(k0 + s, k0 + s < k1), fb.range(k0 + s, k0 + s < k1), k0 + s, s, c);
    wait_barrier<(NS - 1) * LOADS>();
#pragma unroll
    for (int e = 0; e < F; ++e) read(lds, 0, e);
    int s = 0;
    for (int k = k0; k < k1; ++k) {
        const uint8_t* st = lds + s * Tile::STAGE;
        const v4u da = fa.range(k + NS, k + NS < k1), db = fb.range(k + NS, k + NS < k1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TI; ++i) {
#pragma unroll
            for (int e = EACH * i; e < EACH * (i + 1) && e < F; ++e) read(st, 1, e);
            products(0, i);
        }
        wait_barrier<(NS - 2) * LOADS>();
        const int next = s + 1 == NS ? 0 : s + 1;
        st = lds + next * Tile::STAGE;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TI; ++i) {
#pragma unroll
            for (int e = EACH * i; e < EACH * (i + 1) && e < F; ++e) read(st, 0, e);
#pragma unroll
            for (int c = LEACH * i; c < LEACH * (i + 1) && c < LOADS; ++c) load(da, db, k + NS, s, c);
            products(1, i);
        }
        s = next;
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");   // the empty loads past the last stage
    if constexpr (SUMS) sums.leave(a, sl, m0, slot, wm);
    __syncthreads();
    dense_leave<bf16, Tile>(a, sl, acc, reinterpret_cast<float*>(lds) + wid * Tile::STRIP, m0, n0, slot, wm, wn);
}

template <bool AX, bool BX, bool SUMS, typename Tile>
__global__ __launch_bounds__(Tile::THREADS, Tile::OCC) void k_dense_dma(DenseArgs a, DenseShare sh) {
    dense_each(sh, [&](int64_t tile, int k0, int k1, int slot) {
        dense_dma_tile<AX, BX, SUMS, Tile>(a, DenseSlots{sh.part, sh.groups}, tile_pos(tile, sh.tiles_m, sh.tiles_n, 4), k0, k1,
                                     slot);
    });
}

}  // namespace nfq
