// dense_f32.hip -- the tiled product of fp32 operands.
//
// An fp32 value is three bf16 planes, x = h + m + l: each the rest rounded to
// bf16's 8 bits, so the 24 bits are held exactly.  Six products (h h, h m, m h, m m,
// h l, l h) leave out m l, l m and l l: of a value in [1, 2) |m| <= 2^-8 and |l| <=
// 2^-17, so at most 2^-24 of the product, half a step of fp32.  That is fp32 accuracy at a
// sixth of the bf16 rate, where the fp32 instruction has a sixteenth.  The planes are
// formed once per workgroup, on the way from memory to LDS through registers, so
// operands need no alignment and no launch ahead.
//
// Bound by forming the planes beside the products: 4096 x 4096 x 4096 620 us (222
// TFLOP/s; the fp32 library's product 153), where six bf16 products at a library's 1350
// TFLOP/s are 611.  Over fewer K steps a tile's start and stores weigh: 5003 x 1000 ->
// 1544 backward, the pair of products 202 us under a trace, MFMA 48% of the SIMD-cycles,
// VALU 46%; 32768 x 256 -> 256, eight steps of 32 a tile, 33 us a call, MFMA 25%, VALU 30%.
#include "dense_kernel.h"
#include "dense_split.h"

namespace nfq {
namespace {

// An operand's share of a stage by way of registers: CH groups of 8 values a thread.
template <bool ACROSS, int R, int KB, int THREADS>
struct DenseStage {
    static constexpr int CH = R * KB / 8 / THREADS;
    static_assert(R * KB / 8 % THREADS == 0, "groups spread evenly");
    static constexpr int PER = (ACROSS ? R : KB) / 8;              // groups of a row in memory
    Raw8<float> v[CH];
    // Rows row0 .. of `rows`, k's k0 .. of K.
    __device__ __forceinline__ void load(const float* base, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int64_t K) {
        const bool inside = row0 + R <= rows && k0 + KB <= K;
#pragma unroll
        for (int q = 0; q < CH; ++q) {
            const int id = threadIdx.x + THREADS * q, i = id / PER, c = 8 * (id % PER);
            const int64_t major = (ACROSS ? k0 : row0) + i, minor = (ACROSS ? row0 : k0) + c;
            const float* p = base + major * ld + minor;
            if (inside) v[q].load(p, 8);
            else dense_load(v[q], p, major < (ACROSS ? K : rows) ? (ACROSS ? rows : K) - minor : 0);
        }
    }
    __device__ __forceinline__ void store(uint8_t* planes) const {
#pragma unroll
        for (int q = 0; q < CH; ++q) {
            const int id = threadIdx.x + THREADS * q;
            uint8_t* to = planes + dense_place<ACROSS, R, KB>(id / PER, id % PER);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = v[q][e];
            v8bf p[3];
            dense_split(x, p);
#pragma unroll
            for (int s = 0; s < 3; ++s) *reinterpret_cast<v8bf*>(to + s * R * KB * 2) = p[s];
        }
    }
};

// Products of one stage, row tiles i0 .. i1 - 1 of a wave; of a row tile the
// planes' products of the least first.
template <bool AX, bool BX, typename Tile>
struct StageProducts {
    v8bf b[3][Tile::TJ];
    __device__ __forceinline__ explicit StageProducts(const uint8_t* st, int brow) {
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int j = 0; j < Tile::TJ; ++j)
                b[p][j] = dense_fragment<BX, Tile::BN, 32>(st + 3 * Tile::PLANE_A + p * Tile::PLANE_B, brow + 16 * j, 0);
    }
    __device__ __forceinline__ void run(const uint8_t* st, v4f (&acc)[Tile::TI][Tile::TJ], DenseSums<Tile>& sums, int arow,
                                        int i0, int i1) const {
#pragma unroll
        for (int i = i0; i < i1; ++i) {
            v8bf a[3];
#pragma unroll
            for (int p = 0; p < 3; ++p) a[p] = dense_fragment<AX, Tile::BM, 32>(st + p * Tile::PLANE_A, arow + 16 * i, 0);
            constexpr int pa[6] = {0, 2, 1, 0, 1, 0}, pb[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
            for (int q = 0; q < 6; ++q)
#pragma unroll
                for (int j = 0; j < Tile::TJ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[pb[q]][j], a[pa[q]], acc[i][j], 0, 0, 0);
            if constexpr (AX) sums.add(i, a);
        }
    }
};

// One barrier a stage: while stage k is multiplied, stage k + 1 is split into the
// other half of LDS and stage k + 2 is on its way from memory.  One half of the
// waves splits before its products and the other between them, so that a SIMD's
// two waves use the VALU and the matrix core in turn.
template <bool AX, bool BX, typename Tile>
__device__ __forceinline__ void dense_f32_tile(const DenseArgs& a, const DenseSlots& sl, const TilePos& pos, int k0, int k1,
                                               int slot) {
    constexpr int TI = Tile::TI, TJ = Tile::TJ;
    static_assert(Tile::KB == 32 && Tile::P == 3 && Tile::NS == 2, "two stages of three planes");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wid / Tile::WN, wn = wid % Tile::WN;
    const int64_t m0 = pos.tm * Tile::BM, n0 = pos.tn * Tile::BN;
    v4f acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    DenseStage<AX, Tile::BM, 32, Tile::THREADS> ra;
    DenseStage<BX, Tile::BN, 32, Tile::THREADS> rb;
    auto load = [&](int k) {
        ra.load(static_cast<const float*>(a.A), a.lda, m0, a.M, static_cast<int64_t>(k) * 32, k < k1 ? a.K : 0);
        rb.load(static_cast<const float*>(a.B), a.ldb, n0, a.N, static_cast<int64_t>(k) * 32, k < k1 ? a.K : 0);
    };
    auto store = [&](int s) {
        ra.store(lds + s * Tile::STAGE);
        rb.store(lds + s * Tile::STAGE + 3 * Tile::PLANE_A);
    };
    DenseSums<Tile> sums(AX && a.sums && pos.tn == 0, wn);
    const int arow = 16 * TI * wm, brow = 16 * TJ * wn;
    load(k0);
    store(0);
    load(k0 + 1);
    __syncthreads();
    int s = 0;
    for (int k = k0; k < k1; ++k, s ^= 1) {
        const uint8_t* st = lds + s * Tile::STAGE;
        const StageProducts<AX, BX, Tile> stage(st, brow);
        const bool first = wid < Tile::WAVES / 2;
        if (first) {
            store(s ^ 1);
            load(k + 2);
        }
        stage.run(st, acc, sums, arow, 0, TI / 2);
        if (!first) {
            store(s ^ 1);
            load(k + 2);
        }
        stage.run(st, acc, sums, arow, TI / 2, TI);
        __syncthreads();
    }
    if constexpr (AX) sums.leave(a, sl, m0, slot, wm);
    dense_leave<float, Tile>(a, sl, acc, reinterpret_cast<float*>(lds) + wid * Tile::STRIP, m0, n0, slot, wm, wn);
}

template <bool AX, bool BX, typename Tile>
__global__ __launch_bounds__(Tile::THREADS, Tile::OCC) void k_dense_f32(DenseArgs a, DenseShare sh) {
    dense_each(sh, [&](int64_t tile, int k0, int k1, int slot) {
        dense_f32_tile<AX, BX, Tile>(a, DenseSlots{sh.part, sh.groups}, tile_pos(tile, sh.tiles_m, sh.tiles_n, 4), k0, k1,
                                     slot);
    });
}

template <typename Tile>
__global__ __launch_bounds__(Tile::THREADS, Tile::OCC) void k_dense_f32_pair(DensePair pr) {
    dense_each_pair(pr, [&](int which, int64_t tile, int k0, int k1, int slot) {
        const TilePos pos = tile_pos(tile, pr.tiles_m[which], pr.tiles_n[which], 4);
        const DenseSlots sl{pr.part, pr.groups};
        if (which == 0) dense_f32_tile<false, true, Tile>(pr.a[0], sl, pos, k0, k1, slot);
        else dense_f32_tile<true, true, Tile>(pr.a[1], sl, pos, k0, k1, slot);
    });
}

// As with bf16, larger tiles split each value fewer times: 256 x 128 once for 256 or 128
// products, 64 x 64 once for 64 (4.8 us a step of 64 k's against 8 times 0.9).
using Small = DenseTile<float, 2, 2, 2, 2, 2>;     // 64 x 64, four waves, up to three workgroups a CU
using Mid = DenseTile<float, 2, 4, 4, 2, 2>;       // 128 x 128, eight waves, a workgroup a CU
using Big = DenseTile<float, 4, 2, 4, 4, 2>;       // 256 x 128, eight waves, a workgroup a CU

template <bool AX, bool BX>
void launch(const DenseArgs& a, const DensePlan& p, float* part, hipStream_t st) {
    if (p.kind == DENSE_SMALL) launch_dense_tile<float, Small, &k_dense_f32<AX, BX, Small>>(a, p, part, st);
    else if (p.kind == DENSE_MID) launch_dense_tile<float, Mid, &k_dense_f32<AX, BX, Mid>>(a, p, part, st);
    else launch_dense_tile<float, Big, &k_dense_f32<AX, BX, Big>>(a, p, part, st);
}

}  // namespace

void launch_dense_f32(const DenseArgs& a, DenseForm form, const DensePlan& p, float* part, hipStream_t st) {
    if (form == DENSE_FORWARD) launch<false, false>(a, p, part, st);
    else if (form == DENSE_DX) launch<false, true>(a, p, part, st);
    else launch<true, true>(a, p, part, st);
}

void launch_dense_pair_f32(const DenseArgs& dx, const DenseArgs& dw, const DensePlan& p, float* part, hipStream_t st) {
    if (p.kind == DENSE_SMALL) launch_dense_pair_tile<float, Small, &k_dense_f32_pair<Small>>(dx, dw, p, part, st);
    else if (p.kind == DENSE_MID) launch_dense_pair_tile<float, Mid, &k_dense_f32_pair<Mid>>(dx, dw, p, part, st);
    else launch_dense_pair_tile<float, Big, &k_dense_f32_pair<Big>>(dx, dw, p, part, st);
}

}  // namespace nfq
