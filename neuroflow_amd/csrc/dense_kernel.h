// dense_kernel.h -- what the tiled products of bf16 (dense_dma.h) and of fp32
// operands (dense_f32.hip) on the matrix cores share.
//
//   z[m][n] = sum_k a[m][k] b[n][k] + bias[n] + r[m][n],   C = act(z)
//
// Products are v_mfma_f32_16x16x32_bf16's: of bf16 values exact, sums fp32.  (The
// 32 x 32 x 16 one has the higher rate on zeros and the lower one on data, where
// power bounds the clock: 8192^3 in one run 863 us against 797.)
//
// An operand may lie along k or across it (the backward products read W, dz and
// x where they are): the stage in LDS then has rows of k, and the operands come
// from it by ds_read_b64_tr_b16, which hands each lane four values down a column.
#pragma once

#include <type_traits>

#include "block_gemm_kernel.h"
#include "dense.h"

namespace nfq {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;

// Tiles of BM x BN, WM x WN waves of TI x TJ 16 x 16 tiles each; a stage is KB
// values of k of every row in P planes, NS stages; OCC waves a SIMD.
template <typename T, int WM_, int WN_, int TI_, int TJ_, int NS_, int OCC_ = 2>
struct DenseTile {
    static constexpr int WM = WM_, WN = WN_, TI = TI_, TJ = TJ_, NS = NS_, OCC = OCC_;
    static constexpr int P = std::is_same_v<T, float> ? 3 : 1, KB = std::is_same_v<T, float> ? 32 : 64;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, PER_CU = 4 * OCC / WAVES;
    static constexpr int BM = 16 * TI * WM, BN = 16 * TJ * WN;
    static constexpr int PLANE_A = BM * KB * 2, PLANE_B = BN * KB * 2;       // bytes
    static constexpr int STAGE = P * (PLANE_A + PLANE_B);
    static constexpr int STRIP_ROW = 16 * TJ + 4, STRIP = 16 * STRIP_ROW;   // floats of a wave's 16 rows on their way out
    static constexpr int LDS = NS * STAGE > WAVES * STRIP * 4 ? NS * STAGE : WAVES * STRIP * 4;
    static_assert(PER_CU * LDS <= 160 * 1024, "a CU's LDS");
};

// Where 8 values lie in a plane: along k row `i` of the tile's R, group `c` of
// its KB / 8; across k row `i` of KB, group `c` of R / 8.  The groups of a row
// are permuted so that the rows that a read takes at once lie in different banks.
template <bool ACROSS, int R, int KB>
__device__ __forceinline__ int dense_place(int i, int c) {
    if constexpr (!ACROSS) {
        constexpr int G = KB / 8;
        return i * KB * 2 + 16 * (c ^ ((i >> 1) & (G - 1)));
    } else {
        constexpr int S = R / 16;                                  // pairs of groups: what a transposing read takes of a row
        const int f = ((i & 3) | ((i >> 1) & 4)) & (S - 1);
        return i * R * 2 + 16 * (((((c >> 1) ^ f)) << 1) | (c & 1));
    }
}

// A 16-row fragment of 32 k's: lane (r, g) = (l % 16, l / 16) has row row0 + r, k's
// k0 + 8 g .. + 7.
template <bool ACROSS, int R, int KB>
__device__ __forceinline__ v8bf dense_fragment(const uint8_t* plane, int row0, int k0) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    if constexpr (!ACROSS) {
        return *reinterpret_cast<const v8bf*>(plane + dense_place<false, R, KB>(row0 + r, k0 / 8 + g));
    } else {
        // Lane i of a group of 16 addresses row i / 4 and columns 4 (i % 4) .. + 3.
        union {
            v4s half[2];
            v8bf all;
        } u;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int k = k0 + 8 * g + 4 * q + (r >> 2), c = row0 + 4 * (r & 3);
            const uint8_t* p = plane + dense_place<true, R, KB>(k, c >> 3) + 2 * (c & 7);
            u.half[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)p);
        }
        return u.all;
    }
}

// Four outputs of a row from column n on: bias, residual, activation, one rounding.
template <typename T>
__device__ __forceinline__ void dense_finish(const DenseArgs& a, int64_t m, int64_t n, const v4f& s) {
    typedef T v4t __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (n + 3 < a.N) {
        v4f z = s;
        if (a.bias) {
#pragma unroll
            for (int v = 0; v < 4; ++v) z[v] += a.bias[n + v];
        }
        if (a.R) {
            const v4t r = *reinterpret_cast<const v4t*>(static_cast<const T*>(a.R) + m * a.ldr + n);
#pragma unroll
            for (int v = 0; v < 4; ++v) z[v] += to_f32(r[v]);
        }
        v4t y;
        if (a.Z) {
#pragma unroll
            for (int v = 0; v < 4; ++v) y[v] = from_f32<T>(z[v]);
            *reinterpret_cast<v4t*>(static_cast<T*>(a.Z) + m * a.ldz + n) = y;
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) y[v] = from_f32<T>(activate_rt(z[v], a.act));
        *reinterpret_cast<v4t*>(static_cast<T*>(a.C) + m * a.ldc + n) = y;
        return;
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        if (n + v >= a.N) return;
        float z = s[v] + (a.bias ? a.bias[n + v] : 0.0f);
        if (a.R) z += to_f32(static_cast<const T*>(a.R)[m * a.ldr + n + v]);
        if (a.Z) static_cast<T*>(a.Z)[m * a.ldz + n + v] = from_f32<T>(z);
        static_cast<T*>(a.C)[m * a.ldc + n + v] = from_f32<T>(activate_rt(z, a.act));
    }
}

// V values at p, together (at any element alignment) unless the row ends there.
template <typename T, bool STREAM, int V>
__device__ __forceinline__ void dense_put(T* p, const float (&y)[V], int64_t left) {
    if (left >= V) {
        typedef T vt __attribute__((ext_vector_type(V), aligned(sizeof(T))));
        vt o;
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = from_f32<T>(y[v]);
        if constexpr (STREAM) __builtin_nontemporal_store(o, reinterpret_cast<vt*>(p));
        else *reinterpret_cast<vt*>(p) = o;
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < left) p[v] = from_f32<T>(y[v]);
    }
}

// A wave's TI x TJ tiles of sums to rows m0 .., columns n0 .. of C, through its
// strip of LDS, so that loads and stores are whole lines.
// STREAM: non-temporal stores, of results; what the next launch reads stays in the caches.
template <typename T, typename Tile, bool STREAM>
__device__ __forceinline__ void dense_store(const DenseArgs& a, const v4f (&acc)[Tile::TI][Tile::TJ], float* strip,
                                            int64_t m0, int64_t n0) {
    constexpr int V = 16 / sizeof(T), LPR = 16 * Tile::TJ / V, RPI = 64 / LPR;   // values a lane, lanes a row, rows a store
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int row = lane / LPR, col = V * (lane % LPR);
    const int64_t n = n0 + col, left = a.N - n;
    float b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) b[v] = a.bias && v < left ? a.bias[n + v] : 0.0f;
#pragma unroll
    for (int i = 0; i < Tile::TI; ++i) {
        // The residual's values first: they arrive under the strip's round trip.
        typedef T vt __attribute__((ext_vector_type(V), aligned(sizeof(T))));
        vt res[16 / RPI];
        if (a.R) {
#pragma unroll
            for (int q = 0; q < 16 / RPI; ++q) {
                const int64_t m = m0 + 16 * i + RPI * q + row;
                const T* p = static_cast<const T*>(a.R) + m * a.ldr + n;
                if (m < a.M && left >= V) {
                    res[q] = *reinterpret_cast<const vt*>(p);
                } else {
                    const int64_t have = m < a.M ? left : 0;
#pragma unroll
                    for (int v = 0; v < V; ++v) res[q][v] = v < have ? p[v] : T(0.0f);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < Tile::TJ; ++j)
            *reinterpret_cast<v4f*>(strip + r * Tile::STRIP_ROW + 16 * j + 4 * g) = acc[i][j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int q = 0; q < 16 / RPI; ++q) {
            const int64_t m = m0 + 16 * i + RPI * q + row;
            const float* p = strip + (RPI * q + row) * Tile::STRIP_ROW + col;
            float y[V];
#pragma unroll
            for (int v = 0; v < V; v += 4) {
                const v4f z = *reinterpret_cast<const v4f*>(p + v);
#pragma unroll
                for (int u = 0; u < 4; ++u) y[v + u] = z[u] + b[v + u];
            }
            if (a.R) {
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] += to_f32(res[q][v]);
            }
            if (m >= a.M) continue;
            if (a.Z) dense_put<T, STREAM, V>(static_cast<T*>(a.Z) + m * a.ldz + n, y, left);
            if (a.act == NFLOW_ACT_RELU) {
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = activate<ACT_RELU>(y[v]);
            } else if (a.act == NFLOW_ACT_GELU_TANH) {
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = activate<ACT_GELU_TANH>(y[v]);
            }
            dense_put<T, STREAM, V>(static_cast<T*>(a.C) + m * a.ldc + n, y, left);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// Eight elements at p, of which the first `left` exist (the rest are 0).  At the
// end of a row eight loads at once, those past the last of the last: under
// conditions of their own each would wait for the one before it.
template <typename T>
__device__ __forceinline__ void dense_load(Raw8<T>& v, const T* p, int64_t left) {
    if (left >= 8) {
        v.load(p, 8);
        return;
    }
    const int n = static_cast<int>(left);
#pragma unroll
    for (int e = 0; e < 8; ++e) v.q[e] = T(0.0f);
    if (n <= 0) return;
    T x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[e < n ? e : n - 1];
#pragma unroll
    for (int e = 0; e < 8; ++e) v.q[e] = e < n ? x[e] : T(0.0f);
}

// ---- how a product is dealt out -------------------------------------------------------
// Workgroup i computes whole tiles i, i + groups, ... (`whole` of them), and where
// tiles are left, `rest` of them, their K steps are dealt out evenly: it takes
// steps [i, i + 1) rest ksteps / groups of those tiles one after another, which
// reach into at most two.  A part of a tile leaves its fp32 sums in a slot (two a
// workgroup, BM x BN each), and a second launch joins a tile's slots in the
// workgroups' order.
struct DenseSlots {
    float* part;        // 2 groups slots of BM x BN, then as many of BM: the sums of a's rows
    int groups;
};
struct DenseShare {
    int64_t tiles_m, tiles_n;
    int groups, whole, rest, ksteps;
    float* part;
    __host__ __device__ int64_t step_of(int i) const { return static_cast<int64_t>(i) * rest * ksteps / groups; }
};

// Calls f(tile, first step, end, slot or -1) for the work of this workgroup, all
// waves of it together at each call's start.  Neighbouring workgroups are on one
// XCD (gemm_tile_of_block).
template <typename F>
__device__ __forceinline__ void dense_each(const DenseShare& sh, F f) {
    int i = gemm_tile_of_block(blockIdx.x, sh.groups, 8);
    // Where every tile has as many workgroups, neighbours take the same steps of
    // different tiles: an XCD then reads a run of k of both operands once.
    if (sh.rest > 0 && sh.whole == 0 && sh.groups % sh.rest == 0) i = i % sh.rest * (sh.groups / sh.rest) + i / sh.rest;
    int64_t at = sh.rest ? sh.step_of(i) : 0;
    const int64_t end = sh.rest ? sh.step_of(i + 1) : 0;
    for (int n = 0; n < sh.whole || at < end; ++n) {
        int64_t tile = static_cast<int64_t>(n) * sh.groups + i;
        int k = 0, stop = sh.ksteps, slot = -1;
        if (n >= sh.whole) {
            const int64_t t = at / sh.ksteps;
            k = static_cast<int>(at - t * sh.ksteps);
            if (k + end - at < stop) stop = static_cast<int>(k + end - at);
            tile = static_cast<int64_t>(sh.whole) * sh.groups + t;
            if (k > 0 || stop < sh.ksteps) slot = 2 * i + n - sh.whole;
            at += stop - k;
        }
        if (n) __syncthreads();
        f(tile, k, stop, slot);
    }
}

// What becomes of a wave's sums: the results, or a slot's.
template <typename T, typename Tile>
__device__ __forceinline__ void dense_leave(const DenseArgs& a, const DenseSlots& sh, const v4f (&acc)[Tile::TI][Tile::TJ],
                                            float* strip, int64_t m0, int64_t n0, int slot, int wm, int wn) {
    const int i = 16 * Tile::TI * wm, j = 16 * Tile::TJ * wn;
    if (slot >= 0) {
        const DenseArgs p{nullptr, nullptr, 0, 0, Tile::BM, Tile::BN, 0, nullptr, nullptr, 0, NFLOW_ACT_NONE,
                          sh.part + static_cast<int64_t>(slot) * Tile::BM * Tile::BN, Tile::BN, nullptr, 0, nullptr};
        dense_store<float, Tile, false>(p, acc, strip, i, j);
    } else {
        dense_store<T, Tile, true>(a, acc, strip, m0 + i, n0 + j);
    }
}

// The sums of a's rows ride along in the tiles of the first columns: a product
// with ones for every row tile, the waves of a row of waves taking them in turn.
template <typename Tile>
struct DenseSums {
    static constexpr int N = (Tile::TI + Tile::WN - 1) / Tile::WN;
    v4f s[N];
    int mine;           // the wave's column of waves, or one that no row tile has
    __device__ __forceinline__ DenseSums(bool wanted, int wn) : mine(wanted ? wn : Tile::WN) {
#pragma unroll
        for (int n = 0; n < N; ++n) s[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    template <int P>
    __device__ __forceinline__ void add(int i, const v8bf (&a)[P]) {
        if (i % Tile::WN != mine) return;
        v8bf ones;
#pragma unroll
        for (int e = 0; e < 8; ++e) ones[e] = static_cast<bf16>(1.0f);
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
            s[i / Tile::WN] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, a[p], s[i / Tile::WN], 0, 0, 0);
    }
    __device__ __forceinline__ void leave(const DenseArgs& a, const DenseSlots& sh, int64_t m0, int slot, int wm) const {
        const int r = threadIdx.x & 63;
        if (mine == Tile::WN || r >= 16) return;
        float* to = slot >= 0 ? sh.part + 2 * static_cast<int64_t>(sh.groups) * Tile::BM * Tile::BN +
                                    static_cast<int64_t>(slot) * Tile::BM
                              : a.sums + m0;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = mine + n * Tile::WN, row = 16 * (Tile::TI * wm + i) + r;
            if (i < Tile::TI && (slot >= 0 || m0 + row < a.M)) to[row] = s[n][0];
        }
    }
};

// kJoinRows rows of a shared tile from row0 on: the sum of its slots, of
// workgroups i .. stop - 1, and the epilogue.  `late`: the tile is the second that
// workgroup i had a part of.  Bound by the slots' bytes, from the caches, or their
// latency: 128 slots of a tile of 64 x 64 13 us, where each waits for the last 40.
constexpr int kJoinRows = 8;
template <typename T, int BM, int BN>
__device__ __forceinline__ void dense_join(const DenseArgs& a, const DenseSlots& sl, const TilePos& pos, int row0, int i,
                                           int stop, bool late) {
    const int64_t m0 = pos.tm * BM + row0, n0 = pos.tn * BN;
    constexpr int Q = kJoinRows * BN / 4, TH = Q < 256 ? Q : 256, PER = Q / TH;   // groups of four values, threads, of each
    const bool sums = a.sums && pos.tn == 0 && threadIdx.x < kJoinRows;
    auto slot_of = [&](int w) { return 2 * static_cast<int64_t>(w) + (w == i && late ? 1 : 0); };
    v4f z[PER];
#pragma unroll
    for (int q = 0; q < PER; ++q) z[q] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (static_cast<int>(threadIdx.x) < TH) {
        // Many slots' loads at once, the last of them read again in place of those past it.
        int w = i;
        auto some = [&](auto many) {
            constexpr int B = decltype(many)::value;
            v4f v[B][PER];
#pragma unroll
            for (int n = 0; n < B; ++n) {
                const float* p = sl.part + slot_of(w + n < stop ? w + n : stop - 1) * BM * BN + row0 * BN;
#pragma unroll
                for (int q = 0; q < PER; ++q) v[n][q] = *reinterpret_cast<const v4f*>(p + 4 * (threadIdx.x + TH * q));
            }
#pragma unroll
            for (int n = 0; n < B; ++n)
#pragma unroll
                for (int q = 0; q < PER; ++q)
                    if (w + n < stop) z[q] += v[n][q];
            w += B;
        };
        while (w + 16 / PER <= stop) some(std::integral_constant<int, 16 / PER>{});
        while (w < stop) some(std::integral_constant<int, 4>{});
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int e = 4 * (threadIdx.x + TH * q);
            if (m0 + e / BN < a.M) dense_finish<T>(a, m0 + e / BN, n0 + e % BN, z[q]);
        }
    }
    if (!sums) return;
    float s = 0.0f;
#pragma unroll 16
    for (int w = i; w < stop; ++w)
        s += sl.part[(2 * static_cast<int64_t>(sl.groups) * BN + slot_of(w)) * BM + row0 + threadIdx.x];
    if (m0 + threadIdx.x < a.M) a.sums[m0 + threadIdx.x] = s;
}
// The first workgroup, of `groups` that `steps` are dealt out to, that begins at
// step `at` or past it.
__host__ __device__ inline int dense_from(int64_t at, int64_t steps, int groups) {
    return static_cast<int>((at * groups + steps - 1) / steps);
}

// A workgroup for kJoinRows rows of a tile of those that are left.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void k_dense_join(DenseArgs a, DenseShare sh) {
    const int t = blockIdx.x / (BM / kJoinRows);
    const int64_t first = static_cast<int64_t>(t) * sh.ksteps, last = first + sh.ksteps, all = static_cast<int64_t>(sh.rest) * sh.ksteps;
    int i = dense_from(first, all, sh.groups);
    const bool late = sh.step_of(i) > first;
    if (late) --i;                                                       // began in the tile before
    const int stop = dense_from(last, all, sh.groups);
    if (stop == i + 1) return;                                           // one workgroup's: stored
    dense_join<T, BM, BN>(a, DenseSlots{sh.part, sh.groups},
                          tile_pos(static_cast<int64_t>(sh.whole) * sh.groups + t, sh.tiles_m, sh.tiles_n, 4),
                          kJoinRows * (blockIdx.x % (BM / kJoinRows)), i, stop, late);
}

// ---- two products in one launch ------------------------------------------------------------
// dx and dW with all of their K steps dealt out evenly in one row, dx's tiles
// first: one launch and one join where each by itself would leave CUs idle at
// its end and more parts of tiles behind.
struct DensePair {
    DenseArgs a[2];
    int64_t tiles_m[2], tiles_n[2];
    int ksteps[2];
    int64_t first[2], steps;     // step at which each begins, and all of them
    int groups;
    float* part;
    __host__ __device__ int64_t step_of(int i) const { return i * steps / groups; }
    // The product, tile and first step of the tile that step `at` is in.
    __device__ __forceinline__ int64_t tile_of(int64_t at, int& which, int64_t& begin) const {
        which = at >= first[1] ? 1 : 0;
        const int64_t t = (at - first[which]) / ksteps[which];
        begin = first[which] + t * ksteps[which];
        return t;
    }
};

// Calls f(product, its tile, first step, end, slot or -1) for this workgroup's work.
template <typename F>
__device__ __forceinline__ void dense_each_pair(const DensePair& pr, F f) {
    const int i = gemm_tile_of_block(blockIdx.x, pr.groups, 8);
    const int64_t from = pr.step_of(i), end = pr.step_of(i + 1);
    for (int64_t at = from; at < end;) {
        int which;
        int64_t begin;
        const int64_t t = pr.tile_of(at, which, begin);
        const int ks = pr.ksteps[which], k = static_cast<int>(at - begin);
        const int stop = end - begin < ks ? static_cast<int>(end - begin) : ks;
        if (at > from) __syncthreads();
        f(which, t, k, stop, k == 0 && stop == ks ? -1 : 2 * i + (at > from ? 1 : 0));
        at = begin + stop;
    }
}

// The same for the tile that workgroup i begins within, if it is the first to.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void k_dense_join_pair(DensePair pr) {
    const int i = blockIdx.x / (BM / kJoinRows) + 1;
    const int64_t at = pr.step_of(i);
    int which;
    int64_t first;
    const int64_t t = pr.tile_of(at, which, first);
    const int64_t before = pr.step_of(i - 1);
    if (at == first || before > first) return;
    dense_join<T, BM, BN>(pr.a[which], DenseSlots{pr.part, pr.groups}, tile_pos(t, pr.tiles_m[which], pr.tiles_n[which], 4),
                          kJoinRows * (blockIdx.x % (BM / kJoinRows)), i - 1,
                          dense_from(first + pr.ksteps[which], pr.steps, pr.groups), before < first);
}

// Lets `kernel` have its tile's LDS, once on every device.
template <typename Tile, auto kernel>
void dense_lds() {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return;
    const uint64_t bit = uint64_t{1} << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return;
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, Tile::LDS);
    done.fetch_or(bit, std::memory_order_relaxed);
}

// dx and dW by `kernel`, and their join.
template <typename T, typename Tile, auto kernel>
void launch_dense_pair_tile(const DenseArgs& dx, const DenseArgs& dw, const DensePlan& p, float* part, hipStream_t st) {
    dense_lds<Tile, kernel>();
    DensePair pr{{dx, dw}, {}, {}, {}, {}, 0, p.groups, part};
    for (int j = 0; j < 2; ++j) {
        pr.tiles_m[j] = (pr.a[j].M + Tile::BM - 1) / Tile::BM;
        pr.tiles_n[j] = (pr.a[j].N + Tile::BN - 1) / Tile::BN;
        pr.ksteps[j] = static_cast<int>((pr.a[j].K + Tile::KB - 1) / Tile::KB);
        pr.first[j] = pr.steps;
        pr.steps += pr.tiles_m[j] * pr.tiles_n[j] * pr.ksteps[j];
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(p.groups)), dim3(Tile::THREADS), Tile::LDS, st, pr);
    hipLaunchKernelGGL((k_dense_join_pair<T, Tile::BM, Tile::BN>),
                       dim3(static_cast<unsigned>((p.groups - 1) * (Tile::BM / kJoinRows))), dim3(256), 0, st, pr);
}

// `kernel` over a product as the plan has it, and the join of what is shared.
template <typename T, typename Tile, auto kernel>
void launch_dense_tile(const DenseArgs& a, const DensePlan& p, float* part, hipStream_t st) {
    dense_lds<Tile, kernel>();
    const int64_t tm = (a.M + Tile::BM - 1) / Tile::BM, tn = (a.N + Tile::BN - 1) / Tile::BN, tiles = tm * tn;
    const int ks = static_cast<int>((a.K + Tile::KB - 1) / Tile::KB);
    DenseShare sh{tm, tn, static_cast<int>(tiles), 1, 0, ks, part};
    if (p.groups) {
        sh.groups = p.groups;
        sh.whole = static_cast<int>(tiles / p.groups);
        sh.rest = static_cast<int>(tiles % p.groups);
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(sh.groups)), dim3(Tile::THREADS), Tile::LDS, st, a, sh);
    if (sh.rest)
        hipLaunchKernelGGL((k_dense_join<T, Tile::BM, Tile::BN>),
                           dim3(static_cast<unsigned>(sh.rest * (Tile::BM / kJoinRows))), dim3(256), 0, st, a, sh);
}

}  // namespace nfq
