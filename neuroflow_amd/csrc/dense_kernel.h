// dense_kernel.h -- the tiled product of bf16 or fp32 operands on the matrix
// cores.
//
//   z[m][n] = sum_k a[m][k] b[n][k] + bias[n] + r[m][n],   C = act(z)
//
// bf16 operands take v_mfma_f32_16x16x32_bf16: products exact, sums fp32.  An
// fp32 operand is three bf16 planes, x = h + m + l: each plane is the rest
// rounded to bf16's 8 bits, so 24 bits are held exactly, and six products (h h, h
// m, m h, m m, h l, l h) leave out what is at most 2^-26 of the product: fp32
// accuracy at a sixth of the bf16 rate, where the fp32 instruction has a
// sixteenth.
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

template <typename T>
constexpr int dense_planes() { return std::is_same_v<T, float> ? 3 : 1; }

// Eight fp32 values as bf16 planes.  A value that would round to infinity keeps
// a finite first plane; the planes of an infinity or a NaN are NaN past the first.
__device__ __forceinline__ void dense_split(const float (&v)[8], v8bf (&p)[3]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float x = v[e];
        const float top = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
        const bf16 h = fabsf(x) < 0x1.ffp127f ? static_cast<bf16>(x) : static_cast<bf16>(top);
        const float r = x - static_cast<float>(h);
        const bf16 m = static_cast<bf16>(r);
        p[0][e] = h;
        p[1][e] = m;
        p[2][e] = static_cast<bf16>(r - static_cast<float>(m));
    }
}

// Tiles of BM x BN, WM x WN waves of TI x TJ 16 x 16 tiles each; a stage is KB
// values of k of every row, NS stages.
template <typename T, int WM_, int WN_, int TI_, int TJ_, int NS_, int OCC_ = 2>
struct DenseTile {
    static constexpr int WM = WM_, WN = WN_, TI = TI_, TJ = TJ_, NS = NS_, OCC = OCC_;
    static constexpr int P = dense_planes<T>();
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int BM = 16 * TI * WM, BN = 16 * TJ * WN;
    static constexpr int KB = std::is_same_v<T, float> ? 32 : 64;
    static constexpr int PLANE_A = BM * KB * 2, PLANE_B = BN * KB * 2;       // bytes
    static constexpr int STAGE = P * (PLANE_A + PLANE_B);
    static constexpr int STRIP_ROW = 16 * TJ + 4, STRIP = 16 * STRIP_ROW;   // floats of a wave's 16 rows on their way out
    static constexpr int LDS = NS * STAGE > WAVES * STRIP * 4 ? NS * STAGE : WAVES * STRIP * 4;
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

// An operand's share of a stage by way of registers: CH groups of 8 values a thread.
template <typename T, bool ACROSS, int R, int KB, int THREADS>
struct DenseStage {
    static constexpr int CH = R * KB / 8 / THREADS;
    static_assert(R * KB / 8 % THREADS == 0, "groups spread evenly");
    static constexpr int PER = (ACROSS ? R : KB) / 8;              // groups of a row in memory
    Raw8<T> v[CH];
    // Rows row0 .. of `rows`, k's k0 .. of K.
    __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int64_t K) {
        const bool inside = row0 + R <= rows && k0 + KB <= K;
#pragma unroll
        for (int q = 0; q < CH; ++q) {
            const int id = threadIdx.x + THREADS * q, i = id / PER, c = 8 * (id % PER);
            const int64_t major = (ACROSS ? k0 : row0) + i, minor = (ACROSS ? row0 : k0) + c;
            const T* p = base + major * ld + minor;
            if (inside) v[q].load(p, 8);
            else v[q].load(p, major < (ACROSS ? K : rows) ? (ACROSS ? rows : K) - minor : 0);
        }
    }
    __device__ __forceinline__ void store(uint8_t* planes) const {
#pragma unroll
        for (int q = 0; q < CH; ++q) {
            const int id = threadIdx.x + THREADS * q;
            uint8_t* to = planes + dense_place<ACROSS, R, KB>(id / PER, id % PER);
            if constexpr (std::is_same_v<T, float>) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = v[q][e];
                v8bf p[3];
                dense_split(x, p);
#pragma unroll
                for (int s = 0; s < 3; ++s) *reinterpret_cast<v8bf*>(to + s * R * KB * 2) = p[s];
            } else {
                v8bf x;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = v[q].q[e];
                *reinterpret_cast<v8bf*>(to) = x;
            }
        }
    }
};

// Four outputs of a row from column n on: bias, residual, activation, one rounding.
template <typename T>
__device__ __forceinline__ void dense_finish(const DenseArgs& a, int64_t m, int64_t n, const v4f& s) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        if (n + v >= a.N) return;
        float z = s[v] + (a.bias ? a.bias[n + v] : 0.0f);
        if (a.R) z += to_f32(static_cast<const T*>(a.R)[m * a.ldr + n + v]);
        if (a.Z) static_cast<T*>(a.Z)[m * a.ldz + n + v] = from_f32<T>(z);
        static_cast<T*>(a.C)[m * a.ldc + n + v] = from_f32<T>(activate_rt(z, a.act));
    }
}

// V values at p, together where the row allows it.
template <typename T, int V>
__device__ __forceinline__ void dense_put(T* p, const float (&y)[V], bool vec, int64_t left) {
    if (vec) {
        typedef T vt __attribute__((ext_vector_type(V)));
        vt o;
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = from_f32<T>(y[v]);
        __builtin_nontemporal_store(o, reinterpret_cast<vt*>(p));
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < left) p[v] = from_f32<T>(y[v]);
    }
}

// A wave's TI x TJ tiles of sums to rows m0 .., columns n0 .. of C, through its
// strip of LDS, so that loads and stores are whole lines.
template <typename T, typename Tile>
__device__ __forceinline__ void dense_store(const DenseArgs& a, const v4f (&acc)[Tile::TI][Tile::TJ], float* strip,
                                            int64_t m0, int64_t n0) {
    constexpr int V = 16 / sizeof(T), LPR = 16 * Tile::TJ / V, RPI = 64 / LPR;   // values a lane, lanes a row, rows a store
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int row = lane / LPR, col = V * (lane % LPR);
    const int64_t n = n0 + col, left = a.N - n;
    auto whole = [&](const void* p, int64_t ld) { return left >= V && ld % V == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const bool vec = whole(a.C, a.ldc), vecz = whole(a.Z, a.ldz), vecr = whole(a.R, a.ldr);
    float b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) b[v] = a.bias && v < left ? a.bias[n + v] : 0.0f;
#pragma unroll
    for (int i = 0; i < Tile::TI; ++i) {
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
            if (m >= a.M) continue;
            if (a.R) {
                const T* rr = static_cast<const T*>(a.R) + m * a.ldr + n;
                if (vecr) {
                    typedef T vt __attribute__((ext_vector_type(V)));
                    const vt x = *reinterpret_cast<const vt*>(rr);
#pragma unroll
                    for (int v = 0; v < V; ++v) y[v] += to_f32(x[v]);
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) y[v] += v < left ? to_f32(rr[v]) : 0.0f;
                }
            }
            if (a.Z) dense_put<T, V>(static_cast<T*>(a.Z) + m * a.ldz + n, y, vecz, left);
            if (a.act == NFLOW_ACT_RELU) {
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = activate<ACT_RELU>(y[v]);
            } else if (a.act == NFLOW_ACT_GELU_TANH) {
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = activate<ACT_GELU_TANH>(y[v]);
            }
            dense_put<T, V>(static_cast<T*>(a.C) + m * a.ldc + n, y, vec, left);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

struct DenseShare {
    int64_t tiles_m, tiles_n;
    int splits, per;    // runs of `per` stages of K
    float* part;        // (splits, M, N) sums, where splits > 1
    int blocks;
};

// One stage's products: every 32 k's, the planes' products of the least first.
template <typename T, bool AX, bool BX, typename Tile>
__device__ __forceinline__ void dense_step(const uint8_t* st, v4f (&acc)[Tile::TI][Tile::TJ], int arow, int brow) {
    constexpr int P = Tile::P, TI = Tile::TI, TJ = Tile::TJ, KB = Tile::KB;
    const uint8_t* sb = st + P * Tile::PLANE_A;
#pragma unroll
    for (int k = 0; k < KB; k += 32) {
        v8bf bf[P][TJ];
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < TJ; ++j)
                bf[p][j] = dense_fragment<BX, Tile::BN, KB>(sb + p * Tile::PLANE_B, brow + 16 * j, k);
#pragma unroll
        for (int i = 0; i < TI; ++i) {
            v8bf af[P];
#pragma unroll
            for (int p = 0; p < P; ++p) af[p] = dense_fragment<AX, Tile::BM, KB>(st + p * Tile::PLANE_A, arow + 16 * i, k);
            if constexpr (P == 1) {
#pragma unroll
                for (int j = 0; j < TJ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[0][j], af[0], acc[i][j], 0, 0, 0);
            } else {
                constexpr int pa[6] = {0, 2, 1, 0, 1, 0}, pb[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
                for (int q = 0; q < 6; ++q)
#pragma unroll
                    for (int j = 0; j < TJ; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[pb[q]][j], af[pa[q]], acc[i][j], 0, 0, 0);
            }
        }
    }
}

template <typename T, bool AX, bool BX, typename Tile>
__global__ __launch_bounds__(Tile::THREADS, Tile::OCC) void k_dense(DenseArgs a, DenseShare sh) {
    constexpr int TI = Tile::TI, TJ = Tile::TJ, KB = Tile::KB;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wid / Tile::WN, wn = wid % Tile::WN;
    const int64_t t = gemm_tile_of_block(blockIdx.x, sh.blocks, 8);
    const int split = sh.splits > 1 ? static_cast<int>(t % sh.splits) : 0;
    const TilePos pos = tile_pos(sh.splits > 1 ? t / sh.splits : t, sh.tiles_m, sh.tiles_n, 4);
    const int64_t m0 = pos.tm * Tile::BM, n0 = pos.tn * Tile::BN;
    const int ks = static_cast<int>((a.K + KB - 1) / KB);
    const int k0 = split * sh.per, k1 = k0 + sh.per < ks ? k0 + sh.per : ks;

    v4f acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    DenseStage<T, AX, Tile::BM, KB, Tile::THREADS> ra;
    DenseStage<T, BX, Tile::BN, KB, Tile::THREADS> rb;
    auto load = [&](int k) {
        ra.load(static_cast<const T*>(a.A), a.lda, m0, a.M, static_cast<int64_t>(k) * KB, a.K);
        rb.load(static_cast<const T*>(a.B), a.ldb, n0, a.N, static_cast<int64_t>(k) * KB, a.K);
    };
    if (k0 < k1) load(k0);
    for (int k = k0; k < k1; ++k) {
        __syncthreads();                             // the stage's last readers are done
        ra.store(lds);
        rb.store(lds + Tile::P * Tile::PLANE_A);
        __syncthreads();
        if (k + 1 < k1) load(k + 1);
        dense_step<T, AX, BX, Tile>(lds, acc, 16 * TI * wm, 16 * TJ * wn);
    }
    __syncthreads();
    float* strip = reinterpret_cast<float*>(lds) + wid * Tile::STRIP;
    const int64_t mw = m0 + 16 * TI * wm, nw = n0 + 16 * TJ * wn;
    if (sh.splits > 1) {
        const DenseArgs p{nullptr, nullptr, 0, 0, a.M, a.N, a.K, nullptr, nullptr, 0, NFLOW_ACT_NONE,
                          sh.part + split * a.M * a.N, a.N, nullptr, 0};
        dense_store<float, Tile>(p, acc, strip, mw, nw);
    } else {
        dense_store<T, Tile>(a, acc, strip, mw, nw);
    }
}

// Sum of the splits' partial results, in their order, and the epilogue.
template <typename T>
__global__ __launch_bounds__(256) void k_dense_join(DenseArgs a, const float* __restrict__ part, int splits) {
    const int64_t n4 = (a.N + 3) / 4, total = a.M * n4;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t m = i / n4, n = (i - m * n4) * 4;
        v4f z{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < splits; ++s) {
            const float* p = part + (s * a.M + m) * a.N + n;
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (n + v < a.N) z[v] += p[v];
        }
        dense_finish<T>(a, m, n, z);
    }
}

// `kernel` over the tiles of the product and its splits, and their join.
template <typename T, typename Tile, auto kernel>
void launch_dense_tile(const DenseArgs& a, int splits, float* part, hipStream_t st) {
    static const hipError_t once = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, Tile::LDS);
    (void)once;
    const int64_t tm = (a.M + Tile::BM - 1) / Tile::BM, tn = (a.N + Tile::BN - 1) / Tile::BN;
    const int ks = static_cast<int>((a.K + Tile::KB - 1) / Tile::KB);
    const DenseShare sh{tm, tn, splits, (ks + splits - 1) / splits, part, static_cast<int>(tm * tn * splits)};
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(sh.blocks)), dim3(Tile::THREADS), Tile::LDS, st, a, sh);
    if (splits > 1)
        hipLaunchKernelGGL((k_dense_join<T>), dim3(grid_for(a.M * ((a.N + 3) / 4), 256, 8)), dim3(256), 0, st, a, part,
                           splits);
}

}  // namespace nfq
