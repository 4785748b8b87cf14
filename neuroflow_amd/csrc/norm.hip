// norm.hip -- layer norm, forward (to the activation's type or straight to
// 128-block FP8) and backward (include/nflow_block.h).
#include <type_traits>

#include "norm_dev.h"

namespace nfq {
namespace {

// The result from a deviation from the mean.
__device__ __forceinline__ float norm_value(float d, float rstd, float w, float b) {
    return __builtin_fmaf(d * rstd, w, b);
}

struct NormArgs {
    const void* x;
    int64_t M, D, ldx;
    const float* weight;
    const float* bias;
    float eps;
    void* y;
    int64_t ldy;
    uint8_t* codes;
    float* scales;
    float* mean;
    float* rstd;
};

// ---- rows in registers --------------------------------------------------------
// L threads hold a row of at most 8 L NV values: thread t the eight values from
// column 8 (t + L j) on, j < NV.  One read of x: the sum, the squares about the
// mean (no cancellation however far the mean is from 0) and the result are
// formed from registers, while the next row's loads are in flight.  weight and
// bias stay in registers over all of a thread's rows.  HBM bound: 32768 x 256
// fp32 13.4 us, 5.0 TB/s.
template <typename T, bool FP8, int L, int NV>
__global__ __launch_bounds__(row_threads<L>()) void k_norm(NormArgs a, int64_t per) {
    constexpr int G = row_threads<L>() / L;              // rows a workgroup holds
    __shared__ float part[2][L <= 64 ? 1 : L / 64];
    const int t = threadIdx.x % L;
    const int D = static_cast<int>(a.D);
    const float inv_d = 1.0f / static_cast<float>(D);
    const bool whole = D == 8 * L * NV;                    // every thread's every vector is
    float w[NV][8], b[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = 8 * (t + L * j);
        load_param(a.weight, c, D, 1.0f, w[j]);
        load_param(a.bias, c, D, 0.0f, b[j]);
    }
    Raw8<T> next[NV];
    auto fetch = [&](int64_t m) {
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (t + L * j);
            next[j].load(x + c, m < a.M ? D - c : 0);
        }
    };
    // A workgroup takes a run of rows, G at a time: neighbouring rows' scales
    // (and statistics) then meet in one L2 on their way out.
    int64_t m = blockIdx.x * per + threadIdx.x / L;
    const int64_t end = blockIdx.x * per + per < a.M ? blockIdx.x * per + per : a.M;
    fetch(m < end ? m : a.M);
    for (int64_t i = 0; i < per; i += G, m += G) {
        // Beyond a partial last round the lanes of absent rows work on zeros and
        // store nothing: the workgroup's barriers and the DPP reductions stay whole.
        const bool on = m < end;
        float v[NV][8], vs[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = next[j][e];
            vs[j] = pair_sum<8>(v[j]);
        }
        const float s = pair_sum<NV>(vs);
        fetch(i + G < per && m + G < end ? m + G : a.M);
        const float mean = row_sum<L>(s, part, 0) * inv_d;
        float q = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = D - 8 * (t + L * j);          // only a row's last vector is partial
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] -= mean;
            if (!whole && left < 8) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = e < left ? v[j][e] : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) q = __builtin_fmaf(v[j][e], v[j][e], q);
        }
        const float rstd = norm_rstd(__builtin_fmaf(row_sum<L>(q, part, 1), inv_d, a.eps));
        if (on && t == 0) {
            if (a.mean) a.mean[m] = mean;
            if (a.rstd) a.rstd[m] = rstd;
        }
        float y[NV][8];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) y[j][e] = norm_value(v[j][e], rstd, w[j][e], b[j][e]);
        if constexpr (!FP8) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = 8 * (t + L * j);
                store8(static_cast<T*>(a.y) + m * a.ldy + c, on ? D - c : 0, y[j]);
            }
        } else {
            // 16 threads hold a block of 128; columns past D count as 0.  Every
            // lane inverts its own block's scale: shared among the lanes, as the
            // quantise has it, the inverses lengthen a row's chain of reductions.
            // At 16384 x 4096 bf16: 47.4 us, 4.3 TB/s, the VALU's issue as busy as
            // HBM (50.2 us with divisions and the cap at every value).
            const int kb = static_cast<int>(blk_count(D));
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = 8 * (t + L * j), left = D - c;
                if (!whole && left < 8) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[j][e] = e < left ? y[j][e] : 0.0f;
                }
                float amax = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = amax_of(amax, y[j][e]);
                const float sc = blk_scale(max16(amax));
                const v2u q8 = blk_codes8(y[j], blk_inverse(sc));
                if (on && c / kBlk < kb) {
                    *reinterpret_cast<v2u*>(a.codes + m * kb * kBlk + c) = q8;
                    if (t % 16 == 0) a.scales[c / kBlk * a.M + m] = sc;
                }
            }
        }
    }
}

// ---- rows of any length ---------------------------------------------------------
// Past the register kernels' widths: one workgroup per row, three passes over
// it (the second and third from the caches).
template <typename T, bool FP8>
__global__ __launch_bounds__(kNormThreads) void k_norm_rows(NormArgs a) {
    __shared__ float part[kNormThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
        float s = 0.0f;
        for (int64_t c = tid; c < a.D; c += kNormThreads) s += to_f32(x[c]);
        const float mean = block_sum(s, part) / static_cast<float>(a.D);
        float q = 0.0f;
        for (int64_t c = tid; c < a.D; c += kNormThreads) {
            const float d = to_f32(x[c]) - mean;
            q = __builtin_fmaf(d, d, q);
        }
        const float rstd = 1.0f / sqrtf(block_sum(q, part) / static_cast<float>(a.D) + a.eps);
        if (tid == 0) {
            if (a.mean) a.mean[m] = mean;
            if (a.rstd) a.rstd[m] = rstd;
        }
        auto value = [&](int64_t c) {
            return norm_value(to_f32(x[c]) - mean, rstd, a.weight ? a.weight[c] : 1.0f, a.bias ? a.bias[c] : 0.0f);
        };
        if constexpr (!FP8) {
            T* y = static_cast<T*>(a.y) + m * a.ldy;
            for (int64_t c = tid; c < a.D; c += kNormThreads) y[c] = from_f32<T>(value(c));
        } else {
            const int64_t kb = blk_count(a.D);
            for (int64_t b = wave; b < kb; b += kNormThreads / 64) {
                const int64_t c = b * kBlk + 2 * lane;
                const float v0 = c < a.D ? value(c) : 0.0f, v1 = c + 1 < a.D ? value(c + 1) : 0.0f;
                const float sc = blk_scale(wave_max(amax_of(amax_of(0.0f, v0), v1)));
                const float inv = blk_inverse(sc);
                const uint32_t w = fp8_quant(v0, inv) | fp8_quant(v1, inv) << 8;
                *reinterpret_cast<uint16_t*>(a.codes + m * kb * kBlk + c) =
                    static_cast<uint16_t>(c + 1 < a.D ? w : (c < a.D ? w & 0xFFu : 0u));
                if (lane == 0) a.scales[b * a.M + m] = sc;
            }
        }
    }
}

struct NormGradArgs {
    const void* dy;
    const void* x;
    int64_t M, D, lddy, ldx;
    const float* weight;
    const float* mean;
    const float* rstd;
    void* dx;
    int64_t lddx;
    float* part;        // (workgroups, 2, D) partial dweight and dbias, or null
    int64_t rows_per;   // rows of a workgroup's share (k_norm_grad_params)
};

// ---- backward, rows in registers ---------------------------------------------------
// The layout of k_norm.  dx needs two sums over the row, of g and g h; the
// parameters' gradients are sums over rows of dy h and dy, which every thread
// keeps for its columns over all of its rows, and a workgroup joins over its G
// rows in LDS at the end: one partial row per workgroup, so the partials are a
// small part of the traffic (256 of them against M rows).  1024 threads: G =
// 1024 / L rows at once.  x and dy are read once.  HBM bound: 16384 x 4096 bf16
// 78.4 us with the join below, 5.1 TB/s.
template <typename T, int L, int NV, int TH, bool AHEAD>
__global__ __launch_bounds__(TH) void k_norm_grad(NormGradArgs a) {
    constexpr int G = TH / L, W = TH / 64;
    __shared__ float2 part[2][W];
    constexpr int SLOTS = L == 16 ? W : G;               // sums a column has after the waves' own
    __shared__ __attribute__((aligned(16))) float join[SLOTS > 1 ? SLOTS * 8 * L : 8];
    const int t = threadIdx.x % L, grp = threadIdx.x / L;
    const int D = static_cast<int>(a.D);
    const float inv_d = 1.0f / static_cast<float>(D);
    float w[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        load_param(a.weight, 8 * (t + L * j), D, 1.0f, w[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[j][e] = db[j][e] = 0.0f;
    }
    Raw8<T> nx[NV], ny[NV];
    float nmean = 0.0f, nrstd = 0.0f;
    auto fetch = [&](int64_t m) {
        const bool on = m < a.M;
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
        const T* dy = static_cast<const T*>(a.dy) + m * a.lddy;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (t + L * j);
            nx[j].load(x + c, on ? D - c : 0);
            ny[j].load(dy + c, on ? D - c : 0);
        }
        nmean = on ? a.mean[m] : 0.0f;
        nrstd = on ? a.rstd[m] : 0.0f;
    };
    // Row i of group grp: neighbouring rows lie in different workgroups, so a
    // few rows already spread over the chip.  Every group of a workgroup runs
    // the same number of rounds; one past the last row works on zeros.
    const int64_t grid = gridDim.x, rounds = (a.M + grid * G - 1) / (grid * G);
    auto row = [&](int64_t i) { return (i * G + grp) * grid + blockIdx.x; };
    if (AHEAD) fetch(row(0));
    for (int64_t i = 0; i < rounds; ++i) {
        const int64_t m = row(i);
        if (!AHEAD) fetch(m);
        float h[NV][8], g[NV][8], s1 = 0.0f, s2 = 0.0f;
        const float rstd = nrstd;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[j][e] = (nx[j][e] - nmean) * rstd;
                const float y = ny[j][e];
                dw[j][e] = __builtin_fmaf(y, h[j][e], dw[j][e]);
                db[j][e] += y;
                g[j][e] = y * w[j][e];                 // 0 past column D, as y is
                s1 += g[j][e];
                s2 = __builtin_fmaf(g[j][e], h[j][e], s2);
            }
        if (AHEAD) fetch(row(i + 1));
        if constexpr (L <= 64) {
            s1 = lanes_reduce<L, SumOp>(s1);
            s2 = lanes_reduce<L, SumOp>(s2);
        } else {
            s1 = wave_sum(s1);
            s2 = wave_sum(s2);
            if ((threadIdx.x & 63) == 0) part[i & 1][threadIdx.x >> 6] = make_float2(s1, s2);
            __syncthreads();
            s1 = s2 = 0.0f;
#pragma unroll
            for (int k = 0; k < L / 64; ++k) {
                const float2 p = part[i & 1][grp * (L / 64) + k];
                s1 += p.x;
                s2 += p.y;
            }
        }
        const float c1 = s1 * inv_d, c2 = s2 * inv_d;
        if (m < a.M) {
            T* dx = static_cast<T*>(a.dx) + m * a.lddx;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = 8 * (t + L * j);
                float o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = rstd * (g[j][e] - __builtin_fmaf(h[j][e], c2, c1));
                store8(dx + c, D - c, o);
            }
        }
    }
    if (!a.part) return;
    // One vector of columns at a time: a wave's four rows by the permlane swaps
    // (L = 16), then the groups' sums to LDS and a thread per column.
    float* out = a.part + blockIdx.x * 2 * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float s[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s[e] = k ? db[j][e] : dw[j][e];
                if constexpr (L == 16) s[e] = rows_sum(s[e]);
            }
            const int c = 8 * L * j;
            if constexpr (SLOTS == 1) {
                store8(out + k * a.D + c + 8 * t, D - c - 8 * t, s);
            } else {
                __syncthreads();
                const int slot = L == 16 ? threadIdx.x >> 6 : grp;
                if (L != 16 || (threadIdx.x & 63) < 16) {
                    *reinterpret_cast<v4f*>(join + slot * 8 * L + 8 * t) = v4f{s[0], s[1], s[2], s[3]};
                    *reinterpret_cast<v4f*>(join + slot * 8 * L + 8 * t + 4) = v4f{s[4], s[5], s[6], s[7]};
                }
                __syncthreads();
                for (int u = threadIdx.x; u < 8 * L && c + u < D; u += TH) {
                    float z = join[u];
#pragma unroll
                    for (int q = 1; q < SLOTS; ++q) z += join[q * 8 * L + u];
                    out[k * a.D + c + u] = z;
                }
            }
        }
}

// ---- backward, rows of any length ---------------------------------------------------
// Past the register kernel's widths: dx a workgroup per row in two passes, the
// parameters' partial sums a thread per column in a kernel of their own.
// dx, one block per row.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void k_norm_grad_rows(NormGradArgs a) {
    __shared__ float part[kNormThreads / 64];
    const int tid = threadIdx.x;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
        const T* dy = static_cast<const T*>(a.dy) + m * a.lddy;
        T* dx = static_cast<T*>(a.dx) + m * a.lddx;
        const float mean = a.mean[m], rstd = a.rstd[m];
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t c = tid; c < a.D; c += kNormThreads) {
            const float g = to_f32(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            s1 += g;
            s2 += g * ((to_f32(x[c]) - mean) * rstd);
        }
        const float c1 = block_sum(s1, part) / static_cast<float>(a.D);
        const float c2 = block_sum(s2, part) / static_cast<float>(a.D);
        for (int64_t c = tid; c < a.D; c += kNormThreads) {
            const float g = to_f32(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            const float h = (to_f32(x[c]) - mean) * rstd;
            dx[c] = from_f32<T>(rstd * (g - c1 - h * c2));
        }
    }
}

// Partial sums of dy * h and dy over a block's rows, a thread per column.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void k_norm_grad_params(NormGradArgs a) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x;
    if (c >= a.D) return;
    const int64_t m0 = blockIdx.y * a.rows_per, m1 = m0 + a.rows_per < a.M ? m0 + a.rows_per : a.M;
    float dw = 0.0f, db = 0.0f;
    for (int64_t m = m0; m < m1; ++m) {
        const float g = to_f32(static_cast<const T*>(a.dy)[m * a.lddy + c]);
        dw += g * ((to_f32(static_cast<const T*>(a.x)[m * a.ldx + c]) - a.mean[m]) * a.rstd[m]);
        db += g;
    }
    a.part[blockIdx.y * 2 * a.D + c] = dw;
    a.part[(blockIdx.y * 2 + 1) * a.D + c] = db;
}

// The partial sums' layout is (workgroups, 2 D): dweight's D columns, dbias's.
// A launch and a few latencies: 4 to 5 us.
__global__ __launch_bounds__(1024) void k_norm_grad_join(const float* __restrict__ part, int64_t P, int64_t D,
                                                         float* __restrict__ dweight, float* __restrict__ dbias) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    float v = 0.0f;
    if (n < 2 * D) {
#pragma unroll 8
        for (int64_t p = wave; p < P; p += 16) v += part[p * 2 * D + n];
    }
    s[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && n < 2 * D) {
        float z = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) z += s[k][lane];
        float* out = n < D ? dweight : dbias;
        if (out) out[n < D ? n : n - D] = z;
    }
}

// Workgroups (and partial rows) of the backward pass.
int64_t grad_blocks(int64_t M) { return std::min<int64_t>(M, num_cus()); }

size_t grad_space(int64_t M, int64_t D) {
    return static_cast<size_t>(grad_blocks(M)) * 2 * static_cast<size_t>(D) * sizeof(float);
}

template <typename T, bool FP8, int L, int NV>
void launch_norm(const NormArgs& a, hipStream_t st) {
    constexpr int threads = row_threads<L>(), G = threads / L;
    static const int64_t most = resident(k_norm<T, FP8, L, NV>, threads);
    const int64_t groups = (a.M + G - 1) / G, per = (groups + most - 1) / most * G;
    hipLaunchKernelGGL((k_norm<T, FP8, L, NV>), dim3(static_cast<unsigned>((a.M + per - 1) / per)), dim3(threads), 0, st,
                       a, per);
}

// The fewest threads that hold a row in 8 NV values each: fewer threads a row
// means more rows at once and shorter reductions.
template <typename T, bool FP8>
void launch_norm_rows(const NormArgs& a, hipStream_t st) {
    if (a.D <= 128) launch_norm<T, FP8, 16, 1>(a, st);
    else if (a.D <= 256) launch_norm<T, FP8, 16, 2>(a, st);
    else if (a.D <= 512) launch_norm<T, FP8, 64, 1>(a, st);
    else if (a.D <= 1024) launch_norm<T, FP8, 64, 2>(a, st);
    else if (a.D <= 2048) launch_norm<T, FP8, 64, 4>(a, st);
    else if (a.D <= 4096) launch_norm<T, FP8, 256, 2>(a, st);
    else if (a.D <= 8192) launch_norm<T, FP8, 256, 4>(a, st);
    else if (a.D <= kNormRegMax) launch_norm<T, FP8, 1024, 2>(a, st);
    else hipLaunchKernelGGL((k_norm_rows<T, FP8>), dim3(row_grid(a.M)), dim3(kNormThreads), 0, st, a);
}

// 1024 threads (16 waves a CU) with the next row's loads ahead while a thread
// holds 8 columns; at 16 columns without them, which fits 128 registers: 81.7
// us at 16384 x 4096 bf16 against 89.8 with half the threads and loads ahead.
// fp32 at 256 threads a row does not fit and takes that form.
template <typename T>
void launch_norm_grad(const NormGradArgs& a, unsigned nb, hipStream_t st) {
    auto go = [&](auto k, int threads) { hipLaunchKernelGGL(k, dim3(nb), dim3(threads), 0, st, a); };
    if (a.D <= 128) go(k_norm_grad<T, 16, 1, 1024, true>, 1024);
    else if (a.D <= 256) go(k_norm_grad<T, 16, 2, 1024, false>, 1024);
    else if (a.D <= 512) go(k_norm_grad<T, 64, 1, 1024, true>, 1024);
    else if (a.D <= 1024) go(k_norm_grad<T, 64, 2, 1024, false>, 1024);
    else if (a.D <= 2048) go(k_norm_grad<T, 256, 1, 1024, true>, 1024);
    else if (a.D <= 4096 && std::is_same_v<T, float>) go(k_norm_grad<float, 256, 2, 512, true>, 512);
    else if (a.D <= 4096) go(k_norm_grad<bf16, 256, 2, 1024, false>, 1024);
    else if (a.D <= 8192) go(k_norm_grad<T, 1024, 1, 1024, true>, 1024);
    else if (a.D <= kNormRegMax) go(k_norm_grad<T, 1024, 2, 1024, false>, 1024);
    else {
        if (a.part) {
            const unsigned gc = static_cast<unsigned>((a.D + kNormThreads - 1) / kNormThreads);
            hipLaunchKernelGGL((k_norm_grad_params<T>), dim3(gc, nb), dim3(kNormThreads), 0, st, a);
        }
        hipLaunchKernelGGL((k_norm_grad_rows<T>), dim3(row_grid(a.M)), dim3(kNormThreads), 0, st, a);
    }
}

int check_norm(const char* what, const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, float eps) {
    if (!dtype_ok(dtype)) return bad_arg(what, "unknown dtype");
    if (M < 0 || D <= 0) return bad_arg(what, "bad dims");
    if (ldx < D) return bad_arg(what, "row stride smaller than a row");
    if (!(eps >= 0.0f)) return bad_arg(what, "eps must not be negative or NaN");
    if (M > 0 && !x) return bad_arg(what, "null x");
    return NFLOW_OK;
}

template <bool FP8>
int norm_forward(const char* what, const NormArgs& a, int dtype, void* stream) {
    hipStream_t st = as_stream(stream);
    if (dtype == NFLOW_DTYPE_BF16) launch_norm_rows<bf16, FP8>(a, st);
    else launch_norm_rows<float, FP8>(a, st);
    return launch_status(what);
}

}  // namespace
}  // namespace nfq

using namespace nfq;

extern "C" {

int nflow_layer_norm_forward(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const float* weight,
                             const float* bias, float eps, void* y, int64_t ldy, float* mean, float* rstd,
                             void* stream) {
    clear_error();
    const char* what = "layer_norm_forward";
    if (int rc = check_norm(what, x, dtype, M, D, ldx, eps)) return rc;
    if (ldy < D) return bad_arg(what, "row stride smaller than a row");
    if (M == 0) return NFLOW_OK;
    if (!y) return bad_arg(what, "null y");
    if (rows_clash(x, ldx, y, ldy, M, D, dtype_size(dtype))) return bad_arg(what, kOverlap);
    return norm_forward<false>(what, NormArgs{x, M, D, ldx, weight, bias, eps, y, ldy, nullptr, nullptr, mean, rstd},
                               dtype, stream);
}

int nflow_layer_norm_fp8_block(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const float* weight,
                               const float* bias, float eps, uint8_t* codes, float* scales, float* mean,
                               float* rstd, void* stream) {
    clear_error();
    const char* what = "layer_norm_fp8_block";
    if (int rc = check_norm(what, x, dtype, M, D, ldx, eps)) return rc;
    if (M == 0) return NFLOW_OK;
    if (!codes || !scales) return bad_arg(what, "null codes or scales");
    if (!aligned(codes, 16)) return bad_arg(what, "codes must be 16-byte aligned");
    return norm_forward<true>(what, NormArgs{x, M, D, ldx, weight, bias, eps, nullptr, 0, codes, scales, mean, rstd},
                              dtype, stream);
}

int nflow_layer_norm_backward_workspace(int64_t M, int64_t D, size_t* bytes) {
    clear_error();
    if (!bytes) return bad_arg("layer_norm_backward_workspace", "null output");
    *bytes = 0;
    if (M < 0 || D <= 0) return bad_arg("layer_norm_backward_workspace", "bad dims");
    *bytes = grad_space(M, D);
    return NFLOW_OK;
}

int nflow_layer_norm_backward(const void* dy, const void* x, int dtype, int64_t M, int64_t D, int64_t lddy,
                              int64_t ldx, const float* weight, const float* mean, const float* rstd, void* dx,
                              int64_t lddx, float* dweight, float* dbias, void* workspace, size_t workspace_bytes,
                              void* stream) {
    clear_error();
    const char* what = "layer_norm_backward";
    if (int rc = check_norm(what, x, dtype, M, D, ldx, 0.0f)) return rc;
    if (lddy < D || lddx < D) return bad_arg(what, "row stride smaller than a row");
    if (M > 0 && (!dy || !mean || !rstd || !dx)) return bad_arg(what, "null dy, mean, rstd or dx");
    if (rows_clash(dy, lddy, dx, lddx, M, D, dtype_size(dtype)) || rows_clash(x, ldx, dx, lddx, M, D, dtype_size(dtype)))
        return bad_arg(what, kOverlap);
    if (int rc = check_workspace(what, workspace, workspace_bytes, grad_space(M, D))) return rc;
    hipStream_t st = as_stream(stream);
    const int64_t nb = grad_blocks(M);
    const bool params = dweight || dbias;
    if (M == 0 && !params) return NFLOW_OK;
    const NormGradArgs a{dy, x, M, D, lddy, ldx, weight, mean, rstd, dx, lddx,
                         params ? static_cast<float*>(workspace) : nullptr, nb ? (M + nb - 1) / nb : 0};
    if (M > 0) {
        if (dtype == NFLOW_DTYPE_BF16) launch_norm_grad<bf16>(a, static_cast<unsigned>(nb), st);
        else launch_norm_grad<float>(a, static_cast<unsigned>(nb), st);
    }
    if (params)
        hipLaunchKernelGGL(k_norm_grad_join, dim3(static_cast<unsigned>((2 * D + 63) / 64)), dim3(1024), 0, st, a.part,
                           nb, D, dweight, dbias);
    return launch_status(what);
}

}  // extern "C"
