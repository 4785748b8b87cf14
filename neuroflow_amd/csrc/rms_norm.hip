// rms_norm.hip -- RMS norm with the residual's addition, forward (to the
// activation's type or straight to 128-block FP8) and backward
// (include/nflow_residual.h).
#include <type_traits>

#include "nflow_residual.h"
#include "norm_dev.h"

namespace nfq {
namespace {

struct RmsArgs {
    const void* x;
    int64_t M, D, ldx;
    const void* r;
    int64_t ldr;
    const float* weight;
    float eps;
    void* y;
    int64_t ldy;
    uint8_t* codes;
    float* scales;
    void* sum;
    int64_t ldsum;
    float* rstd;
};

// The first `left` of eight codes, zero past them.  The values there are 0 times
// the row's rstd, which is a NaN or an infinity for some rows.
__device__ __forceinline__ v2u codes_below(v2u q, int left) {
    const uint64_t keep = left > 0 ? (uint64_t{1} << (8 * left)) - 1 : 0;
    return v2u{q[0] & static_cast<uint32_t>(keep), q[1] & static_cast<uint32_t>(keep >> 32)};
}

// ---- rows in registers --------------------------------------------------------
// The layout of k_norm: L threads hold a row, thread t the eight values from
// column 8 (t + L j) on.  x and the residual are read once, the next row's while
// this one is worked on; the sum of squares is about 0, so one reduction a row.
// The norm is of t in fp32; what is stored as the sum is t rounded once.
//
// HBM bound.  32768 x 256 fp32 with residual and sum 22.6 us (134 MB, 5.9 TB/s:
// part of it stays in the Infinity Cache), 16384 x 4096 bf16 to FP8 98 us (472 MB,
// 4.8 TB/s; 19.5 VALU instructions a value, the VALU busy a third of the time).  The
// sum goes past the caches (store8_stream): the next kernel reads y.
template <typename T, bool FP8, bool RES, int L, int NV>
__global__ __launch_bounds__(row_threads<L>()) void k_rms(RmsArgs a, int64_t per) {
    constexpr int G = row_threads<L>() / L;              // rows a workgroup holds
    __shared__ float part[2][L <= 64 ? 1 : L / 64];
    const int t = threadIdx.x % L;
    const int D = static_cast<int>(a.D);
    const float inv_d = 1.0f / static_cast<float>(D);
    float w[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) load_param(a.weight, 8 * (t + L * j), D, 1.0f, w[j]);
    Raw8<T> nx[NV], nr[RES ? NV : 1];
    auto fetch = [&](int64_t m) {
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
        const T* r = static_cast<const T*>(a.r) + m * a.ldr;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (t + L * j);
            nx[j].load(x + c, m < a.M ? D - c : 0);
            if constexpr (RES) nr[j].load(r + c, m < a.M ? D - c : 0);
        }
    };
    int64_t m = blockIdx.x * per + threadIdx.x / L;
    const int64_t end = blockIdx.x * per + per < a.M ? blockIdx.x * per + per : a.M;
    fetch(m < end ? m : a.M);
    int set = 0;
    for (int64_t i = 0; i < per; i += G, m += G, set ^= 1) {
        // Beyond a partial last round the lanes of absent rows work on zeros and
        // store nothing: the workgroup's barriers and the DPP reductions stay whole.
        const bool on = m < end;
        float v[NV][8], q = 0.0f;                        // 0 past column D, as the loads are
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[j][e] = RES ? nx[j][e] + nr[j][e] : nx[j][e];
                q = __builtin_fmaf(v[j][e], v[j][e], q);
            }
        fetch(i + G < per && m + G < end ? m + G : a.M);
        if constexpr (RES) {
            if (a.sum) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int c = 8 * (t + L * j);
                    store8_stream(static_cast<T*>(a.sum) + m * a.ldsum + c, on ? D - c : 0, v[j]);
                }
            }
        }
        const float rstd = norm_rstd(__builtin_fmaf(row_sum<L>(q, part, set), inv_d, a.eps));
        if (on && t == 0 && a.rstd) a.rstd[m] = rstd;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = v[j][e] * rstd * w[j][e];
        if constexpr (!FP8) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = 8 * (t + L * j);
                store8(static_cast<T*>(a.y) + m * a.ldy + c, on ? D - c : 0, v[j]);
            }
        } else {
            const int kb = static_cast<int>(blk_count(D));
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = 8 * (t + L * j);           // 16 threads hold a block of 128
                float amax = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = amax_of(amax, v[j][e]);
                const float sc = blk_scale(max16(amax));
                v2u q8 = blk_codes8(v[j], blk_inverse(sc));
                if (D - c < 8) q8 = codes_below(q8, D - c);
                if (on && c / kBlk < kb) {
                    __builtin_nontemporal_store(q8, reinterpret_cast<v2u*>(a.codes + m * kb * kBlk + c));
                    if (t % 16 == 0) a.scales[c / kBlk * a.M + m] = sc;
                }
            }
        }
    }
}

// ---- rows of any length ---------------------------------------------------------
// Past the register kernels' widths: one workgroup per row, two passes over it
// (the second from the caches).  The second reads each element where it writes
// the sum, so that the sum may lie in x or the residual.
template <typename T, bool FP8>
__global__ __launch_bounds__(kNormThreads) void k_rms_rows(RmsArgs a) {
    __shared__ float part[kNormThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
        const T* r = a.r ? static_cast<const T*>(a.r) + m * a.ldr : nullptr;
        T* sum = a.r && a.sum ? static_cast<T*>(a.sum) + m * a.ldsum : nullptr;
        auto total = [&](int64_t c) { return r ? to_f32(x[c]) + to_f32(r[c]) : to_f32(x[c]); };
        float q = 0.0f;
        for (int64_t c = tid; c < a.D; c += kNormThreads) {
            const float t = total(c);
            q = __builtin_fmaf(t, t, q);
        }
        const float rstd = norm_rstd(block_sum(q, part) / static_cast<float>(a.D) + a.eps);
        if (tid == 0 && a.rstd) a.rstd[m] = rstd;
        auto value = [&](int64_t c) {
            const float t = total(c);
            if (sum) sum[c] = from_f32<T>(t);
            return t * rstd * (a.weight ? a.weight[c] : 1.0f);
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

struct RmsGradArgs {
    const void* dy;
    const void* t;
    int64_t M, D, lddy, ldt;
    const float* weight;
    const float* rstd;
    const void* ds;
    int64_t ldds;
    void* dt;
    int64_t lddt;
    float* part;        // (workgroups, D) partial dweight, or null
    int64_t rows_per;   // rows of a workgroup's share (k_rms_grad_weight)
};

// ---- backward, rows in registers ---------------------------------------------------
// The layout of k_norm_grad: with h = t rstd and g = dy w, dt = rstd (g - h mean(g h))
// + dsum needs one sum over the row; dweight is a sum over rows of dy h, which every
// thread keeps for its columns over all of its rows and a workgroup joins over its
// G rows in LDS at the end, and a second launch over the workgroups in their order.
//
// HBM bound: 16384 x 4096 bf16 with dsum 95 us (537 MB, 5.6 TB/s: three parts read
// to one written) and 4.7 for the join of 256 partial rows.  AHEAD, the next row's
// loads under this one's work, where its registers leave the occupancy: else the
// workgroup's other waves hide them.
template <typename T, bool ADD, int L, int NV, int TH, bool AHEAD>
__global__ __launch_bounds__(TH) void k_rms_grad(RmsGradArgs a) {
    constexpr int G = TH / L, W = TH / 64;
    __shared__ float part[2][W];
    constexpr int SLOTS = L == 16 ? W : G;               // sums a column has after the waves' own
    __shared__ __attribute__((aligned(16))) float join[SLOTS > 1 ? SLOTS * 8 * L : 8];
    const int t = threadIdx.x % L, grp = threadIdx.x / L;
    const int D = static_cast<int>(a.D);
    const float inv_d = 1.0f / static_cast<float>(D);
    float w[NV][8], dw[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        load_param(a.weight, 8 * (t + L * j), D, 1.0f, w[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[j][e] = 0.0f;
    }
    Raw8<T> nx[NV], ny[NV], ns[ADD ? NV : 1];
    float nrstd = 0.0f;
    auto fetch = [&](int64_t m) {
        const bool on = m < a.M;
        const T* x = static_cast<const T*>(a.t) + m * a.ldt;
        const T* dy = static_cast<const T*>(a.dy) + m * a.lddy;
        const T* ds = static_cast<const T*>(a.ds) + m * a.ldds;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (t + L * j);
            nx[j].load(x + c, on ? D - c : 0);
            ny[j].load(dy + c, on ? D - c : 0);
            if constexpr (ADD) ns[j].load(ds + c, on ? D - c : 0);
        }
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
        float h[NV][8], g[NV][8], s[ADD ? NV : 1][8], sum = 0.0f;
        const float rstd = nrstd;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[j][e] = nx[j][e] * rstd;
                const float y = ny[j][e];
                dw[j][e] = __builtin_fmaf(y, h[j][e], dw[j][e]);
                g[j][e] = y * w[j][e];                 // 0 past column D, as y is
                sum = __builtin_fmaf(g[j][e], h[j][e], sum);
                if constexpr (ADD) s[j][e] = ns[j][e];
            }
        if (AHEAD) fetch(row(i + 1));
        if constexpr (L <= 64) {
            sum = lanes_reduce<L, SumOp>(sum);
        } else {
            sum = wave_sum(sum);
            if ((threadIdx.x & 63) == 0) part[i & 1][threadIdx.x >> 6] = sum;
            __syncthreads();
            sum = 0.0f;
#pragma unroll
            for (int k = 0; k < L / 64; ++k) sum += part[i & 1][grp * (L / 64) + k];
        }
        const float c2 = sum * inv_d;
        if (m < a.M) {
            T* dt = static_cast<T*>(a.dt) + m * a.lddt;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = 8 * (t + L * j);
                float o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[e] = rstd * __builtin_fmaf(-h[j][e], c2, g[j][e]);
                    if constexpr (ADD) o[e] += s[j][e];
                }
                store8_stream(dt + c, D - c, o);
            }
        }
    }
    if (!a.part) return;
    // One vector of columns at a time: a wave's four rows by the permlane swaps
    // (L = 16), then the groups' sums to LDS and a thread per column.
    float* out = a.part + blockIdx.x * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s[e] = dw[j][e];
            if constexpr (L == 16) s[e] = rows_sum(s[e]);
        }
        const int c = 8 * L * j;
        if constexpr (SLOTS == 1) {
            store8(out + c + 8 * t, D - c - 8 * t, s);
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
                out[c + u] = z;
            }
        }
    }
}

// ---- backward, rows of any length ---------------------------------------------------
// Past the register kernel's widths: dt a workgroup per row in two passes, the
// weight's partial sums a thread per column in a kernel of their own, ahead of
// the other, which may overwrite its inputs.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void k_rms_grad_rows(RmsGradArgs a) {
    __shared__ float part[kNormThreads / 64];
    const int tid = threadIdx.x;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const T* x = static_cast<const T*>(a.t) + m * a.ldt;
        const T* dy = static_cast<const T*>(a.dy) + m * a.lddy;
        const T* ds = a.ds ? static_cast<const T*>(a.ds) + m * a.ldds : nullptr;
        T* dt = static_cast<T*>(a.dt) + m * a.lddt;
        const float rstd = a.rstd[m];
        float s = 0.0f;
        for (int64_t c = tid; c < a.D; c += kNormThreads)
            s = __builtin_fmaf(to_f32(dy[c]) * (a.weight ? a.weight[c] : 1.0f), to_f32(x[c]) * rstd, s);
        const float c2 = block_sum(s, part) / static_cast<float>(a.D);
        for (int64_t c = tid; c < a.D; c += kNormThreads) {
            const float g = to_f32(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            const float o = rstd * __builtin_fmaf(-(to_f32(x[c]) * rstd), c2, g);
            dt[c] = from_f32<T>(ds ? o + to_f32(ds[c]) : o);
        }
    }
}

// Partial sums of dy * h over a block's rows, a thread per column.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void k_rms_grad_weight(RmsGradArgs a) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x;
    if (c >= a.D) return;
    const int64_t m0 = blockIdx.y * a.rows_per, m1 = m0 + a.rows_per < a.M ? m0 + a.rows_per : a.M;
    float dw = 0.0f;
    for (int64_t m = m0; m < m1; ++m)
        dw = __builtin_fmaf(to_f32(static_cast<const T*>(a.dy)[m * a.lddy + c]),
                            to_f32(static_cast<const T*>(a.t)[m * a.ldt + c]) * a.rstd[m], dw);
    a.part[blockIdx.y * a.D + c] = dw;
}

// dweight = the sum of part (P, D) over P, every sixteenth row a wave, the waves'
// sums in turn.
__global__ __launch_bounds__(1024) void k_rms_grad_join(const float* __restrict__ part, int64_t P, int64_t D,
                                                        float* __restrict__ dweight) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    float v = 0.0f;
    if (n < D) {
#pragma unroll 8
        for (int64_t p = wave; p < P; p += 16) v += part[p * D + n];
    }
    s[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && n < D) {
        float z = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) z += s[k][lane];
        dweight[n] = z;
    }
}

// Workgroups (and partial rows) of the backward pass.
int64_t rms_grad_blocks(int64_t M) { return std::min<int64_t>(M, num_cus()); }

size_t rms_grad_space(int64_t M, int64_t D) {
    return static_cast<size_t>(rms_grad_blocks(M)) * static_cast<size_t>(D) * sizeof(float);
}

template <typename T, bool FP8, bool RES, int L, int NV>
void launch_rms(const RmsArgs& a, hipStream_t st) {
    constexpr int threads = row_threads<L>(), G = threads / L;
    static const int64_t most = resident(k_rms<T, FP8, RES, L, NV>, threads);
    const int64_t groups = (a.M + G - 1) / G, per = (groups + most - 1) / most * G;
    hipLaunchKernelGGL((k_rms<T, FP8, RES, L, NV>), dim3(static_cast<unsigned>((a.M + per - 1) / per)), dim3(threads), 0,
                       st, a, per);
}

// The fewest threads that hold a row in 8 NV values each: fewer threads a row
// means more rows at once and shorter reductions.
template <typename T, bool FP8, bool RES>
void launch_rms_rows(const RmsArgs& a, hipStream_t st) {
    if (a.D <= 128) launch_rms<T, FP8, RES, 16, 1>(a, st);
    else if (a.D <= 256) launch_rms<T, FP8, RES, 16, 2>(a, st);
    else if (a.D <= 512) launch_rms<T, FP8, RES, 64, 1>(a, st);
    else if (a.D <= 1024) launch_rms<T, FP8, RES, 64, 2>(a, st);
    else if (a.D <= 2048) launch_rms<T, FP8, RES, 64, 4>(a, st);
    else if (a.D <= 4096) launch_rms<T, FP8, RES, 256, 2>(a, st);
    else if (a.D <= 8192) launch_rms<T, FP8, RES, 256, 4>(a, st);
    else if (a.D <= kNormRegMax) launch_rms<T, FP8, RES, 1024, 2>(a, st);
    else hipLaunchKernelGGL((k_rms_rows<T, FP8>), dim3(row_grid(a.M)), dim3(kNormThreads), 0, st, a);
}

// Threads a row and a workgroup as launch_norm_grad has them.
template <typename T, bool ADD>
void launch_rms_grad(const RmsGradArgs& a, unsigned nb, hipStream_t st) {
    auto go = [&](auto k, int threads) { hipLaunchKernelGGL(k, dim3(nb), dim3(threads), 0, st, a); };
    if (a.D <= 128) go(k_rms_grad<T, ADD, 16, 1, 1024, true>, 1024);
    else if (a.D <= 256) go(k_rms_grad<T, ADD, 16, 2, 1024, false>, 1024);
    else if (a.D <= 512) go(k_rms_grad<T, ADD, 64, 1, 1024, true>, 1024);
    else if (a.D <= 1024) go(k_rms_grad<T, ADD, 64, 2, 1024, false>, 1024);
    else if (a.D <= 2048) go(k_rms_grad<T, ADD, 256, 1, 1024, true>, 1024);
    else if (a.D <= 4096) go(k_rms_grad<T, ADD, 256, 2, 1024, false>, 1024);
    else if (a.D <= 8192) go(k_rms_grad<T, ADD, 1024, 1, 1024, true>, 1024);
    else if (a.D <= kNormRegMax) go(k_rms_grad<T, ADD, 1024, 2, 1024, false>, 1024);
    else {
        if (a.part) {
            const unsigned gc = static_cast<unsigned>((a.D + kNormThreads - 1) / kNormThreads);
            hipLaunchKernelGGL((k_rms_grad_weight<T>), dim3(gc, nb), dim3(kNormThreads), 0, st, a);
        }
        hipLaunchKernelGGL((k_rms_grad_rows<T>), dim3(row_grid(a.M)), dim3(kNormThreads), 0, st, a);
    }
}

// What both forward entry points check; *run: whether there is work.
int check_rms(const char* what, const RmsArgs& a, int dtype, bool* run) {
    *run = false;
    if (!dtype_ok(dtype)) return bad_arg(what, "unknown dtype");
    if (a.M < 0 || a.D <= 0) return bad_arg(what, "bad dims");
    if (a.ldx < a.D || (a.r && a.ldr < a.D) || (a.sum && a.ldsum < a.D) || (a.y && a.ldy < a.D))
        return bad_arg(what, "row stride smaller than a row");
    if (!(a.eps >= 0.0f)) return bad_arg(what, "eps must not be negative or NaN");
    if (a.sum && !a.r) return bad_arg(what, "a sum without a residual");
    if (a.M == 0) return NFLOW_OK;
    if (!a.x) return bad_arg(what, "null x");
    const size_t e = dtype_size(dtype);
    for (int k = 0; k < 2; ++k) {
        const void* out = k ? a.sum : a.y;
        const int64_t ld = k ? a.ldsum : a.ldy;
        if (!out) continue;
        if (rows_clash(a.x, a.ldx, out, ld, a.M, a.D, e) || (a.r && rows_clash(a.r, a.ldr, out, ld, a.M, a.D, e)))
            return bad_arg(what, kOverlap);
    }
    if (a.y && a.sum && (a.y == a.sum || rows_clash(a.y, a.ldy, a.sum, a.ldsum, a.M, a.D, e)))
        return bad_arg(what, "y and sum overlap");
    // What lies alone in memory, of which weight is an input.
    const Span w(a.weight, a.D, sizeof(float)), rs(a.rstd, a.M, sizeof(float)), c(a.codes, a.M * blk_count(a.D) * kBlk, 1),
        sc(a.scales, a.M * blk_count(a.D), sizeof(float));
    const Span y(a.y, a.M, a.D, a.ldy, e), s(a.sum, a.M, a.D, a.ldsum, e);
    for (const Span& m : {Span(a.x, a.M, a.D, a.ldx, e), Span(a.r, a.M, a.D, a.ldr, e), w, y, s})
        if (meet(m, rs) || meet(m, c) || meet(m, sc)) return bad_arg(what, kShared);
    if (meet(w, y) || meet(w, s) || meet(rs, c) || meet(rs, sc) || meet(c, sc)) return bad_arg(what, kShared);
    *run = true;
    return NFLOW_OK;
}

template <bool FP8>
int rms_forward(const char* what, const RmsArgs& a, int dtype, void* stream) {
    hipStream_t st = as_stream(stream);
    if (dtype == NFLOW_DTYPE_BF16) {
        if (a.r) launch_rms_rows<bf16, FP8, true>(a, st);
        else launch_rms_rows<bf16, FP8, false>(a, st);
    } else {
        if (a.r) launch_rms_rows<float, FP8, true>(a, st);
        else launch_rms_rows<float, FP8, false>(a, st);
    }
    return launch_status(what);
}

}  // namespace
}  // namespace nfq

using namespace nfq;

extern "C" {

int nflow_rms_norm_forward(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const void* residual,
                           int64_t ldr, const float* weight, float eps, void* y, int64_t ldy, void* sum,
                           int64_t ldsum, float* rstd, void* stream) {
    clear_error();
    const char* what = "rms_norm_forward";
    const RmsArgs a{x, M, D, ldx, residual, ldr, weight, eps, y, ldy, nullptr, nullptr, sum, ldsum, rstd};
    bool run = false;
    if (int rc = check_rms(what, a, dtype, &run)) return rc;
    if (!run) return NFLOW_OK;
    if (!y) return bad_arg(what, "null y");
    return rms_forward<false>(what, a, dtype, stream);
}

int nflow_rms_norm_fp8(const void* x, int dtype, int64_t M, int64_t D, int64_t ldx, const void* residual,
                       int64_t ldr, const float* weight, float eps, uint8_t* codes, float* scales, void* sum,
                       int64_t ldsum, float* rstd, void* stream) {
    clear_error();
    const char* what = "rms_norm_fp8";
    const RmsArgs a{x, M, D, ldx, residual, ldr, weight, eps, nullptr, 0, codes, scales, sum, ldsum, rstd};
    bool run = false;
    if (int rc = check_rms(what, a, dtype, &run)) return rc;
    if (!run) return NFLOW_OK;
    if (!codes || !scales) return bad_arg(what, "null codes or scales");
    if (!aligned(codes, 16)) return bad_arg(what, "codes must be 16-byte aligned");
    return rms_forward<true>(what, a, dtype, stream);
}

int nflow_rms_norm_backward_workspace(int64_t M, int64_t D, size_t* bytes) {
    clear_error();
    if (!bytes) return bad_arg("rms_norm_backward_workspace", "null output");
    *bytes = 0;
    if (M < 0 || D <= 0) return bad_arg("rms_norm_backward_workspace", "bad dims");
    *bytes = rms_grad_space(M, D);
    return NFLOW_OK;
}

int nflow_rms_norm_backward(const void* dy, const void* t, int dtype, int64_t M, int64_t D, int64_t lddy,
                            int64_t ldt, const float* weight, const float* rstd, const void* dsum, int64_t lddsum,
                            void* dt, int64_t lddt, float* dweight, void* workspace, size_t workspace_bytes,
                            void* stream) {
    clear_error();
    const char* what = "rms_norm_backward";
    if (!dtype_ok(dtype)) return bad_arg(what, "unknown dtype");
    if (M < 0 || D <= 0) return bad_arg(what, "bad dims");
    if (lddy < D || ldt < D || lddt < D || (dsum && lddsum < D)) return bad_arg(what, "row stride smaller than a row");
    if (M > 0 && (!dy || !t || !rstd || !dt)) return bad_arg(what, "null dy, t, rstd or dt");
    const size_t e = dtype_size(dtype);
    if (rows_clash(dy, lddy, dt, lddt, M, D, e) || rows_clash(t, ldt, dt, lddt, M, D, e) ||
        (dsum && rows_clash(dsum, lddsum, dt, lddt, M, D, e)))
        return bad_arg(what, kOverlap);
    const Span w(weight, D, sizeof(float)), rs(rstd, M, sizeof(float)), dw(dweight, D, sizeof(float)), d(dt, M, D, lddt, e);
    for (const Span& m : {w, rs, d, Span(dy, M, D, lddy, e), Span(t, M, D, ldt, e), Span(dsum, M, D, lddsum, e)})
        if (meet(m, dw)) return bad_arg(what, kShared);
    if (meet(w, d) || meet(rs, d)) return bad_arg(what, kShared);
    if (int rc = check_workspace(what, workspace, workspace_bytes, rms_grad_space(M, D))) return rc;
    hipStream_t st = as_stream(stream);
    const int64_t nb = rms_grad_blocks(M);
    if (M == 0 && !dweight) return NFLOW_OK;
    const RmsGradArgs a{dy, t, M, D, lddy, ldt, weight, rstd, dsum, lddsum, dt, lddt,
                        dweight ? static_cast<float*>(workspace) : nullptr, nb ? (M + nb - 1) / nb : 0};
    if (M > 0) {
        const unsigned n = static_cast<unsigned>(nb);
        if (dtype == NFLOW_DTYPE_BF16) {
            if (dsum) launch_rms_grad<bf16, true>(a, n, st);
            else launch_rms_grad<bf16, false>(a, n, st);
        } else {
            if (dsum) launch_rms_grad<float, true>(a, n, st);
            else launch_rms_grad<float, false>(a, n, st);
        }
    }
    if (dweight)
        hipLaunchKernelGGL(k_rms_grad_join, dim3(static_cast<unsigned>((D + 63) / 64)), dim3(1024), 0, st, a.part, nb, D,
                           dweight);
    return launch_status(what);
}

}  // extern "C"
