// dense.hip -- the linear layer in bf16 or fp32, forward and backward
// (include/nflow_residual.h): the cut of its products, the gradient ahead of the
// activation, and the entry points.
#include <type_traits>

#include "dense.h"

namespace nfq {
namespace {

// ---- dz and dbias ------------------------------------------------------------------

// act'(z) times dy.  For GELU with p = 1 / (1 + 2^(z (k1 + k3 z^2))), z p is the
// activation (gelu_tanh) and its slope p + z p (1 - p) 2 c (1 + 3 * 0.044715 z^2);
// 1 - p from whichever side has no cancellation.  Past |z| = 64 the slope is 0 or
// 1 to all bits, and z is held there, so that no infinity meets a 0.
__device__ __forceinline__ float act_grad(float dy, float z, int act) {
    if (act == NFLOW_ACT_RELU) return z > 0.0f ? dy : (z != z ? z : 0.0f);
    const float k1 = -0x1.26aec2p+1f;       // -2 sqrt(2 / pi) log2(e)
    const float k3 = -0x1.a5a7cep-4f;       // 0.044715 k1
    const float c2 = 0x1.988454p+0f;        // 2 sqrt(2 / pi)
    const float c6 = 0x1.b6676cp-3f;        // 3 * 0.044715 c2
    z = z > 64.0f ? 64.0f : (z < -64.0f ? -64.0f : z);
    const float zz = z * z;
    const float e = __builtin_amdgcn_exp2f(z * __builtin_fmaf(k3, zz, k1));
    const float p = __builtin_amdgcn_rcpf(1.0f + e);
    const float q = z > 0.0f ? e * p : 1.0f - p;
    return dy * __builtin_fmaf(z * p * q, __builtin_fmaf(c6, zz, c2), p);
}

// dz = dy act'(pre), and the sums of dz's columns over this workgroup's rows:
// a thread has eight columns and every eighth row, and the eight threads of a
// column join in LDS.  With no activation only the sums.
//
// HBM bound beside the slope's VALU work: 65536 x 1024 bf16 with GELU 80 us (403 MB, 5.0
// TB/s, VALU 58%).  A pass of its own: dx and dW both read dz, at tiles of 256 four
// times each, and the slope would be taken at every read.
//
// dz is rounded to the activations' type, and the products take it as it is returned.
// In bf16 that is a second rounding of half a step beside dx's and dW's own: in the
// 2-norm they are 2.3e-3 from the formula, where a dz kept in fp32 leaves 1.7e-3.  The
// rest of it would be a second bf16 operand, and both products (280 of the 345 us of
// 65536 x 1024 -> 1024) twice the work.  dbias, which costs nothing more, sums dz
// ahead of the rounding.
constexpr int kDzCols = 256, kDzRows = 8;            // of a workgroup at a time
struct DzArgs {
    const void* dy;
    const void* pre;
    void* dz;
    int64_t M, N, lddy, ldpre, lddz;
    int act;
    float* part;        // (row runs, N), or null
    int64_t rows_per;
};
template <typename T>
__global__ __launch_bounds__(256) void k_dense_dz(DzArgs a) {
    __shared__ __attribute__((aligned(16))) float join[kDzRows][kDzCols];
    const int c = 8 * (threadIdx.x & 31), g = threadIdx.x >> 5;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * kDzCols + c, left = a.N - n;
    const int64_t m0 = blockIdx.y * a.rows_per, m1 = m0 + a.rows_per < a.M ? m0 + a.rows_per : a.M;
    float s[8] = {};
    auto run = [&](int64_t have) {
#pragma unroll 4
        for (int64_t m = m0 + g; m < m1; m += kDzRows) {
            float d[8];
            load8(static_cast<const T*>(a.dy) + m * a.lddy + n, have, d);
            if (a.act != NFLOW_ACT_NONE) {
                float z[8];
                load8(static_cast<const T*>(a.pre) + m * a.ldpre + n, have, z);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = act_grad(d[e], z[e], a.act);
                store8(static_cast<T*>(a.dz) + m * a.lddz + n, have, d);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += d[e];
        }
    };
    if (left >= 8) run(8);                           // without the ends of rows in its loop: loads stay in flight
    else if (left > 0) run(left);
    if (!a.part) return;
#pragma unroll
    for (int e = 0; e < 8; e += 4) *reinterpret_cast<v4f*>(&join[g][c + e]) = v4f{s[e], s[e + 1], s[e + 2], s[e + 3]};
    __syncthreads();
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kDzCols + threadIdx.x;
    if (col >= a.N) return;
    float z = 0.0f;
#pragma unroll
    for (int k = 0; k < kDzRows; ++k) z += join[k][threadIdx.x];
    a.part[blockIdx.y * a.N + col] = z;
}

// dbias = the sum of part (P, N) over P.
__global__ __launch_bounds__(256) void k_dense_dbias(const float* __restrict__ part, int64_t P, int64_t N,
                                                     float* __restrict__ dbias) {
    __shared__ float s[16][17];
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 16 + c;
    float v = 0.0f;
    if (n < N) {
#pragma unroll 8
        for (int64_t p = g; p < P; p += 16) v += part[p * N + n];
    }
    s[g][c] = v;
    __syncthreads();
    if (g == 0 && n < N) {
        float z = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) z += s[k][c];
        dbias[n] = z;
    }
}

// Runs of rows of the sums: four workgroups a CU, of 32 rows at least.
int64_t dz_runs(int64_t M, int64_t N) {
    const int64_t cols = (N + kDzCols - 1) / kDzCols;
    return std::max<int64_t>(1, std::min<int64_t>((M + 31) / 32, 4 * num_cus() / std::max<int64_t>(cols, 1)));
}

// ---- the cut -----------------------------------------------------------------------------

// The cut with the least estimated time, in us: `steps` of 64 k's, of which a
// workgroup alone on its CU takes `alone` each and n together `each` apiece, and
// `tile` for what a tile does outside its K loop.  Dealt out whole, the busiest
// CU has ceil(tiles / CUs) of them.  Dealt out to `groups` workgroups, with the K
// steps of what is left shared evenly, every CU is as busy as the next, for the
// shared parts' way through the caches and a second launch.  The times rank the
// cuts of one product; as times they are low where few steps leave a tile's first
// loads and stores bare (a product of 1537 x 2021 -> 1001 10.6 us for the 22.5 of a
// trace, dx of 65536 x 1024 -> 1024 117 for 139 to 154, 32768 x 256 -> 256 in fp32 24 for
// 37.5).  They are those of steps at 256 to 1024 tiles of 16 and 64 steps, but for fp32
// tiles of 64: 69 x 4864 -> 2688 and 1024 x 2048 -> 1024.  `across`: a step of the backward
// products to one of the forward's, in fp32, whose planes of operands across k go to
// LDS and come from it in more pieces (us, by tiles of 64, 128 and 256: 1024 x 1024 x 1024
// backward 62, 43, 43; 83 x 1536 x 1024 31, 26, 35; 64 x 1536 x 1024 22, 24, 36).
struct Cut {
    DenseKind kind;
    int bm, bn, per_cu;
    double alone, each, tile, across;
    double step(DenseForm form, double per) const {
        return (form == DENSE_FORWARD ? 1.0 : across) * std::max(alone, per * each);
    }
    double tiles(int64_t M, int64_t N) const {
        return std::ceil(static_cast<double>(M) / bm) * std::ceil(static_cast<double>(N) / bn);
    }
    // `steps` of 64 k's evenly dealt out to `groups` workgroups, `occ` a CU, in `pieces` of
    // tiles each, of which `parts` in all are shared, `deep` to a tile: a join of 32, 64 and
    // 128 slots of 64 x 64 takes 5.0, 7.8 and 12.5 us.
    DensePlan shared(DenseForm form, int occ, int groups, double steps, double pieces, double parts, double deep) const {
        const size_t slot = static_cast<size_t>(bm) * (bn + 1) * sizeof(float);
        const double us = (steps / groups + 0.5) * step(form, occ) + pieces * occ * tile + 3.0 +
                          2 * parts * static_cast<double>(slot) / 5e6 + 0.07 * deep;
        return DensePlan{kind, groups, round16(2 * groups * slot), us};
    }
};
const Cut kCutsBf16[] = {{DENSE_SMALL, 64, 64, 3, 0.233, 0.182, 0.7, 1.0},
                         {DENSE_TALL, 128, 64, 2, 0.294, 0.273, 1.2, 1.0},
                         {DENSE_MID, 128, 128, 2, 0.613, 0.435, 2.4, 1.0},
                         {DENSE_DEEP, 128, 128, 1, 0.481, 0.476, 2.6, 1.0},
                         {DENSE_BIG, 256, 256, 1, 1.43, 1.50, 5.3, 1.0}};
const Cut kCutsF32[] = {{DENSE_SMALL, 64, 64, 3, 1.45, 0.90, 1.0, 1.7},
                        {DENSE_MID, 128, 128, 1, 2.66, 2.66, 2.5, 1.12},
                        {DENSE_BIG, 256, 128, 1, 4.77, 4.77, 5.0, 1.0}};
template <typename F>
void each_cut(int dtype, F f) {
    if (dtype == NFLOW_DTYPE_F32) {
        for (const Cut& c : kCutsF32) f(c);
    } else {
        for (const Cut& c : kCutsBf16) f(c);
    }
}
double steps_of(int64_t K) { return static_cast<double>((K + 63) / 64); }

// The least estimated time of tiles.
DensePlan tiles_plan(DenseForm form, int64_t M, int64_t N, int64_t K, int dtype) {
    const double cus = num_cus(), steps = steps_of(K);
    DensePlan best{DENSE_MID, 0, 0, HUGE_VAL};
    each_cut(dtype, [&](const Cut& c) {
        const double tiles = c.tiles(M, N), per = std::ceil(tiles / cus);
        const double us = steps * c.step(form, per) + per * c.tile;
        if (us < best.us) best = DensePlan{c.kind, 0, 0, us};
        for (int occ = 1; occ <= c.per_cu; ++occ) {
            // Every workgroup that fits, or where there is little to share 8, 4 or 2 steps to
            // each: fewer parts to join (us, every workgroup against those: 64 x 8192 -> 64 bf16 31 : 9.6,
            // 42 x 64 -> 2792 fp32 backward 84 : 18).
            for (int least = occ == 1 ? 8 : 1; least > 0; least /= 2) {
                const double most = least == 1 ? occ * cus : std::floor(tiles * steps / least);
                if (most > occ * cus || (least > 1 && most <= tiles)) continue;
                const int groups = static_cast<int>(most);
                const int64_t whole = static_cast<int64_t>(tiles) / groups, rest = static_cast<int64_t>(tiles) % groups;
                if (rest == 0 || rest * steps < groups) continue;
                const DensePlan p = c.shared(form, occ, groups, tiles * steps, static_cast<double>(whole + 2),
                                             static_cast<double>(groups + rest), static_cast<double>(groups) / rest);
                if (p.us < best.us) best = p;
            }
        }
    });
    return best;
}

// ---- few rows ----------------------------------------------------------------------------

// How a bf16 operand's rows lie: as the tiles' DMA takes them, at whole 4-byte words or
// at any element.  Of the latter two the tiles take copies; k_dense_few, which reads
// operands in place, is held up by rows off whole words.  (fp32 operands: as the DMA
// takes them, for all that it matters.)
enum Lie { LIE_GROUPS, LIE_WORDS, LIE_ANY };
Lie lie_of(const void* p, int64_t ld, int64_t cols, int dtype) {
    if (dtype != NFLOW_DTYPE_BF16 || dense_fetchable(p, ld, cols)) return LIE_GROUPS;
    return aligned(p, 4) && ld % 2 == 0 ? LIE_WORDS : LIE_ANY;
}

size_t copy_space(int64_t rows, int64_t cols) { return round16(static_cast<size_t>(rows * dense_pitch(cols)) * 2); }

// x (M, K) and W (N, K) of a forward product, few rows of x.
struct FewRows {
    int64_t M, N, K;
    int dtype;
    // A call of k_dense_few's, in us: a weight's pieces of 128 bytes, sixteen waves a CU, or
    // its way from HBM.  A piece waits for 16 rows of the weight and M of x, for each of
    // x's 0.052 us in whole groups, 0.077 in words, 0.18 at any element.
    double us(Lie x, Lie w) const {
        const double bytes = static_cast<double>(K) * dtype_size(dtype), columns = std::ceil(static_cast<double>(N) / 16);
        const double full = columns / num_cus(), pieces = std::ceil(bytes / 128) * std::ceil(full) / 16;
        const double row = x == LIE_GROUPS ? 0.052 : x == LIE_WORDS ? 0.077 : 0.18;
        const double weight = w == LIE_ANY ? 3.1 : 0.95 + 0.5 * std::min(full, 1.0);
        return 3.0 + std::max(N * bytes / 5e6, pieces * (weight + row * M));
    }
    // The tiles' copies of what they cannot fetch: room, and us (a launch that overlaps the
    // product's, and the bytes at a copy's rate).
    size_t copied(Lie x, Lie w) const { return (x ? copy_space(M, K) : 0) + (w ? copy_space(N, K) : 0); }
    double copy_us(Lie x, Lie w) const { return x || w ? 2.0 + 2 * static_cast<double>(copied(x, w)) / 5e6 : 0.0; }
    // Whether it is estimated faster than tiles whose call is estimated at `tiles` us: they
    // gain with much to sum in few columns or with a large weight, by the rate that they read
    // it at, and lose their copies.  Measured, us a call, few against tiles: bf16, one row
    // of 4096 -> 4096 7.9 : 14.0, of 16384 -> 256 19.5 : 15.7; 32 rows of 1024 -> 4096 5.5 :
    // 7.6, of 4096 -> 16384 52.7 : 34.0; of rows in words, 17 of 16382 -> 16384 185 : 367, 32 of
    // 4094 -> 1024 13.7 : 17.4; at any element, one of 1023 -> 16384 15.7 : 22.5, 17 of 4095 ->
    // 1024 27.9 : 17.4, 32 of 8191 -> 4096 75.9 : 43.1.  fp32, 16 rows of 4096 -> 4096
    // 19.0 : 26.5, 32 of 4096 -> 256 24.4 : 11.6, of 16384 -> 4096 93.7 : 89.6.  Over 500 sizes
    // of rows off 16-byte groups the choice takes 1% longer than the faster of the two, the
    // worst 1.4 times as long.
    bool faster(Lie x, Lie w, double tiles) const {
        const double read = static_cast<double>(N) * K / (dtype == NFLOW_DTYPE_F32 ? 0.75e6 : 2e6);
        return us(x, w) <= std::max(tiles, read) + copy_us(x, w);
    }
    // Tiles' calls: the least that any is, and a plan's.
    double least() const { return 4.0 + std::min(6.0, 0.2 * steps_of(K)); }
    static double call(const DensePlan& tiles) { return tiles.us + (tiles.groups ? 7.0 : 4.0); }
};

DensePlan dense_plan(DenseForm form, int64_t M, int64_t N, int64_t K, int dtype, Lie x = LIE_GROUPS, Lie w = LIE_GROUPS) {
    if (form != DENSE_FORWARD || M > kDenseFewRows) return tiles_plan(form, M, N, K, dtype);
    const FewRows f{M, N, K, dtype};
    const DensePlan few{DENSE_FEW, 0, 0, f.us(x, w)};
    if (f.faster(x, w, f.least())) return few;
    const DensePlan tiles = tiles_plan(form, M, N, K, dtype);
    return f.faster(x, w, FewRows::call(tiles)) ? few : tiles;
}

// dx (M, K) and dW (N, K) of fp32 in one launch, where that is faster than the two
// by themselves, which pay a launch more (us: 2048 x 2048 x 2048 171 against 196,
// 20000 x 256 x 768 118 against 136); else groups is 0.  In bf16, where the parts of
// shared tiles weigh six times as much against the products, it is not (4096 x
// 1024 x 1024 44 against 45, 65536 x 1024 x 1024 343 against 302).
DensePlan pair_plan(int64_t M, int64_t N, int64_t K, int dtype, const DensePlan& x, const DensePlan& w) {
    DensePlan best{DENSE_MID, 0, 0, 0.0};
    if (dtype != NFLOW_DTYPE_F32 || M <= 0 || N <= 0 || K <= 0) return best;
    best.us = x.us + w.us + 3.0;
    for (const Cut& c : kCutsF32) {
        const double tx = c.tiles(M, K), tw = c.tiles(N, K), steps = tx * steps_of(N) + tw * steps_of(M);
        for (int occ = 1; occ <= c.per_cu; ++occ) {
            const int groups = static_cast<int>(std::min<double>(occ * num_cus(), std::floor(steps / 2)));
            if (groups < 2 || (occ > 1 && groups <= num_cus())) continue;
            // Tiles of one length in whole rounds: none is shared.
            const bool even = steps_of(N) == steps_of(M) && std::fmod(tx + tw, groups) == 0.0;
            const double deep = std::max(steps_of(N), steps_of(M)) * groups / steps;
            const DensePlan p = c.shared(DENSE_DW, occ, groups, steps, std::ceil((tx + tw) / groups) + (even ? 0 : 1),
                                         even ? 0 : 2.0 * groups, even ? 0 : deep);
            if (p.us < best.us) best = p;
        }
    }
    return best;
}

int product(const char* what, DenseForm form, const DensePlan& p, const DenseArgs& a, int dtype, void* ws, hipStream_t st) {
    if (a.M == 0 || a.N == 0) return NFLOW_OK;
    bool many = false;
    const bool b16 = dtype == NFLOW_DTYPE_BF16;
    // A launch has at most 2^32 threads: 512 for each tile (of 64 x 64 or more) dealt out whole.
    each_cut(dtype, [&](const Cut& c) { many |= c.kind == p.kind && !p.groups && c.tiles(a.M, a.N) > (1 << 23) - 1; });
    if (many) return bad_arg(what, "too many results for one launch");
    if (p.kind == DENSE_FEW) {
        if (b16) launch_dense_few<bf16>(a, st);
        else launch_dense_few<float>(a, st);
    } else {
        if (b16) launch_dense_bf16(a, form, p, static_cast<float*>(ws), st);
        else launch_dense_f32(a, form, p, static_cast<float*>(ws), st);
    }
    return launch_status(what);
}

// ---- operands that the tiled product of bf16 cannot fetch where they lie ---------------------

// Operands on their way into a product; those that need it are copied to `to`, all by one launch.
struct Copies {
    DensePack m[3] = {};
    int n = 0;
    size_t bytes = 0;
    // p and its row stride, as the product takes them.
    void take(const void*& p, int64_t& ld, int64_t rows, int64_t cols, void* to) {
        if (dense_fetchable(p, ld, cols)) return;
        uint8_t* at = static_cast<uint8_t*>(to) + bytes;
        m[n++] = DensePack{p, at, rows, cols, ld};
        bytes += copy_space(rows, cols);
        p = at;
        ld = dense_pitch(cols);
    }
};

int check_sizes(const char* what, int64_t M, int64_t N, int64_t K, int dtype) {
    if (M < 0 || N < 0 || K < 0) return bad_arg(what, "bad dims");
    if (!dtype_ok(dtype)) return bad_arg(what, "unknown dtype");
    const int64_t top = std::max(std::max(M, N), K);
    if (K > NFLOW_DENSE_MAX_K || N > NFLOW_DENSE_MAX_K || top > INT64_C(1) << 35)
        return bad_arg(what, "more than NFLOW_DENSE_MAX_K columns, or too many rows");
    auto many = [](int64_t m, int64_t n) { return ((m + 63) / 64) * ((n + 63) / 64) > INT32_MAX / 16; };
    if (many(M, N) || many(M, K) || many(N, K)) return bad_arg(what, "too many results for one launch");
    return NFLOW_OK;
}

int check_act(const char* what, int act) {
    if (act != NFLOW_ACT_NONE && act != NFLOW_ACT_RELU && act != NFLOW_ACT_GELU_TANH)
        return bad_arg(what, "unknown activation");
    return NFLOW_OK;
}

// What a call launches and the room it takes.
struct ForwardPlan {
    DensePlan p;
    size_t parts = 0;
    bool tiled = false;      // on operands that the DMA fetches
    ForwardPlan(int64_t M, int64_t N, int64_t K, int dtype, Lie x, Lie w)
        : p(dense_plan(DENSE_FORWARD, M, N, K, dtype, x, w)) {
        if (M == 0 || N == 0 || K == 0) return;
        parts = p.bytes;
        tiled = dtype == NFLOW_DTYPE_BF16 && p.kind != DENSE_FEW;
    }
};
// The room for x and W that both lie in groups, or the most that it is for what `copies` says.
size_t forward_space(int64_t M, int64_t N, int64_t K, int dtype, int copies) {
    if (M == 0 || N == 0 || K == 0) return 0;
    if (!copies || dtype != NFLOW_DTYPE_BF16) return ForwardPlan(M, N, K, dtype, LIE_GROUPS, LIE_GROUPS).parts;
    const FewRows f{M, N, K, dtype};
    DensePlan tiles{DENSE_FEW, 0, 0, 0.0};
    size_t bytes = 0;
    for (Lie x : {LIE_GROUPS, LIE_WORDS, LIE_ANY})
        for (Lie w : {LIE_GROUPS, LIE_WORDS, LIE_ANY}) {
            if (copies == 2 && (x == LIE_ANY || w == LIE_ANY)) continue;
            if (M <= kDenseFewRows && f.faster(x, w, f.least())) continue;
            if (tiles.kind == DENSE_FEW) tiles = tiles_plan(DENSE_FORWARD, M, N, K, dtype);
            if (M <= kDenseFewRows && f.faster(x, w, FewRows::call(tiles))) continue;
            bytes = std::max(bytes, tiles.bytes + f.copied(x, w));
        }
    return bytes;
}
struct BackwardPlan {
    DensePlan x, w, pair;
    size_t sums = 0, x_parts = 0, bytes;
    BackwardPlan(int64_t M, int64_t N, int64_t K, int dtype)
        : x(dense_plan(DENSE_DX, M, K, N, dtype)), w(dense_plan(DENSE_DW, N, K, M, dtype)),
          pair(pair_plan(M, N, K, dtype, x, w)) {
        if (M > 0) sums = round16(static_cast<size_t>(dz_runs(M, N) * N) * sizeof(float));
        bytes = sums;
        if (M == 0 || N == 0 || K == 0) return;
        x_parts = x.bytes;
        bytes += std::max(x.bytes + w.bytes, pair.bytes);
    }
};

}  // namespace
}  // namespace nfq

using namespace nfq;

extern "C" {

int nflow_dense_linear_workspace(int64_t M, int64_t N, int64_t K, int dtype, int copies, size_t* bytes) {
    clear_error();
    const char* what = "dense_linear_workspace";
    if (!bytes) return bad_arg(what, "null output");
    *bytes = 0;
    if (int rc = check_sizes(what, M, N, K, dtype)) return rc;
    *bytes = forward_space(M, N, K, dtype, copies);
    return NFLOW_OK;
}

int nflow_dense_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* W, int64_t ldw,
                       int64_t N, const float* bias, const void* residual, int64_t ldr, int activation, void* y,
                       int64_t ldy, void* pre, int64_t ldpre, void* workspace, size_t workspace_bytes,
                       void* stream) {
    clear_error();
    const char* what = "dense_linear";
    if (int rc = check_sizes(what, M, N, K, dtype)) return rc;
    if (int rc = check_act(what, activation)) return rc;
    if (ldx < K || ldw < K || ldy < N || (residual && ldr < N) || (pre && ldpre < N))
        return bad_arg(what, "row stride smaller than a row");
    const ForwardPlan plan(M, N, K, dtype, lie_of(x, ldx, K, dtype), lie_of(W, ldw, K, dtype));
    Copies copies;
    const void *px = x, *pw = W;
    int64_t lx = ldx, lw = ldw;
    if (plan.tiled) {
        copies.take(px, lx, M, K, static_cast<uint8_t*>(workspace) + plan.parts);
        copies.take(pw, lw, N, K, static_cast<uint8_t*>(workspace) + plan.parts);
    }
    if (int rc = check_workspace(what, workspace, workspace_bytes, plan.parts + copies.bytes)) return rc;
    if (M == 0 || N == 0) return NFLOW_OK;
    if (!y) return bad_arg(what, "null y");
    if (K > 0 && (!x || !W)) return bad_arg(what, "null x or W");
    const size_t e = dtype_size(dtype);
    const Span sx(x, M, K, ldx, e), sw(W, N, K, ldw, e), sr(residual, M, N, ldr, e), sy(y, M, N, ldy, e), sp(pre, M, N, ldpre, e);
    const Span sb(bias, N, sizeof(float));
    for (const Span& m : {sx, sw, sb})
        if (meet(m, sy) || meet(m, sp)) return bad_arg(what, kShared);
    if (meet(sy, sp) || meet(sr, sp) ||
        (residual && rows_clash(residual, ldr, y, ldy, M, N, e)))
        return bad_arg(what, kShared);
    hipStream_t st = as_stream(stream);
    if (copies.n) launch_dense_pack(copies.m, st);
    const DenseArgs a{px, pw, lx, lw, M, N, K, bias, residual, ldr, activation, y, ldy, pre, ldpre, nullptr};
    return product(what, DENSE_FORWARD, plan.p, a, dtype, workspace, st);
}

int nflow_dense_linear_backward_workspace(int64_t M, int64_t N, int64_t K, int dtype, int copies, size_t* bytes) {
    clear_error();
    const char* what = "dense_linear_backward_workspace";
    if (!bytes) return bad_arg(what, "null output");
    *bytes = 0;
    if (int rc = check_sizes(what, M, N, K, dtype)) return rc;
    *bytes = BackwardPlan(M, N, K, dtype).bytes;
    if (copies && dtype == NFLOW_DTYPE_BF16) *bytes += copy_space(M, N) + copy_space(N, K) + copy_space(M, K);
    return NFLOW_OK;
}

int nflow_dense_linear_backward(const void* dy, int dtype, int64_t M, int64_t N, int64_t lddy, const void* x,
                                int64_t ldx, const void* W, int64_t ldw, int64_t K, int activation, const void* pre,
                                int64_t ldpre, void* dz, int64_t lddz, void* dx, int64_t lddx, void* dW,
                                int64_t lddw, float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "dense_linear_backward";
    if (int rc = check_sizes(what, M, N, K, dtype)) return rc;
    if (int rc = check_act(what, activation)) return rc;
    const bool act = activation != NFLOW_ACT_NONE;
    if (!act && (pre || dz)) return bad_arg(what, "pre and dz are of an activation, and there is none");
    if (lddy < N || (dW && ldx < K) || (dx && ldw < K) || (act && (ldpre < N || lddz < N)) || (dx && lddx < K) ||
        (dW && lddw < K))
        return bad_arg(what, "row stride smaller than a row");
    const BackwardPlan plan(M, N, K, dtype);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    Copies copies;
    const void *g = act ? dz : dy, *px = x, *pw = W;
    int64_t lg = act ? lddz : lddy, lx = ldx, lw = ldw;
    if (dtype == NFLOW_DTYPE_BF16 && M > 0 && N > 0 && K > 0) {
        if (dx || dW) copies.take(g, lg, M, N, ws + plan.bytes);
        if (dx) copies.take(pw, lw, N, K, ws + plan.bytes);
        if (dW) copies.take(px, lx, M, K, ws + plan.bytes);
    }
    if (int rc = check_workspace(what, workspace, workspace_bytes, plan.bytes + copies.bytes)) return rc;
    if (M > 0 && N > 0) {
        if (!dy || (act && (!pre || !dz))) return bad_arg(what, "null dy, pre or dz");
        if (K > 0 && ((dx && !W) || (dW && !x))) return bad_arg(what, "null x or W");
    }
    const size_t e = dtype_size(dtype);
    const Span sdz(dz, M, N, lddz, e), sx(dW ? x : nullptr, M, K, ldx, e), sw(dx ? W : nullptr, N, K, ldw, e),
        sdx(dx, M, K, lddx, e), sdw(dW, N, K, lddw, e), sdb(dbias, N, sizeof(float));
    for (const Span& m : {sx, sw, sdz, Span(dy, M, N, lddy, e), Span(pre, M, N, ldpre, e)})
        if (meet(m, sdx) || meet(m, sdw) || meet(m, sdb)) return bad_arg(what, kShared);
    if (meet(sdx, sdw) || meet(sdx, sdb) || meet(sdw, sdb) || meet(sx, sdz) || meet(sw, sdz) ||
        (act && N > 0 && (rows_clash(dy, lddy, dz, lddz, M, N, e) || rows_clash(pre, ldpre, dz, lddz, M, N, e))))
        return bad_arg(what, kShared);
    // Every result that is wanted is empty.  (dx of no columns of dz is not: zeros.)
    if ((M == 0 || (N == 0 ? !dx : !(act || dx))) && !dW && !dbias) return NFLOW_OK;
    hipStream_t st = as_stream(stream);
    float* sums = reinterpret_cast<float*>(ws);
    const int64_t runs = dz_runs(M, N);
    // With no activation dW's product sums dz's rows on its way; dz's own launch does else.
    float* ride = !act && dW && K > 0 ? dbias : nullptr;
    if (ride) dbias = nullptr;
    if (M > 0 && N > 0 && (act || dbias)) {
        const DzArgs a{dy, pre, dz, M, N, lddy, ldpre, lddz, activation, dbias ? sums : nullptr, (M + runs - 1) / runs};
        const dim3 grid(static_cast<unsigned>((N + kDzCols - 1) / kDzCols), static_cast<unsigned>(runs));
        if (dtype == NFLOW_DTYPE_BF16) hipLaunchKernelGGL((k_dense_dz<bf16>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_dense_dz<float>), grid, dim3(256), 0, st, a);
    }
    if (dbias && N > 0)
        hipLaunchKernelGGL(k_dense_dbias, dim3(static_cast<unsigned>((N + 15) / 16)), dim3(256), 0, st, sums,
                           M > 0 ? runs : 0, N, dbias);
    if (copies.n) launch_dense_pack(copies.m, st);
    if (int rc = launch_status(what)) return rc;
    if (K == 0) return NFLOW_OK;
    const DenseArgs ax{g, pw, lg, lw, M, K, N, nullptr, nullptr, 0, NFLOW_ACT_NONE, dx, lddx, nullptr, 0, nullptr};
    const DenseArgs aw{g, px, lg, lx, N, K, M, nullptr, nullptr, 0, NFLOW_ACT_NONE, dW, lddw, nullptr, 0, ride};
    if (dx && dW && plan.pair.groups) {
        launch_dense_pair_f32(ax, aw, plan.pair, reinterpret_cast<float*>(ws + plan.sums), st);
        return launch_status(what);
    }
    if (dx)
        if (int rc = product(what, DENSE_DX, plan.x, ax, dtype, ws + plan.sums, st)) return rc;
    return dW ? product(what, DENSE_DW, plan.w, aw, dtype, ws + plan.sums + plan.x_parts, st) : NFLOW_OK;
}

int nflow_debug_dense_cut(int form, int64_t M, int64_t N, int64_t K, int dtype, int* kernel, int* groups) {
    clear_error();
    const char* what = "debug_dense_cut";
    if (!kernel || !groups) return bad_arg(what, "null output");
    if (form < 0 || form > 3) return bad_arg(what, "unknown form");
    if (int rc = check_sizes(what, M, N, K, dtype)) return rc;
    const DensePlan p = form == 3 ? BackwardPlan(M, N, K, dtype).pair : dense_plan(static_cast<DenseForm>(form), M, N, K, dtype);
    *kernel = static_cast<int>(p.kind);
    *groups = p.groups;
    return NFLOW_OK;
}

}  // extern "C"
