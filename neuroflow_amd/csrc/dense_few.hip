// dense_few.hip -- the bf16 / fp32 product for few rows: one new token, or a
// small batch of them, against a weight that is read once.
//
// A workgroup owns 16 columns and all the rows; its waves deal 128-byte pieces
// of the weight's rows out among them (wave w takes pieces w, w + W, ...),
// straight from HBM to the MFMA operand registers.  Each wave keeps fp32 sums of
// its pieces, and the workgroup joins them in LDS in the waves' order.  Rows need
// no alignment.
//
// Bound by reading the weight: one row of 4096 -> 4096 bf16 in 7.9 us a call (33.6
// MB, 4.3 TB/s), of 16384 -> 16384 105 (5.1 TB/s).  W waves so that the chip has 16
// waves a CU in all where K has the pieces; four pieces ahead took one row's 4096 ->
// 4096 from 9.7 to 7.9 us.  With more rows the rows' way from the L2, once for every 16
// columns, takes over (32 rows of 4096 -> 16384 52.7 us, one 26.7), and with few
// columns K is split over too few workgroups; where the tiles gain, dense_plan says.
#include "dense_kernel.h"
#include "dense_split.h"

namespace nfq {
namespace {

template <typename T>
constexpr int dense_planes() { return std::is_same_v<T, float> ? 3 : 1; }

// 32 k's of a row as operand planes.
template <typename T>
struct FewOperand {
    v8bf p[dense_planes<T>()];
    __device__ __forceinline__ explicit FewOperand(const Raw8<T>& v) {
        if constexpr (std::is_same_v<T, float>) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = v[e];
            dense_split(x, p);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[0][e] = v.q[e];
        }
    }
};
template <typename T>
__device__ __forceinline__ v4f few_product(const FewOperand<T>& w, const FewOperand<T>& x, v4f acc) {
    if constexpr (std::is_same_v<T, float>) {
        constexpr int pw[6] = {0, 2, 1, 0, 1, 0}, px[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
        for (int q = 0; q < 6; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[pw[q]], x.p[px[q]], acc, 0, 0, 0);
        return acc;
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[0], x.p[0], acc, 0, 0, 0);
    }
}

template <typename T, int RT, int W>
__global__ __launch_bounds__(64 * W) void k_dense_few(DenseArgs a) {
    constexpr int H = std::is_same_v<T, float> ? 1 : 2, KP = 32 * H;    // 32-k steps of a piece
    __shared__ __attribute__((aligned(16))) v4f red[W][RT][64];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
    const int pieces = static_cast<int>((a.K + KP - 1) / KP);

    v4f acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // Rows past the last (of W or of x) read row 0: their products are never stored.
    const T* wrow = static_cast<const T*>(a.B) + (n0 + r < a.N ? n0 + r : 0) * a.ldb;
    const T* xrow[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
        xrow[i] = static_cast<const T*>(a.A) + (16 * i + r < a.M ? 16 * i + r : 0) * a.lda;
    // A piece of the weight and of the rows, AHEAD of the wave's pieces in flight.
    constexpr int AHEAD = RT == 1 ? 4 : 2;
    struct Piece {
        Raw8<T> w[H], x[RT][H];
    };
    auto fetch = [&](int k, Piece& o) {
        if (k >= pieces) return;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int64_t c = static_cast<int64_t>(k) * KP + 32 * h + 8 * g;
            dense_load(o.w[h], wrow + c, a.K - c);
#pragma unroll
            for (int i = 0; i < RT; ++i) dense_load(o.x[i][h], xrow[i] + c, a.K - c);
        }
    };
    auto step = [&](const Piece& o) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const FewOperand<T> wp(o.w[h]);
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[i] = few_product<T>(wp, FewOperand<T>(o.x[i][h]), acc[i]);
        }
    };
    Piece next[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) fetch(wid + n * W, next[n]);
    for (int k = wid; k < pieces; k += AHEAD * W) {
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
            if (k + n * W < pieces) {
                step(next[n]);
                fetch(k + (n + AHEAD) * W, next[n]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) red[wid][i][lane] = acc[i];
    __syncthreads();
    for (int i = wid; i < RT; i += W) {
        v4f z = red[0][i][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) z += red[w][i][lane];
        if (16 * i + r < a.M) dense_finish<T>(a, 16 * i + r, n0 + 4 * g, z);
    }
}

template <typename T, int RT>
void launch_rt(const DenseArgs& a, hipStream_t st) {
    const int64_t groups = (a.N + 15) / 16, pieces = (a.K * static_cast<int64_t>(sizeof(T)) + 127) / 128;
    const int64_t want = std::min<int64_t>(pieces, 16 * num_cus() / std::max<int64_t>(groups, 1));
    auto go = [&](auto k, int w) { hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(groups)), dim3(64 * w), 0, st, a); };
    if (want > 8) go(k_dense_few<T, RT, 16>, 16);
    else if (want > 4) go(k_dense_few<T, RT, 8>, 8);
    else go(k_dense_few<T, RT, 4>, 4);
}

}  // namespace

template <typename T>
void launch_dense_few(const DenseArgs& a, hipStream_t st) {
    if (a.M <= 16) launch_rt<T, 1>(a, st);
    else launch_rt<T, 2>(a, st);
}
template void launch_dense_few<float>(const DenseArgs&, hipStream_t);
template void launch_dense_few<bf16>(const DenseArgs&, hipStream_t);

}  // namespace nfq
