// dense_bf16.hip -- the tiled product of bf16 operands: its tiles, and the copies
// of operands that the LDS-DMA cannot fetch.
#include "dense_dma.h"

namespace nfq {
namespace {

// A larger tile reads its operands fewer times and has more products to each LDS read,
// a smaller one leaves fewer CUs idle; two workgroups a CU hide one's start and stores
// under the other's products, four stages in LDS what one's loads take.  dense_plan
// chooses by the time of a K step, measured with each.
using Small = DenseTile<bf16, 2, 2, 2, 2, 3, 3>;    // 64 x 64, four waves, three workgroups a CU
using Mid = DenseTile<bf16, 2, 2, 4, 4, 2>;         // 128 x 128, four waves, two workgroups a CU
using Tall = DenseTile<bf16, 2, 2, 4, 2, 3>;        // 128 x 64, four waves, two workgroups a CU
using Deep = DenseTile<bf16, 2, 4, 4, 2, 4>;        // 128 x 128, eight waves, a workgroup a CU, loads three stages ahead
using Big = DenseTile<bf16, 2, 4, 8, 4, 2>;         // 256 x 256, eight waves, a workgroup a CU

template <bool AX, bool BX, bool SUMS = false>
void launch(const DenseArgs& a, const DensePlan& p, float* part, hipStream_t st) {
    if (p.kind == DENSE_BIG) launch_dense_tile<bf16, Big, &k_dense_dma<AX, BX, SUMS, Big>>(a, p, part, st);
    else if (p.kind == DENSE_TALL) launch_dense_tile<bf16, Tall, &k_dense_dma<AX, BX, SUMS, Tall>>(a, p, part, st);
    else if (p.kind == DENSE_DEEP) launch_dense_tile<bf16, Deep, &k_dense_dma<AX, BX, SUMS, Deep>>(a, p, part, st);
    else if (p.kind == DENSE_MID) launch_dense_tile<bf16, Mid, &k_dense_dma<AX, BX, SUMS, Mid>>(a, p, part, st);
    else launch_dense_tile<bf16, Small, &k_dense_dma<AX, BX, SUMS, Small>>(a, p, part, st);
}

// Eight values moved down by n, zeros after them.
__device__ __forceinline__ Raw8<bf16>::vec values_down(const Raw8<bf16>::vec& v, int n) {
    union {
        Raw8<bf16>::vec v;
        uint64_t u[2];
    } x{v};
    if (n >= 4) {
        x.u[0] = x.u[1];
        x.u[1] = 0;
        n -= 4;
    }
    if (n > 0) {
        x.u[0] = x.u[0] >> (16 * n) | x.u[1] << (64 - 16 * n);
        x.u[1] >>= 16 * n;
    }
    return x.v;
}

// Up to three matrices copied to rows of dense_pitch(cols) values, zero past
// cols: a wave takes 512 columns of four rows, 16 bytes a lane.  Bound by a load's way
// and a store's: 1537 x 2021 and 1001 x 2021 (21 MB in all) 9 us under a trace.  With
// it the layer of these takes 30 us a call; by way of registers to LDS, without, 42.
struct PackArgs {
    DensePack m[3];
    int64_t first[3];       // group of four rows of each matrix
    int64_t groups;
};
__global__ __launch_bounds__(256) void k_dense_pack(PackArgs a) {
    int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (; id < a.groups; id += static_cast<int64_t>(gridDim.x) * 4) {
        const int w = id < a.first[1] ? 0 : id < a.first[2] ? 1 : 2;
        const DensePack& m = a.m[w];
        const int64_t row = 4 * (id - a.first[w]), pitch = dense_pitch(m.cols);
        const int64_t c = static_cast<int64_t>(blockIdx.y) * 512 + 8 * (threadIdx.x & 63);
        if (c >= m.cols) continue;
        const bf16* from = static_cast<const bf16*>(m.from) + row * m.ld + c;
        bf16* to = static_cast<bf16*>(m.to) + row * pitch + c;
        // The end of a row by the eight values that end there, moved down: one load as anywhere.
        const int over = c + 8 > m.cols ? static_cast<int>(c + 8 - m.cols) : 0;
        Raw8<bf16> v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t at = row + r < m.rows ? r * m.ld : 0;
            if (m.cols >= 8) v[r].load(from + at - over, 8);
            else dense_load(v[r], from + at, m.cols - c);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (m.cols >= 8) v[r].q = values_down(v[r].q, over);
            if (row + r < m.rows) *reinterpret_cast<Raw8<bf16>::vec*>(to + r * pitch) = v[r].q;
        }
    }
}

}  // namespace

void launch_dense_pack(const DensePack (&m)[3], hipStream_t st) {
    PackArgs a;
    int64_t n = 0, cols = 0;
    for (int i = 0; i < 3; ++i) {
        cols = std::max(cols, m[i].cols);
        a.m[i] = m[i];
        a.first[i] = n;
        n += (m[i].rows + 3) / 4;
    }
    a.groups = n;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((n + 3) / 4, 1 << 20)), static_cast<unsigned>((cols + 511) / 512));
    hipLaunchKernelGGL(k_dense_pack, grid, dim3(256), 0, st, a);
}

void launch_dense_bf16(const DenseArgs& a, DenseForm form, const DensePlan& p, float* part, hipStream_t st) {
    if (form == DENSE_FORWARD) launch<false, false>(a, p, part, st);
    else if (form == DENSE_DX) launch<false, true>(a, p, part, st);
    else if (a.sums) launch<true, true, true>(a, p, part, st);
    else launch<true, true>(a, p, part, st);
}

}  // namespace nfq
