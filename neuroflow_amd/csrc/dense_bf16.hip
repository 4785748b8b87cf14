// dense_bf16.hip -- the tiled product of bf16 operands.
#include "dense_dma.h"

namespace nfq {
namespace {

using Small = DenseTile<bf16, 2, 2, 2, 2, 1>;     // 64 x 64, four waves
using Mid = DenseTile<bf16, 2, 2, 4, 4, 1>;       // 128 x 128, four waves
using DmaSmall = DenseTile<bf16, 2, 2, 2, 2, 3>;
using DmaMid = DenseTile<bf16, 2, 2, 4, 4, 2>;
using DmaBig = DenseTile<bf16, 2, 4, 8, 4, 2>;    // 256 x 256, eight waves, a workgroup per CU

// Whether the LDS-DMA can fetch an operand: whole 16-byte groups at 16-byte
// places, and a tile's rows within a buffer's range.
bool dma_ok(const void* p, int64_t ld, int64_t inner) {
    return aligned(p, 16) && ld % 8 == 0 && inner % 8 == 0 && ld < (INT64_C(1) << 21);
}

template <bool AX, bool BX>
void launch(const DenseArgs& a, const DensePlan& p, float* part, hipStream_t st) {
    if (dma_ok(a.A, a.lda, AX ? a.M : a.K) && dma_ok(a.B, a.ldb, BX ? a.N : a.K)) {
        if (p.kind == DENSE_BIG) launch_dense_tile<bf16, DmaBig, &k_dense_dma<AX, BX, DmaBig>>(a, p.splits, part, st);
        else if (p.kind == DENSE_MID) launch_dense_tile<bf16, DmaMid, &k_dense_dma<AX, BX, DmaMid>>(a, p.splits, part, st);
        else launch_dense_tile<bf16, DmaSmall, &k_dense_dma<AX, BX, DmaSmall>>(a, p.splits, part, st);
        return;
    }
    if (p.kind == DENSE_SMALL) launch_dense_tile<bf16, Small, &k_dense<bf16, AX, BX, Small>>(a, p.splits, part, st);
    else launch_dense_tile<bf16, Mid, &k_dense<bf16, AX, BX, Mid>>(a, p.splits, part, st);
}

}  // namespace

template <>
void launch_dense<bf16>(const DenseArgs& a, DenseForm form, const DensePlan& p, float* part, hipStream_t st) {
    if (form == DENSE_FORWARD) launch<false, false>(a, p, part, st);
    else if (form == DENSE_DX) launch<false, true>(a, p, part, st);
    else launch<true, true>(a, p, part, st);
}

}  // namespace nfq
