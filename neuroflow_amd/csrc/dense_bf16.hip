// dense_bf16.hip -- the tiled product of bf16 operands.
#include "dense_kernel.h"

namespace nfq {
namespace {

using Small = DenseTile<bf16, 2, 2, 2, 2, 1>;     // 64 x 64, four waves
using Mid = DenseTile<bf16, 2, 2, 4, 4, 1>;       // 128 x 128, four waves

template <bool AX, bool BX>
void launch(const DenseArgs& a, const DensePlan& p, float* part, hipStream_t st) {
    if (p.kind == DENSE_SMALL) launch_dense_tile<bf16, AX, BX, Small>(a, p.splits, part, st);
    else launch_dense_tile<bf16, AX, BX, Mid>(a, p.splits, part, st);
}

}  // namespace

template <>
void launch_dense<bf16>(const DenseArgs& a, DenseForm form, const DensePlan& p, float* part, hipStream_t st) {
    if (form == DENSE_FORWARD) launch<false, false>(a, p, part, st);
    else if (form == DENSE_DX) launch<false, true>(a, p, part, st);
    else launch<true, true>(a, p, part, st);
}

}  // namespace nfq
