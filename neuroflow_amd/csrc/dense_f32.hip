// dense_f32.hip -- the tiled product of fp32 operands.
#include "dense_kernel.h"

namespace nfq {
namespace {

using Small = DenseTile<float, 2, 2, 2, 2, 1>;     // 64 x 64, four waves
using Mid = DenseTile<float, 2, 2, 4, 4, 1>;       // 128 x 128, four waves

template <bool AX, bool BX>
void launch(const DenseArgs& a, const DensePlan& p, float* part, hipStream_t st) {
    if (p.kind == DENSE_SMALL) launch_dense_tile<float, Small, &k_dense<float, AX, BX, Small>>(a, p.splits, part, st);
    else launch_dense_tile<float, Mid, &k_dense<float, AX, BX, Mid>>(a, p.splits, part, st);
}

}  // namespace

template <>
void launch_dense<float>(const DenseArgs& a, DenseForm form, const DensePlan& p, float* part, hipStream_t st) {
    if (form == DENSE_FORWARD) launch<false, false>(a, p, part, st);
    else if (form == DENSE_DX) launch<false, true>(a, p, part, st);
    else launch<true, true>(a, p, part, st);
}

}  // namespace nfq
