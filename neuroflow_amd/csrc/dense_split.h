// dense_split.h -- an fp32 operand as three bf16 planes (dense_f32.hip, dense_few.hip).
#pragma once

#include "common.h"

namespace nfq {

// Eight fp32 values as planes h + m + l, each the rest rounded to bf16: exact from
// 2^-110 on; below, l's rounding to a bf16 subnormal leaves out up to 2^-134.  A value
// that would round to infinity keeps bf16's largest as its first plane; of an
// infinity or a NaN the third is NaN, and so is what it is multiplied or summed into.
__device__ __forceinline__ void dense_split(const float (&v)[8], v8bf (&p)[3]) {
    constexpr float top = 0x1.fep127f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const __bf16 h = static_cast<__bf16>(__builtin_amdgcn_fmed3f(v[e], -top, top));
        const float r = v[e] - static_cast<float>(h);
        const __bf16 m = static_cast<__bf16>(r);
        p[0][e] = h;
        p[1][e] = m;
        p[2][e] = static_cast<__bf16>(r - static_cast<float>(m));
    }
}

}  // namespace nfq
