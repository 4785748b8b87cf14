// block_dev.h -- device and host helpers shared by the layer norm, the
// 128-block quantise and the block-FP8 product (include/nflow_block.h).
#pragma once

#include <cmath>
#include <string>

#include "common.h"
#include "launch.h"
#include "nflow_block.h"
#include "status.h"

namespace nfq {

constexpr int kBlk = 128;   // values per scale

__host__ __device__ constexpr int64_t blk_count(int64_t n) { return (n + kBlk - 1) / kBlk; }

// ---- element types ----------------------------------------------------------

typedef __bf16 bf16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return static_cast<T>(v); }   // bf16: nearest, ties to even

// Eight consecutive elements at p as floats, of which the first `left` exist
// (the rest are 0).  One or two 16-byte loads at any element alignment.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t left, float (&v)[8]) {
    if (left >= 8) {
        typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
        const vec q = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = to_f32(q[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? to_f32(p[e]) : 0.0f;
    }
}

// Up to eight elements in registers as they come from memory, converted where
// they are used, so that a load can be in flight meanwhile.
template <typename T>
struct Raw8 {
    typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    vec q;
    __device__ __forceinline__ void load(const T* p, int64_t left) {
        if (left >= 8) {
            q = *reinterpret_cast<const vec*>(p);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = e < left ? p[e] : T(0.0f);
        }
    }
    __device__ __forceinline__ float operator[](int e) const { return to_f32(q[e]); }
};

// Eight floats at any element alignment, rounded to T; the first `left` of them.
template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t left, const float (&v)[8]) {
    if (left >= 8) {
        typename Raw8<T>::vec q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = from_f32<T>(v[e]);
        *reinterpret_cast<typename Raw8<T>::vec*>(p) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) p[e] = from_f32<T>(v[e]);
    }
}

// The same past the caches, for results that no kernel reads soon: what the call
// still reads keeps its place there (us: RMS norm with the residual 32768 x 256
// fp32 25.9 -> 24.9, 16384 x 4096 bf16 into FP8 101.4 -> 98.5; clipping 1.3 GB 784
// -> 746).
template <typename T>
__device__ __forceinline__ void store8_stream(T* p, int64_t left, const float (&v)[8]) {
    if (left >= 8) {
        typename Raw8<T>::vec q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = from_f32<T>(v[e]);
        __builtin_nontemporal_store(q, reinterpret_cast<typename Raw8<T>::vec*>(p));
    } else {
        store8(p, left, v);
    }
}

// ---- 128-block scale ----------------------------------------------------------

// Below this a block's codes would need a subnormal scale, whose inverse
// overflows: such a block is all zero codes under scale 1.
constexpr float kBlkTiny = 448.0f * 0x1p-126f;

// The correctly rounded amax / 448 without a division: q is within an ulp of it,
// the remainder a - 448 q is exact (a multiple of 2^-143 for amax >= kBlkTiny),
// and a quotient within an ulp plus its remainder times the correctly rounded
// inverse of the divisor rounds correctly (Markstein's theorem).
__device__ __forceinline__ float blk_scale(float amax) {
    constexpr float kInv = 1.0f / 448.0f;
    const float q = amax * kInv;
    const float s = __builtin_fmaf(__builtin_fmaf(-448.0f, q, amax), kInv, q);
    return amax < kBlkTiny ? 1.0f : (amax == HUGE_VALF ? amax : s);
}

// The four bytes fp8_quant(x[e], inv) under a block's own scale.  There
// |x inv| <= 448 (1 + 2^-22), which the conversion rounds to 448, so no clamp
// is needed; the codec's cap below 2^-6 is (fp8_prerounded); and a NaN keeps
// through, its byte 0x7F or 0xFF (no number's byte) stripped of the sign.
__device__ __forceinline__ uint32_t blk_pack4(float x0, float x1, float x2, float x3, float inv) {
    auto capped = [](float v) {
        const float sub = __builtin_amdgcn_fmed3f(v, -7.0f * 0x1p-9f, 7.0f * 0x1p-9f);
        return fabsf(v) < 0x1p-6f ? sub : v;
    };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(capped(x0 * inv), capped(x1 * inv), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(capped(x2 * inv), capped(x3 * inv), w, true);
    const uint32_t u = static_cast<uint32_t>(w);
    return u & ~(((u & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u);
}

// The codes of 4 W values.  Neither the cap nor the NaN matters but where the
// plain conversion gave +-2^-6 (0x08, the only code the cap changes) or a NaN
// (0x7F); per byte c of u without signs, (c ^ 8) - 1 and c + 1 have their top
// bit set there (a borrow from a flagged byte may flag its neighbour too).  A
// wave that holds one such code goes through blk_pack4: on normal data one value
// in a hundred thousand is one, so one wave of 512 values in two hundred, and more
// where a few large values in a block leave many small ones; the rest pays 5
// instructions a word for the test where the cap and the NaN take 15.
template <int W>
__device__ __forceinline__ void blk_codes(const float (&x)[4 * W], float inv, uint32_t (&w)[W]) {
    uint32_t rare = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, c, true);
        w[i] = static_cast<uint32_t>(c);
        const uint32_t u = w[i] & 0x7F7F7F7Fu;
        rare |= ((u ^ 0x08080808u) - 0x01010101u) | (u + 0x01010101u);
    }
    if (__builtin_amdgcn_ballot_w64((rare & 0x80808080u) != 0)) [[unlikely]] {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = blk_pack4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], inv);
    }
}

typedef uint32_t v2u __attribute__((ext_vector_type(2)));
__device__ __forceinline__ v2u blk_codes8(const float (&x)[8], float inv) {
    uint32_t w[2];
    blk_codes<2>(x, inv, w);
    return v2u{w[0], w[1]};
}

// The correctly rounded 1 / s of a block's scale: the hardware's estimate is
// within an ulp, its remainder 1 - s r is exact, and one step from there rounds
// correctly (compared with the division at every mantissa of nine exponents
// over the scales' range: the same bits).  The fix-up makes 1 / inf 0.
__device__ __forceinline__ float blk_inverse(float s) {
    const float r = __builtin_amdgcn_rcpf(s);
    return __builtin_amdgcn_div_fixupf(__builtin_fmaf(__builtin_fmaf(-s, r, 1.0f), r, r), s, 1.0f);
}

// Scale and inverse of C blocks whose largest magnitudes every one of 16 lanes
// holds: lane l divides for block l % C (C a power of two), and a lane's value
// goes to the 16 by DPP, instead of 2 C divisions (a dozen instructions each) in
// every lane.
// v[l % C], a bit of l at a time by masks: a conditional of two array elements
// would send the array through LDS.
template <int C>
__device__ __forceinline__ float pick(const float (&v)[C], unsigned l) {
    if constexpr (C == 1) {
        return v[0];
    } else {
        const unsigned odd = 0u - (l & 1u);
        float h[C / 2];
#pragma unroll
        for (int k = 0; k < C / 2; ++k)
            h[k] = __uint_as_float((__float_as_uint(v[2 * k + 1]) & odd) | (__float_as_uint(v[2 * k]) & ~odd));
        return pick<C / 2>(h, l >> 1);
    }
}
template <int C, int K = 0>
__device__ __forceinline__ void spread(float v, float (&out)[C]) {
    if constexpr (K < C) {
        out[K] = dpp_mov<0x150 + K>(v);      // row_newbcast: lane K of the 16
        spread<C, K + 1>(v, out);
    }
}
template <int C>
__device__ __forceinline__ void blk_scales(const float (&amax)[C], float& own_scale, float (&inv)[C]) {
    own_scale = blk_scale(pick<C>(amax, threadIdx.x));
    spread<C>(blk_inverse(own_scale), inv);
}

// max that ignores a NaN in v (amax itself is never one).
__device__ __forceinline__ float amax_of(float amax, float v) { return fmaxf(amax, fabsf(v)); }

// ---- reductions over L lanes (16 or 64, aligned) --------------------------------
// Every lane gets the result, the same bits in each: within 16 lanes by DPP,
// then the halves of row pairs and of the wave by the permlane swaps.

struct SumOp {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct MaxOp {
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};

template <typename Op>
__device__ __forceinline__ float cross_rows(float v) {
    const unsigned u = __float_as_uint(v);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = Op::of(__uint_as_float(p[0]), __uint_as_float(p[1]));
    const unsigned w = __float_as_uint(v);
    const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return Op::of(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

template <int L, typename Op>
__device__ __forceinline__ float lanes_reduce(float v) {
    static_assert(L == 16 || L == 64, "lanes");
    v = Op::of(v, dpp_mov<0xB1>(v));     // quad_perm 1,0,3,2
    v = Op::of(v, dpp_mov<0x4E>(v));     // quad_perm 2,3,0,1
    v = Op::of(v, dpp_mov<0x141>(v));    // row_half_mirror
    v = Op::of(v, dpp_mov<0x140>(v));    // row_mirror
    if constexpr (L == 64) v = cross_rows<Op>(v);
    return v;
}
// Sum over the wave's four rows of 16 lanes.
__device__ __forceinline__ float rows_sum(float v) { return cross_rows<SumOp>(v); }
__device__ __forceinline__ float wave_sum(float v) { return lanes_reduce<64, SumOp>(v); }
__device__ __forceinline__ float wave_max(float v) { return lanes_reduce<64, MaxOp>(v); }
__device__ __forceinline__ float max16(float v) { return lanes_reduce<16, MaxOp>(v); }

// ---- checks of the entry points ----------------------------------------------------

inline bool dtype_ok(int dtype) { return dtype == NFLOW_DTYPE_F32 || dtype == NFLOW_DTYPE_BF16; }
inline size_t dtype_size(int dtype) { return dtype == NFLOW_DTYPE_BF16 ? 2 : 4; }

inline int bad_arg(const char* what, const char* why) {
    return set_error(NFLOW_INVALID_ARG, std::string(what) + ": " + why);
}

inline int launch_status(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(NFLOW_INTERNAL, std::string(what) + ": " + hipGetErrorString(e));
    return NFLOW_OK;
}

// The workspace an entry point was given against the bytes it needs.
inline int check_workspace(const char* what, const void* ws, size_t have, size_t need) {
    if (need == 0) return NFLOW_OK;
    if (!ws || have < need) return bad_arg(what, "workspace missing or smaller than its _workspace function says");
    if (!aligned(ws, 16)) return bad_arg(what, "workspace must be 16-byte aligned");
    return NFLOW_OK;
}

// Whether M rows of D elements (of `size` bytes) from a on, `lda` elements apart,
// and such rows from b on share memory in another way than row for row.  Rows at
// one stride are compared exactly, others by the memory they span.
inline bool rows_clash(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t M, int64_t D, size_t size) {
    if (M <= 0 || (a == b && (lda == ldb || M == 1))) return false;
    const auto pa = reinterpret_cast<intptr_t>(a), pb = reinterpret_cast<intptr_t>(b);
    const int64_t e = static_cast<int64_t>(size), row = D * e;
    if (pb >= pa + (M - 1) * lda * e + row || pa >= pb + (M - 1) * ldb * e + row) return false;
    if (lda != ldb || M == 1) return true;
    const int64_t step = lda * e, off = ((pb - pa) % step + step) % step;
    return off < row || off + row > step;
}

// The memory of `rows` rows of `cols` elements (of `size` bytes), `ld` elements apart;
// of a vector the one row.
struct Span {
    intptr_t p;
    int64_t rows, row, step;    // bytes of a row, and from one to the next
    Span(const void* at, int64_t rows_, int64_t cols, int64_t ld, size_t size)
        : p(reinterpret_cast<intptr_t>(at)), rows(rows_), row(cols * static_cast<int64_t>(size)),
          step(ld * static_cast<int64_t>(size)) {}
    Span(const void* at, int64_t n, size_t size) : Span(at, 1, n, n, size) {}
    bool empty() const { return !p || rows <= 0 || row <= 0; }
    intptr_t end() const { return p + (rows - 1) * step + row; }
};
// Whether two share memory.  A row, or rows at the other's stride, may lie between
// the other's rows; rows of different strides are compared by the memory they span.
inline bool meet(const Span& a, const Span& b) {
    if (a.empty() || b.empty() || b.p >= a.end() || a.p >= b.end()) return false;
    if (a.rows > 1 && b.rows > 1 && a.step != b.step) return true;
    if (a.rows == 1 && b.rows == 1) return true;
    const int64_t step = a.rows > 1 ? a.step : b.step, off = ((b.p - a.p) % step + step) % step;
    return off < a.row || off + b.row > step;
}

inline constexpr const char* kShared = "a result shares memory with an input or another result";

inline size_t round16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

}  // namespace nfq
