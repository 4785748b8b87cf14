// block_gemm.hip -- the product of 128-block FP8 codes and the linear layer
// around it, forward and backward (include/nflow_block.h).
#include <cmath>

#include "block_gemm_kernel.h"

namespace nfq {
namespace {

// out[n] = the sum of part (P, N) over P, in an order that depends on P alone:
// 16 columns a workgroup, every sixteenth part a thread, the threads' sums in turn.
struct PartSums {
    const float* part;
    int64_t P, N;
    float* out;
    __host__ __device__ int blocks() const { return out ? static_cast<int>((N + 15) / 16) : 0; }
};
__device__ __forceinline__ void sum_parts(const PartSums& a, int blk) {
    __shared__ float s[16][17];
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int64_t n = static_cast<int64_t>(blk) * 16 + c;
    float v = 0.0f;
    if (n < a.N) {
#pragma unroll 8
        for (int64_t p = g; p < a.P; p += 16) v += a.part[p * a.N + n];
    }
    s[g][c] = v;
    __syncthreads();
    if (g == 0 && n < a.N) {
        float z = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) z += s[k][c];
        a.out[n] = z;
    }
}
__global__ __launch_bounds__(256) void k_sum_parts(PartSums a) { sum_parts(a, blockIdx.x); }

// Sum of the splits' partial results, in their order, and the epilogue.  The
// first workgroups take `sums`, which are a few latencies long and would cost a
// launch of their own (4 to 5 us).  Bound by the partial results' bytes, most of
// them from L2 and the Infinity Cache.
template <typename TO>
__global__ __launch_bounds__(256) void k_block_gemm_join(BlockGemmArgs a, const float* __restrict__ part, int splits,
                                                         PartSums sums) {
    const int first = sums.blocks();
    if (static_cast<int>(blockIdx.x) < first) {
        sum_parts(sums, blockIdx.x);
        return;
    }
    const int64_t n4 = (a.N + 3) / 4, total = a.M * n4;
    const bool vec = a.ldc % 4 == 0 && (reinterpret_cast<uintptr_t>(a.C) & (4 * sizeof(TO) - 1)) == 0;
    const bool vin = a.N % 4 == 0;
    for (int64_t i = static_cast<int64_t>(blockIdx.x - first) * 256 + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x - first) * 256) {
        const int64_t m = i / n4, n = (i - m * n4) * 4;
        v4f z{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < splits; ++s) {
            const float* p = part + (s * a.M + m) * a.N + n;
            if (vin) {
                const v4f q = *reinterpret_cast<const v4f*>(p);
#pragma unroll
                for (int v = 0; v < 4; ++v) z[v] += q[v];
            } else {
                for (int v = 0; v < 4; ++v)
                    if (n + v < a.N) z[v] += p[v];
            }
        }
        store4<TO>(a, m, n, z, vec);
    }
}

using TileBig = BlockTile<2, 4, 8, 4, 2>;     // 256 x 256, eight waves, a workgroup per CU
using TileMid = BlockTile<2, 2, 4, 4, 2>;     // 128 x 128, four waves, two workgroups per CU
using TileSmall = BlockTile<2, 2, 2, 2, 4>;   // 64 x 64, four waves, two workgroups per CU, loads three steps ahead

template <typename T>
GemmShare gemm_share(const BlockGemmArgs& a, int splits, float* part) {
    const int64_t tm = (a.M + T::BM - 1) / T::BM, tn = (a.N + T::BN - 1) / T::BN;
    const int kb = static_cast<int>(blk_count(a.K));
    return GemmShare{tm, tn, splits, (kb + splits - 1) / splits, part, static_cast<int>(tm * tn * splits)};
}

// A kernel with T's stages as its dynamic LDS.
template <typename T, auto k, typename... Args>
void launch_staged(int blocks, hipStream_t st, Args... args) {
    constexpr int bytes = T::NS * T::STAGE;
    static const hipError_t once =
        hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    (void)once;
    hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(blocks)), dim3(T::THREADS), bytes, st, args...);
}

template <typename TO, bool BLOCKS, typename T>
void launch_tiles(const BlockGemmArgs& a, int splits, float* part, hipStream_t st) {
    const GemmShare sh = gemm_share<T>(a, splits, part);
    launch_staged<T, &k_block_gemm<TO, BLOCKS, T>>(sh.blocks, st, a, sh);
}

template <typename TO>
void launch_join(const BlockGemmArgs& a, int splits, const float* part, const PartSums& sums, hipStream_t st) {
    if (splits > 1)
        hipLaunchKernelGGL((k_block_gemm_join<TO>), dim3(sums.blocks() + grid_for(a.M * ((a.N + 3) / 4), 256, 8)),
                           dim3(256), 0, st, a, part, splits, sums);
    else if (sums.out)
        hipLaunchKernelGGL(k_sum_parts, dim3(sums.blocks()), dim3(256), 0, st, sums);
}

// How a product is cut: the kernel or tile, and the number of runs of K blocks
// that its tiles are split into (joined by a second launch).
enum GemmKind { GEMM_FEW, GEMM_SMALL, GEMM_MID, GEMM_BIG };
struct GemmPlan {
    GemmKind kind;
    int splits;
    size_t bytes;       // of the partial results
};

// The cut with the least estimated time, in us.  With n workgroups on the
// busiest CU a K block costs each tile max(alone, n each): alone is what one
// workgroup takes for it by itself (its loads' latency), each what a further
// one adds.  Fitted to MI355X times at 65 to 2048 rows and (N, K) from 1024 to
// 8192, where the cut it picks is within 10% of the best of 15: e.g. bf16 4096 x
// 4096 at 256 rows 22.0 -> 15.2 us by 64 x 64 tiles in place of 128 x 128 ones
// in 8 splits, 1024 x 1024 at 1024 rows 15.7 -> 8.8 us unsplit; at 2048 rows
// 128 x 128 tiles are ahead of 64 x 64, 39 against 68 us, and of 256 x 256, 39
// against 52 us, which win from one for every CU on (8192 x 8192 x 8192 460
// against 560 us).  A split pays a launch and its partial results' way through
// the caches; the few-row kernel a CU's rate of reading fragments from L2
// (36 GB/s), or the weight's from HBM.  Outside those sizes the estimate orders
// the cuts but is no time: it has no term for a tile's fill and stores (65536 x
// 1024 x 1024 bf16 estimated 56 us, measured 82), and 16 splits are its most,
// however many CUs a small result leaves idle.
GemmPlan gemm_plan(int64_t M, int64_t N, int64_t K, int out) {
    const bool f32 = out == NFLOW_DTYPE_F32;
    const double cus = num_cus(), kb = static_cast<double>(blk_count(K)), m = static_cast<double>(M),
                 n = static_cast<double>(N);
    struct Cut {
        GemmKind kind;
        double edge, alone, each;
    };
    const Cut cuts[] = {{GEMM_SMALL, 64, f32 ? 0.50 : 0.35, f32 ? 0.39 : 0.25},
                        {GEMM_MID, 128, f32 ? 1.08 : 0.72, f32 ? 0.90 : 0.54},
                        {GEMM_BIG, 256, 1.75, 1.75}};
    GemmPlan best{GEMM_MID, 1, 0};
    double least = HUGE_VAL;
    if (M <= 64) {
        const double groups = std::ceil(n / 16), per_cu = std::ceil(groups / cus), rows = 16 + m;
        least = std::max(n * kb * kBlk / 5.2e6, per_cu * kb * kBlk * rows / 36e3);
        best.kind = GEMM_FEW;
    }
    for (const Cut& c : cuts) {
        if (c.kind == GEMM_BIG && f32) continue;        // its accumulators and operands do not fit the registers
        const double tiles = std::ceil(m / c.edge) * std::ceil(n / c.edge);
        for (int s = 1; s <= 16 && (s == 1 || 2 * s <= kb); s *= 2) {
            const double per = std::ceil(tiles * s / cus), steps = std::ceil(kb / s);
            const double t = steps * std::max(c.alone, per * c.each) + (s > 1 ? 5.0 + s * m * n * 8 / 8e6 : 0.0);
            if (t < least) {
                least = t;
                best = GemmPlan{c.kind, s, s > 1 ? static_cast<size_t>(s) * M * N * sizeof(float) : 0};
            }
        }
    }
    return best;
}

template <typename TO, bool BLOCKS>
void launch_gemm(const BlockGemmArgs& a, const GemmPlan& p, float* part, const PartSums& sums, hipStream_t st) {
    if constexpr (std::is_same_v<TO, bf16>) {
        if (p.kind == GEMM_BIG) launch_tiles<TO, BLOCKS, TileBig>(a, p.splits, part, st);
    }
    if (p.kind == GEMM_MID) launch_tiles<TO, BLOCKS, TileMid>(a, p.splits, part, st);
    if (p.kind == GEMM_SMALL) launch_tiles<TO, BLOCKS, TileSmall>(a, p.splits, part, st);
    launch_join<TO>(a, p.splits, part, sums, st);
}

// a's product, and on its way `sums`, which its caller has asked for.
int block_gemm(const char* what, const BlockGemmArgs& a, void* ws, hipStream_t st, const PartSums& sums = {}) {
    if (a.M == 0 || a.N == 0) {
        if (!sums.out) return NFLOW_OK;
        launch_join<float>(a, 1, nullptr, sums, st);
        return launch_status(what);
    }
    const GemmPlan p = gemm_plan(a.M, a.N, a.K, a.out);
    if (p.kind == GEMM_FEW) {
        launch_block_few(a, st);
        launch_join<float>(a, 1, nullptr, sums, st);
        return launch_status(what);
    }
    float* part = static_cast<float*>(ws);
    if (a.out == NFLOW_DTYPE_BF16) {
        if (a.w_blocks) launch_gemm<bf16, true>(a, p, part, sums, st);
        else launch_gemm<bf16, false>(a, p, part, sums, st);
    } else {
        if (a.w_blocks) launch_gemm<float, true>(a, p, part, sums, st);
        else launch_gemm<float, false>(a, p, part, sums, st);
    }
    return launch_status(what);
}

// The two products of the fp32 backward pass, a (row scales) and b (block
// scales), in one launch where both take 128 x 128 tiles.
int block_gemm_both(const char* what, const BlockGemmArgs& a, const BlockGemmArgs& b, void* ws_a, void* ws_b,
                    hipStream_t st, const PartSums& sums) {
    if (a.M > 0 && a.N > 0 && b.M > 0 && b.N > 0 && a.out == NFLOW_DTYPE_F32 && b.out == NFLOW_DTYPE_F32) {
        const GemmPlan pa = gemm_plan(a.M, a.N, a.K, a.out), pb = gemm_plan(b.M, b.N, b.K, b.out);
        if (pa.kind == GEMM_MID && pb.kind == GEMM_MID) {
            float *fa = static_cast<float*>(ws_a), *fb = static_cast<float*>(ws_b);
            const GemmShare sa = gemm_share<TileMid>(a, pa.splits, fa), sb = gemm_share<TileMid>(b, pb.splits, fb);
            launch_staged<TileMid, &k_block_gemm_pair<TileMid>>(sa.blocks + sb.blocks, st, a, sa, b, sb);
            launch_join<float>(a, pa.splits, fa, sums, st);
            launch_join<float>(b, pb.splits, fb, PartSums{}, st);
            return launch_status(what);
        }
    }
    if (int rc = block_gemm(what, a, ws_a, st, sums)) return rc;
    return block_gemm(what, b, ws_b, st);
}

// What linear runs: a kernel that takes x's values, for few rows or for many
// rows of few K blocks, or the quantise and the product.
enum LinearKind { LINEAR_FEW, LINEAR_ROWS, LINEAR_CODES };
LinearKind linear_kind(int64_t M, int64_t N, int64_t K, int dtype) {
    if (few_values(M, K) && gemm_plan(M, N, K, dtype).kind == GEMM_FEW) return LINEAR_FEW;
    return many_rows_values(M, N, K, dtype) ? LINEAR_ROWS : LINEAR_CODES;
}

int check_gemm(const char* what, const BlockGemmArgs& a) {
    if (!dtype_ok(a.out)) return bad_arg(what, "unknown dtype");
    if (a.M < 0 || a.N < 0 || a.K < 0) return bad_arg(what, "bad dims");
    if (a.K > NFLOW_BLOCK_MAX_K) return bad_arg(what, "a product over more than NFLOW_BLOCK_MAX_K columns");
    if (a.act != NFLOW_ACT_NONE && a.act != NFLOW_ACT_RELU && a.act != NFLOW_ACT_GELU_TANH)
        return bad_arg(what, "unknown activation");
    if (a.ldc < a.N) return bad_arg(what, "row stride smaller than a row");
    if (a.M == 0 || a.N == 0) return NFLOW_OK;
    if (((a.M + 63) / 64) * ((a.N + 63) / 64) > INT32_MAX / 16) return bad_arg(what, "too many results for one launch");
    if (!a.C) return bad_arg(what, "null output");
    if (a.K > 0 && (!a.A || !a.sA || !a.W || !a.sW)) return bad_arg(what, "null codes or scales");
    if (!aligned(a.A, 16) || !aligned(a.W, 16)) return bad_arg(what, "codes must be 16-byte aligned");
    return NFLOW_OK;
}

// The codes and scales of a (rows, cols) matrix in a workspace.
struct BlockSpace {
    size_t codes, scales;
    BlockSpace(int64_t rows, int64_t cols)
        : codes(static_cast<size_t>(rows) * blk_count(cols) * kBlk),
          scales(round16(static_cast<size_t>(rows) * blk_count(cols) * sizeof(float))) {}
    size_t bytes() const { return codes + scales; }
};

size_t matmul_space(int64_t M, int64_t N, int64_t K, int out) {
    return M > 0 && N > 0 ? gemm_plan(M, N, K, out).bytes : 0;
}
// Room for x's codes past a few rows, also at the sizes whose kernel does
// without: which kernel serves a size is then no part of the interface.
size_t linear_space(int64_t M, int64_t N, int64_t K, int dtype) {
    if (M == 0 || N == 0 || linear_kind(M, N, K, dtype) == LINEAR_FEW) return 0;
    return BlockSpace(M, K).bytes() + matmul_space(M, N, K, dtype);
}
struct BackwardSpace {
    BlockSpace rows, cols;
    size_t sums, part_w, part_x;
    BackwardSpace(int64_t M, int64_t N, int64_t K, int dtype)
        : rows(M, N), cols(N, M), sums(round16(static_cast<size_t>(blk_count(M) * N) * sizeof(float))),
          part_w(round16(matmul_space(N, K, M, NFLOW_DTYPE_F32))), part_x(round16(matmul_space(M, K, N, dtype))) {}
    size_t bytes() const { return rows.bytes() + cols.bytes() + sums + part_w + part_x; }
};

// Sizes and type ahead of anything that is worked out from them; *bytes = 0.
int check_sizes(const char* what, int64_t M, int64_t N, int64_t K, int dtype, size_t* bytes) {
    if (!bytes) return bad_arg(what, "null output");
    *bytes = 0;
    if (M < 0 || N < 0 || K < 0) return bad_arg(what, "bad dims");
    if (!dtype_ok(dtype)) return bad_arg(what, "unknown dtype");
    return NFLOW_OK;
}

}  // namespace
}  // namespace nfq

using namespace nfq;

extern "C" {

int nflow_fp8_block_matmul_workspace(int64_t M, int64_t N, int64_t K, int c_dtype, size_t* bytes) {
    clear_error();
    if (int rc = check_sizes("fp8_block_matmul_workspace", M, N, K, c_dtype, bytes)) return rc;
    *bytes = matmul_space(M, N, K, c_dtype);
    return NFLOW_OK;
}

int nflow_fp8_block_matmul(const uint8_t* A, const float* scale_A, const uint8_t* W, const float* scale_W,
                           int w_blocks, int64_t M, int64_t N, int64_t K, const float* bias, int activation,
                           void* C, int c_dtype, int64_t ldc, void* workspace, size_t workspace_bytes,
                           void* stream) {
    clear_error();
    const char* what = "fp8_block_matmul";
    const BlockGemmArgs a{A, scale_A, W, scale_W, w_blocks != 0, M, N, K, bias, activation, C, c_dtype, ldc};
    if (int rc = check_gemm(what, a)) return rc;
    if (int rc = check_workspace(what, workspace, workspace_bytes, matmul_space(M, N, K, c_dtype))) return rc;
    return block_gemm(what, a, workspace, as_stream(stream));
}

int nflow_fp8_block_linear_workspace(int64_t M, int64_t N, int64_t K, int dtype, size_t* bytes) {
    clear_error();
    if (int rc = check_sizes("fp8_block_linear_workspace", M, N, K, dtype, bytes)) return rc;
    *bytes = linear_space(M, N, K, dtype);
    return NFLOW_OK;
}

int nflow_fp8_block_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* W,
                           const float* scale_W, int64_t N, const float* bias, int activation, void* y,
                           int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "fp8_block_linear";
    size_t need = 0;
    if (int rc = check_sizes(what, M, N, K, dtype, &need)) return rc;
    if (int rc = check_workspace(what, workspace, workspace_bytes, linear_space(M, N, K, dtype))) return rc;
    if (ldx < K) return bad_arg(what, "row stride smaller than a row");
    // The codes the product reads: none where it quantises by itself.
    const LinearKind kind = linear_kind(M, N, K, dtype);
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    const BlockSpace xs(M, K);
    float* scales = reinterpret_cast<float*>(codes + xs.codes);
    BlockGemmArgs a{codes, scales, W, scale_W, true, M, N, K, bias, activation, y, dtype, ldy};
    if (kind != LINEAR_CODES) {
        a.A = W;            // not read; check_gemm wants the operands' pointers
        a.sA = scale_W;
    }
    if (int rc = check_gemm(what, a)) return rc;
    if (M == 0 || N == 0) return NFLOW_OK;
    if (K > 0 && !x) return bad_arg(what, "null x");
    if (kind != LINEAR_CODES) {
        if (kind == LINEAR_FEW) launch_block_few_values(a, x, ldx, as_stream(stream));
        else launch_block_rows(a, x, ldx, as_stream(stream));
        return launch_status(what);
    }
    if (K > 0)
        if (int rc = block_quantise(what, x, dtype, M, K, ldx, codes, scales, nullptr, nullptr, nullptr, as_stream(stream)))
            return rc;
    return block_gemm(what, a, codes + xs.bytes(), as_stream(stream));
}

int nflow_fp8_block_linear_backward_workspace(int64_t M, int64_t N, int64_t K, int dtype, size_t* bytes) {
    clear_error();
    if (int rc = check_sizes("fp8_block_linear_backward_workspace", M, N, K, dtype, bytes)) return rc;
    *bytes = BackwardSpace(M, N, K, dtype).bytes();
    return NFLOW_OK;
}

int nflow_fp8_block_linear_backward(const void* dy, int dtype, int64_t M, int64_t N, int64_t lddy,
                                    const uint8_t* x_t, const float* scale_x_t, const uint8_t* W_t,
                                    const float* scale_W_t, int64_t K, void* dx, int64_t lddx, float* dW,
                                    float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "fp8_block_linear_backward";
    size_t need = 0;
    if (int rc = check_sizes(what, M, N, K, dtype, &need)) return rc;
    const BackwardSpace sp(M, N, K, dtype);
    if (int rc = check_workspace(what, workspace, workspace_bytes, sp.bytes())) return rc;
    if (lddy < N) return bad_arg(what, "row stride smaller than a row");
    if (M > 0 && N > 0 && !dy) return bad_arg(what, "null dy");
    hipStream_t st = as_stream(stream);
    // dy's codes and scales along its rows and its columns, the sums of 128 of
    // its rows, the partial results of dW and of dx.
    uint8_t* q = static_cast<uint8_t*>(workspace);
    float* sq = reinterpret_cast<float*>(q + sp.rows.codes);
    uint8_t* t = q + sp.rows.bytes();
    float* stt = reinterpret_cast<float*>(t + sp.cols.codes);
    float* sums = reinterpret_cast<float*>(t + sp.cols.bytes());
    uint8_t* part_w = t + sp.cols.bytes() + sp.sums;
    uint8_t* part_x = part_w + sp.part_w;
    const BlockGemmArgs ax{q, sq, W_t, scale_W_t, true, M, K, N, nullptr, NFLOW_ACT_NONE, dx, dtype, lddx};
    const BlockGemmArgs aw{t, stt, x_t, scale_x_t, false, N, K, M, nullptr, NFLOW_ACT_NONE, dW, NFLOW_DTYPE_F32, K};
    if (dx)
        if (int rc = check_gemm(what, ax)) return rc;
    if (dW)
        if (int rc = check_gemm(what, aw)) return rc;
    if (M > 0 && N > 0 && (dx || dW || dbias))
        if (int rc = block_quantise(what, dy, dtype, M, N, lddy, dx ? q : nullptr, dx ? sq : nullptr,
                                    dW ? t : nullptr, dW ? stt : nullptr, dbias ? sums : nullptr, st))
            return rc;
    const PartSums bias{sums, blk_count(M), N, N > 0 ? dbias : nullptr};
    if (dx && dW) return block_gemm_both(what, aw, ax, part_w, part_x, st, bias);
    return dx ? block_gemm(what, ax, part_x, st, bias)
              : dW ? block_gemm(what, aw, part_w, st, bias) : block_gemm(what, BlockGemmArgs{}, nullptr, st, bias);
}

int nflow_debug_fp8_block_cut(int64_t M, int64_t N, int64_t K, int c_dtype, int* edge, int* splits) {
    clear_error();
    const char* what = "debug_fp8_block_cut";
    if (!edge || !splits) return bad_arg(what, "null output");
    size_t bytes = 0;
    if (int rc = check_sizes(what, M, N, K, c_dtype, &bytes)) return rc;
    const GemmPlan p = gemm_plan(M, N, K, c_dtype);
    *edge = p.kind == GEMM_FEW ? 0 : p.kind == GEMM_SMALL ? TileSmall::BM : p.kind == GEMM_MID ? TileMid::BM : TileBig::BM;
    *splits = p.splits;
    return NFLOW_OK;
}

int nflow_debug_fp8_block_linear_kernel(int64_t M, int64_t N, int64_t K, int dtype, int* kernel, int* workgroups) {
    clear_error();
    const char* what = "debug_fp8_block_linear_kernel";
    if (!kernel || !workgroups) return bad_arg(what, "null output");
    size_t bytes = 0;
    if (int rc = check_sizes(what, M, N, K, dtype, &bytes)) return rc;
    const LinearKind kind = linear_kind(M, N, K, dtype);
    *kernel = static_cast<int>(kind);
    *workgroups = kind == LINEAR_ROWS && N > 0 ? static_cast<int>(block_rows_grid(M, N)) : 0;
    return NFLOW_OK;
}

}  // extern "C"
