// grad_norm.hip -- the norm of many gradient tensors and their clipping by it
// (include/nflow_residual.h).
//
// The tensors are cut into chunks of kChunk elements, numbered through; a
// workgroup takes a run of them.  The first launch sums squares, a double per
// workgroup; the second sums those, in each of its workgroups, and scales.  The
// sums' order depends on the tensors' counts alone.  A table of tensors is a
// kernel's argument: nothing is copied to the device, and a captured launch
// keeps it; more tensors than a table holds take a launch each kTable.
// Squares and sums are doubles: fp32 squares leave fp32's range from 1.8e19 on,
// and the additions run under the loads.
#include <vector>

#include "block_dev.h"
#include "nflow_residual.h"

namespace nfq {
namespace {

constexpr int kThreads = 256;
constexpr int kVecs = 4;                            // loads of 8 elements a thread has in flight
constexpr int64_t kChunk = 8 * kThreads * kVecs;
constexpr int kTable = 120;                         // tensors of a launch: 28 bytes each in 4 KB of arguments
constexpr int kMaxParts = 1024;                     // workgroups, and partial sums, of the first launch

struct GradTable {
    const void* grad[kTable];
    void* out[kTable];
    int64_t count[kTable];                          // negative: bf16
    int first[kTable];                              // chunk
    int tensors, chunks, per;                       // per: chunks of a workgroup
};
static_assert(sizeof(GradTable) + 64 <= 4096, "a kernel's arguments");

// Calls f(tensor, its chunk) for the chunks of this workgroup, in their order.
template <typename F>
__device__ __forceinline__ void each_chunk(const GradTable& t, int block, F f) {
    int c = block * t.per;
    const int end = c + t.per < t.chunks ? c + t.per : t.chunks;
    if (c >= end) return;
    int lo = 0, hi = t.tensors - 1;                 // the last tensor with first <= c: none there is empty
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    for (int i = lo; c < end; ++i) {
        const int next = i + 1 < t.tensors ? t.first[i + 1] : t.chunks, stop = next < end ? next : end;
        for (; c < stop; ++c) f(i, c - t.first[i]);
    }
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}
__device__ __forceinline__ double block_sum64(double v, double* part) {
    v = wave_sum64(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* g, int64_t count, int64_t at) {
    Raw8<T> v[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int64_t c = at + 8 * (static_cast<int64_t>(threadIdx.x) + kThreads * k);
        v[k].load(g + c, count - c);
    }
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double d = static_cast<double>(v[k][e]);
            s = __builtin_fma(d, d, s);
        }
    return s;
}

__global__ __launch_bounds__(kThreads) void k_grad_squares(GradTable t, double* __restrict__ part) {
    __shared__ double red[kThreads / 64];
    double s = 0.0;
    each_chunk(t, blockIdx.x, [&](int i, int c) {
        const int64_t n = t.count[i], at = c * kChunk;
        s += n < 0 ? chunk_squares(static_cast<const bf16*>(t.grad[i]), -n, at)
                   : chunk_squares(static_cast<const float*>(t.grad[i]), n, at);
    });
    s = block_sum64(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm from the partial sums, in every thread.
__device__ __forceinline__ double total_norm(const double* __restrict__ part, int parts, double* red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
    return sqrt(block_sum64(s, red));
}

__global__ __launch_bounds__(kThreads) void k_grad_norm(const double* __restrict__ part, int parts,
                                                        float* __restrict__ norm) {
    __shared__ double red[kThreads / 64];
    const double n = total_norm(part, parts, red);
    if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* g, T* o, int64_t count, int64_t at, float f) {
    Raw8<T> v[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int64_t c = at + 8 * (static_cast<int64_t>(threadIdx.x) + kThreads * k);
        v[k].load(g + c, count - c);
    }
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int64_t c = at + 8 * (static_cast<int64_t>(threadIdx.x) + kThreads * k);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = v[k][e] * f;
        store8(o + c, count - c, y);
    }
}

__global__ __launch_bounds__(kThreads) void k_grad_scale(GradTable t, const double* __restrict__ part, int parts,
                                                         float max_norm, float* __restrict__ norm) {
    __shared__ double red[kThreads / 64];
    const double n = total_norm(part, parts, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
    // A norm that is NaN is not below: the factor is NaN then, and 0 of an infinite one.
    const bool keep = n <= static_cast<double>(max_norm);
    const float f = keep ? 1.0f : static_cast<float>(static_cast<double>(max_norm) / n);
    each_chunk(t, blockIdx.x, [&](int i, int c) {
        const int64_t k = t.count[i], at = c * kChunk;
        if (keep && t.out[i] == t.grad[i]) return;
        if (k < 0) chunk_scale(static_cast<const bf16*>(t.grad[i]), static_cast<bf16*>(t.out[i]), -k, at, f);
        else chunk_scale(static_cast<const float*>(t.grad[i]), static_cast<float*>(t.out[i]), k, at, f);
    });
}

// The tensors with elements, kTable of them a launch.
struct GradPlan {
    std::vector<GradTable> tables;
    std::vector<int> parts;                         // workgroups of each table's first launch
    int total = 0;                                  // of all
};

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

int check_grads(const char* what, const nflow_grad_tensor* tensors, int count, bool pointers) {
    if (count < 0 || (count > 0 && !tensors)) return bad_arg(what, "bad table of tensors");
    int64_t all = 0;
    for (int i = 0; i < count; ++i) {
        const nflow_grad_tensor& t = tensors[i];
        if (!dtype_ok(t.dtype)) return bad_arg(what, "unknown dtype");
        if (t.count < 0) return bad_arg(what, "bad count");
        if (pointers && t.count > 0 && !t.grad) return bad_arg(what, "null gradient");
        all += chunks_of(t.count);
        if (all > INT32_MAX / 2) return bad_arg(what, "too many elements for one call");
    }
    return NFLOW_OK;
}

// Whether memory that is written shares a byte with another tensor's, or an out
// with its own grad in another way than as the same memory: by their places in order.
bool tangled(const nflow_grad_tensor* tensors, int count) {
    struct Span {
        uintptr_t from, to;
        bool written;
    };
    std::vector<Span> spans;
    spans.reserve(2 * static_cast<size_t>(count));
    for (int i = 0; i < count; ++i) {
        const nflow_grad_tensor& t = tensors[i];
        const uintptr_t n = static_cast<uintptr_t>(t.count) * dtype_size(t.dtype);
        if (n == 0) continue;
        const auto g = reinterpret_cast<uintptr_t>(t.grad), o = reinterpret_cast<uintptr_t>(t.out);
        spans.push_back({o, o + n, true});
        if (o != g) spans.push_back({g, g + n, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
    uintptr_t any = 0, written = 0;                 // ends of what came before
    for (const Span& s : spans) {
        if (s.from < (s.written ? any : written)) return true;
        any = std::max(any, s.to);
        if (s.written) written = std::max(written, s.to);
    }
    return false;
}

void seal(GradTable& t, GradPlan& p) {
    const int blocks = std::min(t.chunks, kMaxParts);
    t.per = (t.chunks + blocks - 1) / blocks;
    p.parts.push_back((t.chunks + t.per - 1) / t.per);
    p.total += p.parts.back();
    p.tables.push_back(t);
}

GradPlan grad_plan(const nflow_grad_tensor* tensors, int count) {
    GradPlan p;
    GradTable t{};
    for (int i = 0; i < count; ++i) {
        const nflow_grad_tensor& g = tensors[i];
        if (g.count == 0) continue;
        const int k = t.tensors++;
        t.grad[k] = g.grad;
        t.out[k] = g.out;
        t.count[k] = g.dtype == NFLOW_DTYPE_BF16 ? -g.count : g.count;
        t.first[k] = t.chunks;
        t.chunks += static_cast<int>(chunks_of(g.count));
        if (t.tensors == kTable) {
            seal(t, p);
            t = GradTable{};
        }
    }
    if (t.tensors) seal(t, p);
    return p;
}

size_t grad_space_of(const GradPlan& p) { return round16(static_cast<size_t>(p.total) * sizeof(double)); }

void launch_squares(const GradPlan& p, double* part, hipStream_t st) {
    for (size_t i = 0; i < p.tables.size(); ++i) {
        hipLaunchKernelGGL(k_grad_squares, dim3(p.parts[i]), dim3(kThreads), 0, st, p.tables[i], part);
        part += p.parts[i];
    }
}

template <typename F>
int guarded(const char* what, F f) {
    try {
        return f();
    } catch (const std::exception& e) {
        return set_error(NFLOW_INTERNAL, std::string(what) + ": " + e.what());
    }
}

}  // namespace
}  // namespace nfq

using namespace nfq;

extern "C" {

int nflow_grad_workspace(const nflow_grad_tensor* tensors, int count, size_t* bytes) {
    clear_error();
    const char* what = "grad_workspace";
    if (!bytes) return bad_arg(what, "null output");
    *bytes = 0;
    if (int rc = check_grads(what, tensors, count, false)) return rc;
    return guarded(what, [&] {
        *bytes = grad_space_of(grad_plan(tensors, count));
        return static_cast<int>(NFLOW_OK);
    });
}

int nflow_grad_norm(const nflow_grad_tensor* tensors, int count, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "grad_norm";
    if (int rc = check_grads(what, tensors, count, true)) return rc;
    if (!norm) return bad_arg(what, "null norm");
    return guarded(what, [&] {
        const GradPlan p = grad_plan(tensors, count);
        if (int rc = check_workspace(what, workspace, workspace_bytes, grad_space_of(p))) return rc;
        double* part = static_cast<double*>(workspace);
        launch_squares(p, part, as_stream(stream));
        hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(kThreads), 0, as_stream(stream), part, p.total, norm);
        return launch_status(what);
    });
}

int nflow_grad_clip(const nflow_grad_tensor* tensors, int count, float max_norm, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "grad_clip";
    if (int rc = check_grads(what, tensors, count, true)) return rc;
    if (!norm) return bad_arg(what, "null norm");
    if (!(max_norm >= 0.0f)) return bad_arg(what, "max_norm must not be negative or NaN");
    for (int i = 0; i < count; ++i)
        if (tensors[i].count > 0 && !tensors[i].out) return bad_arg(what, "null out");
    return guarded(what, [&] {
        if (tangled(tensors, count)) return bad_arg(what, "an out overlaps a gradient or another out");
        const GradPlan p = grad_plan(tensors, count);
        if (int rc = check_workspace(what, workspace, workspace_bytes, grad_space_of(p))) return rc;
        double* part = static_cast<double*>(workspace);
        hipStream_t st = as_stream(stream);
        launch_squares(p, part, st);
        if (p.tables.empty())
            hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(kThreads), 0, st, part, 0, norm);
        for (size_t i = 0; i < p.tables.size(); ++i)
            hipLaunchKernelGGL(k_grad_scale, dim3(p.parts[i]), dim3(kThreads), 0, st, p.tables[i], part, p.total, max_norm,
                               i == 0 ? norm : nullptr);
        return launch_status(what);
    });
}

}  // extern "C"
