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
//
// HBM bound: 1.34 GB of bf16 in 60 tensors 268 us for the norm (5.0 TB/s), 690 to
// 750 by box for norm and clipping into other tensors, of which the three passes
// over the data would be 805 at a copy's rate; what is read last is read again
// first.  36 tensors of 6.3 MB: two launches, 4.6 and 6.0 us.
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

// Calls f(tensor, its chunk) for the chunks of this workgroup, first to last or,
// with BACK, last to first.
template <bool BACK, typename F>
__device__ __forceinline__ void each_chunk(const GradTable& t, F f) {
    const int begin = blockIdx.x * t.per, end = begin + t.per < t.chunks ? begin + t.per : t.chunks;
    if (begin >= end) return;
    int c = BACK ? end - 1 : begin, lo = 0, hi = t.tensors - 1;
    while (lo < hi) {                               // the last tensor with first <= c: none in the table is empty
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    if constexpr (BACK) {
        for (int i = lo; c >= begin; --i)
            for (; c >= begin && c >= t.first[i]; --c) f(i, c - t.first[i]);
    } else {
        for (int i = lo; c < end; ++i) {
            const int next = i + 1 < t.tensors ? t.first[i + 1] : t.chunks, stop = next < end ? next : end;
            for (; c < stop; ++c) f(i, c - t.first[i]);
        }
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

// A thread's values of a chunk.  STREAM: past the caches.
template <typename T, bool STREAM>
__device__ __forceinline__ void chunk_load(Raw8<T> (&v)[kVecs], const void* g, int64_t count, int64_t at) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int64_t c = at + 8 * (static_cast<int64_t>(threadIdx.x) + kThreads * k);
        const T* p = static_cast<const T*>(g) + c;
        if (STREAM && count - c >= 8)
            v[k].q = __builtin_nontemporal_load(reinterpret_cast<const typename Raw8<T>::vec*>(p));
        else v[k].load(p, count - c);
    }
}
template <typename T>
__device__ __forceinline__ double chunk_squares(const void* g, int64_t count, int64_t at) {
    Raw8<T> v[kVecs];
    chunk_load<T, false>(v, g, count, at);
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
    each_chunk<false>(t, [&](int i, int c) {
        const int64_t n = t.count[i], at = c * kChunk;
        s += n < 0 ? chunk_squares<bf16>(t.grad[i], -n, at) : chunk_squares<float>(t.grad[i], n, at);
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

// A chunk on its way through the registers.
template <typename T>
struct ChunkScale {
    Raw8<T> v[kVecs];
    __device__ __forceinline__ void load(const void* g, int64_t count, int64_t at) { chunk_load<T, true>(v, g, count, at); }
    __device__ __forceinline__ void store(void* o, int64_t count, int64_t at, float f) const {
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const int64_t c = at + 8 * (static_cast<int64_t>(threadIdx.x) + kThreads * k);
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = v[k][e] * f;
            store8_stream(static_cast<T*>(o) + c, count - c, y);
        }
    }
};

// A workgroup's last chunks first: what the first launch read last is still in
// the Infinity Cache.  The first chunk's values are asked for ahead of the norm.
__global__ __launch_bounds__(kThreads) void k_grad_scale(GradTable t, const double* __restrict__ part, int parts,
                                                         float max_norm, float* __restrict__ norm) {
    __shared__ double red[kThreads / 64];
    float f = 0.0f;
    bool known = false, keep = false;
    auto factor = [&] {
        if (known) return;
        known = true;
        const double n = total_norm(part, parts, red);
        if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
        // A norm that is NaN is not below: the factor is NaN then, and 0 of an infinite one.
        keep = n <= static_cast<double>(max_norm);
        f = keep ? 1.0f : static_cast<float>(static_cast<double>(max_norm) / n);
    };
    each_chunk<true>(t, [&](int i, int c) {
        const int64_t n = t.count[i], at = c * kChunk;
        const bool here = t.out[i] == t.grad[i];
        if (known && keep && here) return;
        if (n < 0) {
            ChunkScale<bf16> v;
            v.load(t.grad[i], -n, at);
            factor();
            if (!(keep && here)) v.store(t.out[i], -n, at, f);
        } else {
            ChunkScale<float> v;
            v.load(t.grad[i], n, at);
            factor();
            if (!(keep && here)) v.store(t.out[i], n, at, f);
        }
    });
}

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

// Whether memory that is written (outs and the norm) shares a byte with another
// tensor's, or an out with its own grad in another way than as the same memory: by
// their places in order.
bool tangled(const nflow_grad_tensor* tensors, int count, const float* norm) {
    struct Bytes {
        uintptr_t from, to;
        bool written;
    };
    std::vector<Bytes> spans;
    spans.reserve(2 * static_cast<size_t>(count) + 1);
    spans.push_back({reinterpret_cast<uintptr_t>(norm), reinterpret_cast<uintptr_t>(norm) + sizeof(float), true});
    for (int i = 0; i < count; ++i) {
        const nflow_grad_tensor& t = tensors[i];
        const uintptr_t n = static_cast<uintptr_t>(t.count) * dtype_size(t.dtype);
        if (n == 0) continue;
        const auto g = reinterpret_cast<uintptr_t>(t.grad), o = reinterpret_cast<uintptr_t>(t.out);
        spans.push_back({o, o + n, true});
        if (o != g) spans.push_back({g, g + n, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Bytes& a, const Bytes& b) { return a.from < b.from; });
    uintptr_t any = 0, written = 0;                 // ends of what came before
    for (const Bytes& s : spans) {
        if (s.from < (s.written ? any : written)) return true;
        any = std::max(any, s.to);
        if (s.written) written = std::max(written, s.to);
    }
    return false;
}

// The next kTable tensors with elements, from `next` on; false when there are none.
bool fill(GradTable& t, const nflow_grad_tensor* tensors, int count, int& next) {
    t.tensors = t.chunks = 0;
    for (; next < count && t.tensors < kTable; ++next) {
        const nflow_grad_tensor& g = tensors[next];
        if (g.count == 0) continue;
        const int k = t.tensors++;
        t.grad[k] = g.grad;
        t.out[k] = g.out;
        t.count[k] = g.dtype == NFLOW_DTYPE_BF16 ? -g.count : g.count;
        t.first[k] = t.chunks;
        t.chunks += static_cast<int>(chunks_of(g.count));
    }
    if (t.tensors == 0) return false;
    const int blocks = std::min(t.chunks, kMaxParts);
    t.per = (t.chunks + blocks - 1) / blocks;
    return true;
}
int blocks_of(const GradTable& t) { return (t.chunks + t.per - 1) / t.per; }

size_t grad_space(int count) { return static_cast<size_t>((count + kTable - 1) / kTable) * kMaxParts * sizeof(double); }

// The launches of the norm; the partial sums' number, and the last table in t.
int launch_squares(const nflow_grad_tensor* tensors, int count, double* part, GradTable& t, hipStream_t st) {
    int parts = 0;
    for (int next = 0; next < count && fill(t, tensors, count, next);) {
        hipLaunchKernelGGL(k_grad_squares, dim3(blocks_of(t)), dim3(kThreads), 0, st, t, part + parts);
        parts += blocks_of(t);
    }
    return parts;
}

}  // namespace
}  // namespace nfq

using namespace nfq;

extern "C" {

int nflow_grad_workspace(int count, size_t* bytes) {
    clear_error();
    if (!bytes) return bad_arg("grad_workspace", "null output");
    *bytes = 0;
    if (count < 0) return bad_arg("grad_workspace", "bad count");
    *bytes = grad_space(count);
    return NFLOW_OK;
}

int nflow_grad_norm(const nflow_grad_tensor* tensors, int count, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "grad_norm";
    if (int rc = check_grads(what, tensors, count, true)) return rc;
    if (!norm) return bad_arg(what, "null norm");
    if (int rc = check_workspace(what, workspace, workspace_bytes, grad_space(count))) return rc;
    double* part = static_cast<double*>(workspace);
    GradTable t;
    const int parts = launch_squares(tensors, count, part, t, as_stream(stream));
    hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(kThreads), 0, as_stream(stream), part, parts, norm);
    return launch_status(what);
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
    if (int rc = check_workspace(what, workspace, workspace_bytes, grad_space(count))) return rc;
    try {
        if (tangled(tensors, count, norm)) return bad_arg(what, "an out or the norm overlaps a gradient or another out");
    } catch (const std::exception& e) {
        return set_error(NFLOW_INTERNAL, std::string(what) + ": " + e.what());
    }
    double* part = static_cast<double*>(workspace);
    hipStream_t st = as_stream(stream);
    GradTable t;
    const int parts = launch_squares(tensors, count, part, t, st);
    if (parts == 0) hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(kThreads), 0, st, part, 0, norm);
    // The norm goes out with one table's launch; t still holds the only table of a few tensors.
    bool first = true;
    for (int next = 0; parts > 0 && (count <= kTable ? first : next < count && fill(t, tensors, count, next)); first = false)
        hipLaunchKernelGGL(k_grad_scale, dim3(blocks_of(t)), dim3(kThreads), 0, st, t, part, parts, max_norm,
                           first ? norm : nullptr);
    return launch_status(what);
}

}  // extern "C"
