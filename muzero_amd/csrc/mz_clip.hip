// Global norm of many tensors and clipping by it (include/mzhip.h).
//
//   norm = sqrt(sum g^2),  out = g * (max_norm / norm) where norm > max_norm, else g
// The table of tensors travels in the kernel arguments (kBatch tensors a launch): nothing is uploaded, so a call may be
// captured and takes other tensors the next time.  A tensor is cut into chunks; workgroups stride over the chunks of all
// tensors.  Squares are summed in f64: exact squares of f32, no overflow, and one fixed order -- a workgroup leaves one
// partial sum, and every workgroup of the next launch adds up all of them itself.
#include "mz_vec.h"
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

namespace {

using mz::bf16;
using mz::f16;
using mz::Vec;

constexpr int kThreads = 256;
constexpr int kBatch = 128;                 // tensors a launch: 128 x 28 bytes of kernel arguments
constexpr long kChunk = 16384;              // elements
constexpr int64_t kMost = int64_t(1) << 43;  // elements: their chunks are counted in 32 bits
constexpr int kPartials = MZ_GLOBAL_NORM_WORKSPACE / sizeof(double);

struct Table {
    const void* in[kBatch];
    void* out[kBatch];
    long elements[kBatch];
    int first[kBatch];                      // chunk of all tensors that the tensor begins with
    signed char dtype[kBatch];
    int n, chunks;
};
static_assert(sizeof(Table) <= 3840, "the table has to fit the kernel arguments");

__device__ inline int tensor_of(const Table& t, int chunk) {
    int i = 0;
    for (int k = 1; k < t.n; ++k) i = t.first[k] <= chunk ? k : i;      // later tensors begin at later chunks
    return i;
}

template <typename T>
__device__ double squares(const T* p, long n) {
    constexpr int V = 16 / sizeof(T);
    double s = 0.0;
    const long whole = n / V;
    for (long i = threadIdx.x; i < whole; i += kThreads) {
        const Vec<T, V> v = mz::load<T, V>(p + i * V);
#pragma unroll
        for (int k = 0; k < V; ++k) s = fma((double)v[k], (double)v[k], s);
    }
    for (long i = whole * V + threadIdx.x; i < n; i += kThreads) s = fma((double)(float)p[i], (double)(float)p[i], s);
    return s;
}

__global__ void __launch_bounds__(kThreads) norm_partials_kernel(Table t, double* partials) {
    __shared__ double scratch[kThreads / 64];
    double s = 0.0;
    for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        const long at = (chunk - t.first[i]) * kChunk, n = t.elements[i] - at < kChunk ? t.elements[i] - at : kChunk;
        if (t.dtype[i] == MZ_F32) s += squares(static_cast<const float*>(t.in[i]) + at, n);
        else if (t.dtype[i] == MZ_F16) s += squares(static_cast<const f16*>(t.in[i]) + at, n);
        else s += squares(static_cast<const bf16*>(t.in[i]) + at, n);
    }
    s = mz::block_sum<kThreads>(s, scratch);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

__device__ inline double norm_of(const double* partials, int n, double* scratch) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) s += partials[i];
    return sqrt(mz::block_sum<kThreads>(s, scratch));
}

__global__ void __launch_bounds__(kThreads) norm_finish_kernel(const double* partials, int n, float* out_norm) {
    __shared__ double scratch[kThreads / 64];
    const double norm = norm_of(partials, n, scratch);
    if (threadIdx.x == 0) *out_norm = (float)norm;
}

template <typename T>
__device__ void scale_chunk(const T* in, T* out, long n, float f) {
    constexpr int V = 16 / sizeof(T);
    const long whole = n / V;
    for (long i = threadIdx.x; i < whole; i += kThreads) {
        const Vec<T, V> v = mz::load<T, V>(in + i * V);
        float r[V];
#pragma unroll
        for (int k = 0; k < V; ++k) r[k] = v[k] * f;
        mz::store<T, V>(out + i * V, r);
    }
    for (long i = whole * V + threadIdx.x; i < n; i += kThreads) out[i] = (T)((float)in[i] * f);
}

__global__ void __launch_bounds__(kThreads) clip_kernel(Table t, const double* partials, int n, double max_norm, float* out_norm) {
    __shared__ double scratch[kThreads / 64];
    const double norm = norm_of(partials, n, scratch);
    if (out_norm && blockIdx.x == 0 && threadIdx.x == 0) *out_norm = (float)norm;
    const float f = norm <= max_norm ? 1.f : (float)(max_norm / norm);        // a NaN norm gives NaN
    for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        if (f == 1.f && t.in[i] == t.out[i]) continue;                        // nothing to change in place
        const long at = (chunk - t.first[i]) * kChunk, m = t.elements[i] - at < kChunk ? t.elements[i] - at : kChunk;
        if (t.dtype[i] == MZ_F32) scale_chunk(static_cast<const float*>(t.in[i]) + at, static_cast<float*>(t.out[i]) + at, m, f);
        else if (t.dtype[i] == MZ_F16) scale_chunk(static_cast<const f16*>(t.in[i]) + at, static_cast<f16*>(t.out[i]) + at, m, f);
        else scale_chunk(static_cast<const bf16*>(t.in[i]) + at, static_cast<bf16*>(t.out[i]) + at, m, f);
    }
}

// Calls f(table, grid) for every launch's part of the tensors; empty tensors are left out.
template <typename F>
void for_each_table(int32_t n, const mz_tensor_t* tensors, void* const* outputs, F f) {
    Table t;
    t.n = t.chunks = 0;
    const int launches = (n + kBatch - 1) / kBatch;            // their workgroups share the room for partial sums
    const int most = kPartials / launches < 2048 ? kPartials / launches : 2048;
    for (int32_t i = 0; i < n; ++i) {
        if (!tensors[i].elements) continue;
        t.in[t.n] = tensors[i].data;
        t.out[t.n] = outputs ? outputs[i] : tensors[i].data;
        t.elements[t.n] = tensors[i].elements;
        t.first[t.n] = t.chunks;
        t.dtype[t.n] = (signed char)tensors[i].dtype;
        t.chunks += (int)((tensors[i].elements + kChunk - 1) / kChunk);
        if (++t.n == kBatch) {
            f(t, t.chunks < most ? t.chunks : most);
            t.n = t.chunks = 0;
        }
    }
    if (t.n) f(t, t.chunks < most ? t.chunks : most);
}

int check(int32_t n, const mz_tensor_t* tensors, void* workspace, int64_t bytes) {
    MZ_REQUIRE(n >= 1 && n <= MZ_GLOBAL_NORM_MAX_TENSORS, "between 1 and %d tensors, got %d", MZ_GLOBAL_NORM_MAX_TENSORS, n);
    MZ_REQUIRE(tensors, "tensors is NULL");
    MZ_REQUIRE(workspace && bytes >= MZ_GLOBAL_NORM_WORKSPACE, "workspace of %lld bytes, %d needed", (long long)bytes, MZ_GLOBAL_NORM_WORKSPACE);
    int64_t total = 0;
    for (int32_t i = 0; i < n; ++i) {
        const int item = mz::dtype_size(tensors[i].dtype);
        MZ_REQUIRE(item, "tensor %d: dtype %d is not one of mz_dtype", i, tensors[i].dtype);
        MZ_REQUIRE(tensors[i].elements >= 0 && tensors[i].elements <= kMost - total, "tensor %d: %lld elements (2^43 in all at most)", i,
                   (long long)tensors[i].elements);
        total += tensors[i].elements;
        MZ_REQUIRE(tensors[i].data || !tensors[i].elements, "tensor %d: data is NULL", i);
        MZ_REQUIRE((uintptr_t)tensors[i].data % item == 0, "tensor %d: data is not aligned to its type", i);
    }
    return MZ_OK;
}

struct Span {
    uintptr_t begin, end;
    int32_t tensor;
    bool written;
};

// No written span may meet another one; a tensor clipped in place has one span.
int check_overlap(int32_t n, const mz_tensor_t* tensors, void* const* outputs) {
    std::vector<Span> spans;
    spans.reserve(2 * (size_t)n);
    for (int32_t i = 0; i < n; ++i) {
        const uintptr_t bytes = (uintptr_t)tensors[i].elements * mz::dtype_size(tensors[i].dtype);
        if (!bytes) continue;
        const uintptr_t in = (uintptr_t)tensors[i].data, out = outputs ? (uintptr_t)outputs[i] : in;
        MZ_REQUIRE(out, "output %d is NULL", i);
        MZ_REQUIRE(out % mz::dtype_size(tensors[i].dtype) == 0, "output %d is not aligned to its type", i);
        spans.push_back({out, out + bytes, i, true});
        if (in != out) spans.push_back({in, in + bytes, i, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    uintptr_t end_any = 0, end_written = 0;
    int32_t by_any = -1, by_written = -1;
    for (const Span& s : spans) {
        const int32_t by = s.written ? (s.begin < end_any ? by_any : -1) : (s.begin < end_written ? by_written : -1);
        MZ_REQUIRE(by < 0, "tensors %d and %d overlap", by, s.tensor);
        if (s.end > end_any) end_any = s.end, by_any = s.tensor;
        if (s.written && s.end > end_written) end_written = s.end, by_written = s.tensor;
    }
    return MZ_OK;
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return mz::fail(MZ_ERR_HIP, "%s launch failed: %s", what, hipGetErrorString(e));
    return MZ_OK;
}

int partials_of(hipStream_t st, int32_t n, const mz_tensor_t* tensors, double* partials) {
    int used = 0;
    for_each_table(n, tensors, nullptr, [&](const Table& t, int grid) {
        norm_partials_kernel<<<grid, kThreads, 0, st>>>(t, partials + used);
        used += grid;
    });
    return used;
}

}  // namespace

extern "C" {

int mz_global_norm(void* stream, int32_t n, const mz_tensor_t* tensors, void* workspace, int64_t workspace_bytes, float* out_norm) {
    const int bad = check(n, tensors, workspace, workspace_bytes);
    if (bad) return bad;
    MZ_REQUIRE(out_norm, "out_norm is NULL");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    double* partials = static_cast<double*>(workspace);
    const int used = partials_of(st, n, tensors, partials);
    norm_finish_kernel<<<1, kThreads, 0, st>>>(partials, used, out_norm);
    return launched("mz_global_norm");
}

int mz_clip_by_global_norm(void* stream, int32_t n, const mz_tensor_t* tensors, void* const* outputs, double max_norm,
                           void* workspace, int64_t workspace_bytes, float* out_norm) {
    int bad = check(n, tensors, workspace, workspace_bytes);
    if (bad) return bad;
    MZ_REQUIRE(out_norm, "out_norm is NULL");
    MZ_REQUIRE(max_norm >= 0, "max_norm must be >= 0");
    try {
        bad = check_overlap(n, tensors, outputs);
    } catch (const std::bad_alloc&) {
        return mz::fail(MZ_ERR_OOM, "no host memory for the overlap check");
    }
    if (bad) return bad;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    double* partials = static_cast<double*>(workspace);
    const int used = partials_of(st, n, tensors, partials);
    float* out = out_norm;
    for_each_table(n, tensors, outputs, [&](const Table& t, int grid) {
        clip_kernel<<<grid, kThreads, 0, st>>>(t, partials, used, max_norm, out);
        out = nullptr;
    });
    if (out) norm_finish_kernel<<<1, kThreads, 0, st>>>(partials, used, out);      // empty tensors only
    return launched("mz_clip_by_global_norm");
}

}  // extern "C"
