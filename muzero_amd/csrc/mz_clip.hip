// Global norm of many tensors and clipping by it (include/mzhip.h).
//
//   norm = sqrt(sum g^2),  out = g * (max_norm / norm) where norm > max_norm, else g
//
// Bound by memory: the norm reads every tensor once, clipping reads it again and writes it.  Tensors are cut into chunks of
// one size, and workgroups stride over the chunks of all tensors.  Squares are summed in f64: exact squares of f32, no
// overflow, and one fixed order -- a workgroup leaves one partial sum, and every workgroup of the second launch adds up all
// of them itself, which takes less than a launch in between.  The table of tensors lies in device memory where the caller
// keeps it (one launch a pass for any number of tensors); otherwise it travels in the kernel arguments, kBatch tensors a
// launch, so that nothing is uploaded for tensors that are others in the next step.  250 M elements f32: 148 us for the norm
// (1 GB: 6.8 TB/s), 421 for clipping (2 GB: 4.75 TB/s, a large copy's rate); 161 tensors of 23 M elements: 12.8 and 23.2 us.
#include "mz_vec.h"
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <new>
#include <vector>

namespace {

using mz::bf16;
using mz::f16;
using mz::Vec;

constexpr int kThreads = 256;
constexpr int kPartials = MZ_GLOBAL_NORM_WORKSPACE / sizeof(double);
constexpr int kBlocks = 2048;               // workgroups of a launch: eight a CU
constexpr int64_t kMost = int64_t(1) << 43;  // elements: their chunks are counted in 32 bits

struct Entry {
    const void* in;
    void* out;
    int64_t elements;
    int32_t first;                          // chunk of all tensors that the tensor begins with
    int32_t dtype;
};
static_assert(sizeof(Entry) == MZ_TENSOR_TABLE_ENTRY, "the header states an entry's size");

constexpr int kBatch = 112;                 // 3584 bytes of kernel arguments
struct InArguments {
    Entry e[kBatch];
    int n, chunks;
    long chunk;                             // elements of a chunk
    __device__ const Entry* entries() const { return e; }
};
struct InMemory {
    const Entry* e;
    int n, chunks;
    long chunk;
    __device__ const Entry* entries() const { return e; }
};

// Index of the tensor that a chunk belongs to: the last that begins at or before it.  The wavefront's lanes look at 64 places
// at once, so 112 tensors take two looks and 8192 three.
__device__ inline int tensor_of(const Entry* e, int n, int chunk) {
    int lo = 0, count = n;
    while (count > 1) {
        const int step = (count + 63) / 64, at = (int)(threadIdx.x & 63) * step;
        const bool before = at < count && e[lo + at].first <= chunk;
        const int last = __popcll(__ballot(before)) - 1;                   // the first place always counts
        lo += last * step;
        count = count - last * step < step ? count - last * step : step;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// vector(index, values) and single(index) over n elements at p, U vectors a thread under way at once
template <bool STREAM, typename T, typename F, typename G>
__device__ inline void walk(const T* p, long n, F vector, G single) {
    constexpr int V = 16 / sizeof(T), U = 4;
    const long whole = n / V;
    for (long i = threadIdx.x; i < whole; i += U * kThreads) {
        Vec<T, V> v[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (i + k * kThreads < whole) v[k] = STREAM ? mz::load_streaming<T, V>(p + (i + k * kThreads) * V) : mz::load<T, V>(p + (i + k * kThreads) * V);
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (i + k * kThreads < whole) vector((i + k * kThreads) * V, v[k]);
    }
    for (long i = whole * V + threadIdx.x; i < n; i += kThreads) single(i);
}

template <bool STREAM, typename T>
__device__ inline double squares(const T* p, long n) {
    double s = 0.0;
    walk<STREAM>(p, n,
         [&](long, const Vec<T, 16 / sizeof(T)>& v) {
#pragma unroll
             for (int k = 0; k < (int)(16 / sizeof(T)); ++k) s = fma((double)v[k], (double)v[k], s);
         },
         [&](long i) { s = fma((double)(float)p[i], (double)(float)p[i], s); });
    return s;
}

// STREAM: tensors that no cache holds until clipping reads them again.  At 1 GB that made this pass 206 -> 148 us, as it no
// longer has to write back what the last clipping left there, and clipping 394 -> 423; at 63 MB, which a cache holds, it
// made clipping 23 -> 31.
template <typename Table, bool STREAM>
__global__ void __launch_bounds__(kThreads) norm_partials_kernel(Table t, double* partials) {
    __shared__ double scratch[kThreads / 64];
    const Entry* e = t.entries();
    double s = 0.0;
    for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
        const int i = tensor_of(e, t.n, chunk);
        const long at = (chunk - e[i].first) * t.chunk, n = e[i].elements - at < t.chunk ? e[i].elements - at : t.chunk;
        if (e[i].dtype == MZ_F32) s += squares<STREAM>(static_cast<const float*>(e[i].in) + at, n);
        else if (e[i].dtype == MZ_F16) s += squares<STREAM>(static_cast<const f16*>(e[i].in) + at, n);
        else s += squares<STREAM>(static_cast<const bf16*>(e[i].in) + at, n);
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

// F: float, or double for a scale below float's smallest normal number, which would lose bits that the product has
template <typename T, typename F>
__device__ inline void scale_chunk(const T* in, T* out, long n, F f) {
    walk<false>(in, n,
         [&](long i, const Vec<T, 16 / sizeof(T)>& v) {
             float r[16 / sizeof(T)];
#pragma unroll
             for (int k = 0; k < (int)(16 / sizeof(T)); ++k) r[k] = (float)(v[k] * f);
             mz::store(out + i, r);
         },
         [&](long i) { out[i] = (T)(float)((float)in[i] * f); });
}

template <typename F>
__device__ inline void scale_part(const Entry& e, long at, long n, F f) {
    if (e.dtype == MZ_F32) scale_chunk(static_cast<const float*>(e.in) + at, static_cast<float*>(e.out) + at, n, f);
    else if (e.dtype == MZ_F16) scale_chunk(static_cast<const f16*>(e.in) + at, static_cast<f16*>(e.out) + at, n, f);
    else scale_chunk(static_cast<const bf16*>(e.in) + at, static_cast<bf16*>(e.out) + at, n, f);
}

template <typename Table>
__global__ void __launch_bounds__(kThreads) clip_kernel(Table t, const double* partials, int n, double max_norm, float* out_norm) {
    __shared__ double scratch[kThreads / 64];
    const Entry* e = t.entries();
    const double norm = norm_of(partials, n, scratch);
    if (out_norm && blockIdx.x == 0 && threadIdx.x == 0) *out_norm = (float)norm;
    const double scale = norm <= max_norm ? 1.0 : max_norm / norm;            // a NaN norm gives NaN
    const float f = (float)scale;
    for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
        const int i = tensor_of(e, t.n, chunk);
        if (f == 1.f && e[i].in == e[i].out) continue;                        // nothing to change in place
        const long at = (chunk - e[i].first) * t.chunk, m = e[i].elements - at < t.chunk ? e[i].elements - at : t.chunk;
        if (scale > 0.0 && scale < 0x1p-126) scale_part(e[i], at, m, scale);
        else scale_part(e[i], at, m, f);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------

struct Total {
    int64_t elements, bytes;
};
constexpr int64_t kCache = int64_t(1) << 28;               // bytes of the last-level cache

int check(int32_t n, const mz_tensor_t* tensors, Total* total) {
    MZ_REQUIRE(n >= 1 && n <= MZ_GLOBAL_NORM_MAX_TENSORS, "between 1 and %d tensors, got %d", MZ_GLOBAL_NORM_MAX_TENSORS, n);
    MZ_REQUIRE(tensors, "tensors is NULL");
    *total = {0, 0};
    for (int32_t i = 0; i < n; ++i) {
        const int item = mz::dtype_size(tensors[i].dtype);
        MZ_REQUIRE(item, "tensor %d: dtype %d is not one of mz_dtype", i, tensors[i].dtype);
        MZ_REQUIRE(tensors[i].elements >= 0 && tensors[i].elements <= kMost - total->elements, "tensor %d: %lld elements (2^43 in all at most)", i,
                   (long long)tensors[i].elements);
        MZ_REQUIRE(tensors[i].data || !tensors[i].elements, "tensor %d: data is NULL", i);
        MZ_REQUIRE((uintptr_t)tensors[i].data % item == 0, "tensor %d: data is not aligned to its type", i);
        total->elements += tensors[i].elements;
        total->bytes += tensors[i].elements * item;
    }
    return MZ_OK;
}

int check_workspace(void* workspace, int64_t bytes, const float* out_norm) {
    MZ_REQUIRE(workspace && bytes >= MZ_GLOBAL_NORM_WORKSPACE, "workspace of %lld bytes, %d needed", (long long)bytes, MZ_GLOBAL_NORM_WORKSPACE);
    MZ_REQUIRE(out_norm, "out_norm is NULL");
    MZ_REQUIRE(mz::aligned(sizeof(double), {workspace}) && mz::aligned(sizeof(float), {out_norm}), "workspace or out_norm is not aligned");
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

int check_written(int32_t n, const mz_tensor_t* tensors, void* const* outputs) {
    try {
        return check_overlap(n, tensors, outputs);
    } catch (const std::bad_alloc&) {
        return mz::fail(MZ_ERR_OOM, "no host memory for the overlap check");
    }
}

// A chunk for each of a launch's workgroups while a chunk still is eight vectors a thread, up to 64 K elements.
long chunk_of(int64_t total) {
    long c = 2048;
    while (c < 65536 && c * kBlocks < total) c <<= 1;
    return c;
}

Entry entry_of(const mz_tensor_t& t, void* out, int32_t first) { return {t.data, out, t.elements, first, t.dtype}; }
int chunks_of(int64_t elements, long chunk) { return (int)((elements + chunk - 1) / chunk); }

// Calls f(table, workgroups) for every launch's part of the tensors; empty tensors are left out.
template <typename F>
void for_each_table(int32_t n, const mz_tensor_t* tensors, void* const* outputs, const Total& total, F f) {
    InArguments t;
    t.n = t.chunks = 0;
    t.chunk = chunk_of(total.elements);
    const int launches = (n + kBatch - 1) / kBatch;            // their workgroups share the room for partial sums
    const int most = kPartials / launches < kBlocks ? kPartials / launches : kBlocks;
    for (int32_t i = 0; i < n; ++i) {
        if (!tensors[i].elements) continue;
        t.e[t.n] = entry_of(tensors[i], outputs ? outputs[i] : tensors[i].data, t.chunks);
        t.chunks += chunks_of(tensors[i].elements, t.chunk);
        if (++t.n == kBatch) {
            f(t, t.chunks < most ? t.chunks : most);
            t.n = t.chunks = 0;
        }
    }
    if (t.n) f(t, t.chunks < most ? t.chunks : most);
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return mz::fail(MZ_ERR_HIP, "%s launch failed: %s", what, hipGetErrorString(e));
    return MZ_OK;
}

template <typename Table>
void launch_partials(const Table& t, int grid, bool stream, hipStream_t st, double* partials) {
    if (stream) norm_partials_kernel<Table, true><<<grid, kThreads, 0, st>>>(t, partials);
    else norm_partials_kernel<Table, false><<<grid, kThreads, 0, st>>>(t, partials);
}
int partials_of(hipStream_t st, int32_t n, const mz_tensor_t* tensors, const Total& total, double* partials) {
    int used = 0;
    for_each_table(n, tensors, nullptr, total, [&](const InArguments& t, int grid) {
        launch_partials(t, grid, total.bytes > kCache, st, partials + used);
        used += grid;
    });
    return used;
}

int check_table(const mz_tensor_table_t* t, const void* device_table) {
    MZ_REQUIRE(t, "table is NULL");
    MZ_REQUIRE(t->entries >= 0 && t->entries <= MZ_GLOBAL_NORM_MAX_TENSORS && t->chunks >= t->entries && t->chunk >= 1, "not a table of mz_tensor_table_build");
    MZ_REQUIRE(device_table || !t->entries, "device_table is NULL");
    return MZ_OK;
}
InMemory in_memory(const mz_tensor_table_t* t, const void* device_table) {
    return {static_cast<const Entry*>(device_table), t->entries, t->chunks, t->chunk};
}
int blocks_of(const mz_tensor_table_t* t) { return t->chunks < kBlocks ? t->chunks : kBlocks; }

}  // namespace

extern "C" {

int mz_global_norm(void* stream, int32_t n, const mz_tensor_t* tensors, void* workspace, int64_t workspace_bytes, float* out_norm) {
    Total total;
    int bad = check(n, tensors, &total);
    if (!bad) bad = check_workspace(workspace, workspace_bytes, out_norm);
    if (bad) return bad;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    double* partials = static_cast<double*>(workspace);
    const int used = partials_of(st, n, tensors, total, partials);
    norm_finish_kernel<<<1, kThreads, 0, st>>>(partials, used, out_norm);
    return launched("mz_global_norm");
}

int mz_clip_by_global_norm(void* stream, int32_t n, const mz_tensor_t* tensors, void* const* outputs, double max_norm,
                           void* workspace, int64_t workspace_bytes, float* out_norm) {
    Total total;
    int bad = check(n, tensors, &total);
    if (!bad) bad = check_workspace(workspace, workspace_bytes, out_norm);
    if (!bad) bad = check_written(n, tensors, outputs);
    if (bad) return bad;
    MZ_REQUIRE(max_norm >= 0, "max_norm must be >= 0");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    double* partials = static_cast<double*>(workspace);
    const int used = partials_of(st, n, tensors, total, partials);
    float* out = out_norm;
    for_each_table(n, tensors, outputs, total, [&](const InArguments& t, int grid) {
        clip_kernel<<<grid, kThreads, 0, st>>>(t, partials, used, max_norm, out);
        out = nullptr;
    });
    if (out) norm_finish_kernel<<<1, kThreads, 0, st>>>(partials, used, out);      // empty tensors only
    return launched("mz_clip_by_global_norm");
}

int mz_tensor_table_build(int32_t n, const mz_tensor_t* tensors, void* const* outputs, void* host_table, mz_tensor_table_t* out_table) {
    Total total;
    const int bad = check(n, tensors, &total);
    if (bad) return bad;
    MZ_REQUIRE(host_table && out_table, "host_table/out_table is NULL");
    Entry* e = static_cast<Entry*>(host_table);
    mz_tensor_table_t t = {};
    t.chunk = chunk_of(total.elements);
    t.large = total.bytes > kCache;
    // a table that clipping may not write still serves the norm
    t.writable = check_written(n, tensors, outputs) == MZ_OK;
    for (int32_t i = 0; i < n; ++i) {
        if (!tensors[i].elements) continue;
        e[t.entries++] = entry_of(tensors[i], outputs ? outputs[i] : tensors[i].data, t.chunks);
        t.chunks += chunks_of(tensors[i].elements, t.chunk);
    }
    *out_table = t;
    return MZ_OK;
}

int mz_tensor_table_global_norm(void* stream, const mz_tensor_table_t* table, const void* device_table, void* workspace,
                                int64_t workspace_bytes, float* out_norm) {
    int bad = check_table(table, device_table);
    if (!bad) bad = check_workspace(workspace, workspace_bytes, out_norm);
    if (bad) return bad;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    double* partials = static_cast<double*>(workspace);
    const int blocks = blocks_of(table);
    if (blocks) launch_partials(in_memory(table, device_table), blocks, table->large, st, partials);
    norm_finish_kernel<<<1, kThreads, 0, st>>>(partials, blocks, out_norm);
    return launched("mz_tensor_table_global_norm");
}

int mz_tensor_table_clip(void* stream, const mz_tensor_table_t* table, const void* device_table, double max_norm, void* workspace,
                         int64_t workspace_bytes, float* out_norm) {
    int bad = check_table(table, device_table);
    if (!bad) bad = check_workspace(workspace, workspace_bytes, out_norm);
    if (bad) return bad;
    MZ_REQUIRE(table->writable, "tensors of the table overlap: they cannot be written");
    MZ_REQUIRE(max_norm >= 0, "max_norm must be >= 0");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    double* partials = static_cast<double*>(workspace);
    const int blocks = blocks_of(table);
    if (!blocks) {
        norm_finish_kernel<<<1, kThreads, 0, st>>>(partials, 0, out_norm);
    } else {
        launch_partials(in_memory(table, device_table), blocks, table->large, st, partials);
        clip_kernel<<<blocks, kThreads, 0, st>>>(in_memory(table, device_table), partials, blocks, max_norm, out_norm);
    }
    return launched("mz_tensor_table_clip");
}

}  // extern "C"
