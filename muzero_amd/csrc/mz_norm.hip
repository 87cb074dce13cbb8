// Group norm with residual and activation over channels-last states, forward and backward (include/mzhip.h).
//
// Per sample n and group g of D = C / G channels, M = positions * D values:
//   mu = sum x / M, v = sum (x - mu)^2 / M, r = 1 / sqrt(v + eps), h = (x - mu) r, z = h w_c + b_c + residual, y = act(z)
//   dz = dy act'(z), db_c = sum dz, dw_c = sum dz h, a = sum_group dz w / M, q = sum_group dz w h / M,
//   dx = r (dz w - a - q h), dresidual = dz
//
// A workgroup takes a tile: whole groups side by side (or a piece of one wide group) x a chunk of positions of one sample.
// A thread keeps one vector of V channels (V divides D: one group a vector) and walks down the positions, so consecutive
// lanes read consecutive addresses.  Statistics are merged as (count, mean, sum of squared deviations): no difference of
// large sums.
#include "mz_vec.h"
#include <cmath>

namespace {

using mz::bf16;
using mz::f16;
using mz::Vec;

constexpr int kThreads = 256;

struct Norm {
    long N, S;
    int C, G, D, act, params_f32;
    float eps;
    long xs[2], rs[2], ds[2];
    int cols, gs, pieces, tiles, splits;      // vectors and groups of a tile, tiles of a sample, chunks of positions
    long chunk;
    const void *x, *res, *w, *b, *dy;
    void *y, *dx, *dres, *dw, *db;
    float *mean, *rstd, *ws;
};

struct Tile {
    long n, s0, s1;
    int split, g0, gs, piece, c0, cols;
};

template <int V>
__device__ Tile tile_of(const Norm& d, long id) {
    Tile t;
    const int tile = (int)(id % d.tiles);
    id /= d.tiles;
    t.split = (int)(id % d.splits);
    t.n = id / d.splits;
    t.s0 = t.split * d.chunk;
    t.s1 = t.s0 + d.chunk < d.S ? t.s0 + d.chunk : d.S;
    const int dv = d.D / V;
    if (d.pieces > 1) {
        t.g0 = tile / d.pieces;
        t.piece = tile % d.pieces;
        t.gs = 1;
        t.c0 = t.g0 * d.D + t.piece * d.cols * V;
        t.cols = dv - t.piece * d.cols < d.cols ? dv - t.piece * d.cols : d.cols;
    } else {
        t.g0 = tile * d.gs;
        t.piece = 0;
        t.gs = d.G - t.g0 < d.gs ? d.G - t.g0 : d.gs;
        t.c0 = t.g0 * d.D;
        t.cols = t.gs * dv;
    }
    return t;
}

struct Stat {
    float n, mean, m2;
};
__device__ inline Stat merge(const Stat& a, const Stat& b) {
    const float n = a.n + b.n, d = b.mean - a.mean, f = n > 0.f ? b.n / n : 0.f;
    return {n, fmaf(d, f, a.mean), a.m2 + b.m2 + d * d * a.n * f};
}

__device__ inline float param(const void* p, int f32, int c, const float*) { return static_cast<const float*>(p)[c]; }
template <typename T>
__device__ inline float param(const void* p, int f32, int c, const T*) {
    return f32 ? static_cast<const float*>(p)[c] : (float)static_cast<const T*>(p)[c];
}
template <typename T, int V>
__device__ inline void load_params(const Norm& d, int c, float (&w)[V], float (&b)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        w[i] = d.w ? param(d.w, d.params_f32, c + i, (const T*)nullptr) : 1.f;
        b[i] = d.b ? param(d.b, d.params_f32, c + i, (const T*)nullptr) : 0.f;
    }
}

__device__ inline float activate(float z, int act) {
    if (act == MZ_ACT_RELU) return z < 0.f ? 0.f : z;
    if (act == MZ_ACT_SILU) return z / (1.f + __expf(-z));
    if (act == MZ_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678f));
    if (act == MZ_ACT_TANH) return tanhf(z);
    return z;
}
__device__ inline float slope(float z, int act) {
    if (act == MZ_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (act == MZ_ACT_SILU) {
        const float s = 1.f / (1.f + __expf(-z));
        return s * fmaf(z, 1.f - s, 1.f);
    }
    if (act == MZ_ACT_GELU) return fmaf(z * 0.39894228f, __expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678f)));
    if (act == MZ_ACT_TANH) {
        const float t = tanhf(z);
        return fmaf(-t, t, 1.f);
    }
    return 1.f;
}

// lanes that share one group's reduction: a power of two, all groups of a tile within the workgroup
__device__ inline int lanes_per_group(int gs) {
    int p = 64;
    while (p * gs > kThreads) p >>= 1;
    return p;
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(Norm d) {
    __shared__ Stat part[kThreads];
    const int t = threadIdx.x, rows = kThreads / d.cols, r = t / d.cols, c = t % d.cols, dv = d.D / V;
    const long total = d.N * d.tiles * d.splits;
    for (long id = blockIdx.x; id < total; id += gridDim.x) {
        const Tile k = tile_of<V>(d, id);
        Stat s = {0.f, 0.f, 0.f};
        if (r < rows && c < k.cols) {
            const T* x = static_cast<const T*>(d.x) + k.n * d.xs[0] + k.c0 + c * V;
            for (long p = k.s0 + r; p < k.s1; p += rows) {
                const Vec<T, V> v = mz::load<T, V>(x + p * d.xs[1]);
                float sum = 0.f, m2 = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) sum += (float)v.v[i];
                const float m = sum / V;
#pragma unroll
                for (int i = 0; i < V; ++i) m2 = fmaf((float)v.v[i] - m, (float)v.v[i] - m, m2);
                s = merge(s, {(float)V, m, m2});
            }
        }
        __syncthreads();
        part[t] = s;
        __syncthreads();
        const int P = lanes_per_group(k.gs), g = t / P, w = d.pieces > 1 ? k.cols : dv;
        if (g < k.gs) {
            Stat a = {0.f, 0.f, 0.f};
            for (int e = t % P; e < rows * w; e += P) a = merge(a, part[e / w * d.cols + g * w + e % w]);
            for (int m = P >> 1; m; m >>= 1) a = merge(a, {__shfl_xor(a.n, m), __shfl_xor(a.mean, m), __shfl_xor(a.m2, m)});
            if (t % P == 0) {
                const long at = ((k.n * d.G + k.g0 + g) * d.splits + k.split) * d.pieces + k.piece;
                d.ws[3 * at] = a.n;
                d.ws[3 * at + 1] = a.mean;
                d.ws[3 * at + 2] = a.m2;
            }
        }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_apply_kernel(Norm d) {
    __shared__ float mean[kThreads], rstd[kThreads];
    const int t = threadIdx.x, rows = kThreads / d.cols, r = t / d.cols, c = t % d.cols, dv = d.D / V;
    const long total = d.N * d.tiles * d.splits;
    for (long id = blockIdx.x; id < total; id += gridDim.x) {
        const Tile k = tile_of<V>(d, id);
        const int P = lanes_per_group(k.gs), g = t / P, parts = d.splits * d.pieces;
        __syncthreads();
        if (g < k.gs) {
            Stat a = {0.f, 0.f, 0.f};
            const long ng = k.n * d.G + k.g0 + g;
            const float* ws = d.ws + 3 * ng * parts;
            for (int e = t % P; e < parts; e += P) a = merge(a, {ws[3 * e], ws[3 * e + 1], ws[3 * e + 2]});
            for (int m = P >> 1; m; m >>= 1) a = merge(a, {__shfl_xor(a.n, m), __shfl_xor(a.mean, m), __shfl_xor(a.m2, m)});
            if (t % P == 0) {
                mean[g] = a.mean;
                rstd[g] = 1.f / sqrtf(a.m2 / a.n + d.eps);
                if (d.mean && k.split == 0 && k.piece == 0) {
                    d.mean[ng] = mean[g];
                    d.rstd[ng] = rstd[g];
                }
            }
        }
        __syncthreads();
        if (r < rows && c < k.cols) {
            const int ch = k.c0 + c * V;
            const float mu = mean[d.pieces > 1 ? 0 : c / dv], rs = rstd[d.pieces > 1 ? 0 : c / dv];
            float w[V], b[V];
            load_params<T, V>(d, ch, w, b);
            const T* x = static_cast<const T*>(d.x) + k.n * d.xs[0] + ch;
            const T* res = d.res ? static_cast<const T*>(d.res) + k.n * d.rs[0] + ch : nullptr;
            T* y = static_cast<T*>(d.y) + k.n * d.S * d.C + ch;
            for (long p = k.s0 + r; p < k.s1; p += rows) {
                const Vec<T, V> v = mz::load<T, V>(x + p * d.xs[1]);
                float f[V];
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = fmaf(((float)v.v[i] - mu) * rs, w[i], b[i]);
                if (res) {
                    const Vec<T, V> u = mz::load<T, V>(res + p * d.rs[1]);
#pragma unroll
                    for (int i = 0; i < V; ++i) f[i] += (float)u.v[i];
                }
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = activate(f[i], d.act);
                mz::store<T, V>(y + p * d.C, f);
            }
        }
    }
}

// h and dz of V values
template <typename T, int V>
__device__ inline void back_values(const Norm& d, const T* x, const T* res, const T* dy, float mu, float rs, const float (&w)[V],
                                   const float (&b)[V], float (&h)[V], float (&dz)[V]) {
    const Vec<T, V> xv = mz::load<T, V>(x), gv = mz::load<T, V>(dy);
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = ((float)xv.v[i] - mu) * rs;
        z[i] = fmaf(h[i], w[i], b[i]);
    }
    if (res) {
        const Vec<T, V> u = mz::load<T, V>(res);
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] += (float)u.v[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) dz[i] = (float)gv.v[i] * slope(z[i], d.act);
}

// ws[(n * splits + split)][2][C] = sums of dz and dz h over the chunk's positions
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_back_sums_kernel(Norm d) {
    __shared__ float part[2][kThreads * V];
    const int t = threadIdx.x, rows = kThreads / d.cols, r = t / d.cols, c = t % d.cols;
    const long total = d.N * d.tiles * d.splits;
    for (long id = blockIdx.x; id < total; id += gridDim.x) {
        const Tile k = tile_of<V>(d, id);
        float s1[V] = {}, s2[V] = {};
        if (r < rows && c < k.cols) {
            const int ch = k.c0 + c * V;
            const long ng = k.n * d.G + ch / d.D;
            const float mu = d.mean[ng], rs = d.rstd[ng];
            float w[V], b[V], h[V], dz[V];
            load_params<T, V>(d, ch, w, b);
            const T* x = static_cast<const T*>(d.x) + k.n * d.xs[0] + ch;
            const T* res = d.res ? static_cast<const T*>(d.res) + k.n * d.rs[0] + ch : nullptr;
            const T* dy = static_cast<const T*>(d.dy) + k.n * d.ds[0] + ch;
            for (long p = k.s0 + r; p < k.s1; p += rows) {
                back_values<T, V>(d, x + p * d.xs[1], res ? res + p * d.rs[1] : nullptr, dy + p * d.ds[1], mu, rs, w, b, h, dz);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s1[i] += dz[i];
                    s2[i] = fmaf(dz[i], h[i], s2[i]);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            part[0][t * V + i] = s1[i];
            part[1][t * V + i] = s2[i];
        }
        __syncthreads();
        float* ws = d.ws + (k.n * d.splits + k.split) * 2 * d.C + k.c0;
        for (int e = t; e < k.cols * V; e += kThreads) {
            float a = 0.f, q = 0.f;
            for (int j = 0; j < rows; ++j) {
                a += part[0][j * d.cols * V + e];
                q += part[1][j * d.cols * V + e];
            }
            ws[e] = a;
            ws[d.C + e] = q;
        }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_back_apply_kernel(Norm d) {
    __shared__ float sa[kThreads], sq[kThreads];
    const int t = threadIdx.x, rows = kThreads / d.cols, r = t / d.cols, c = t % d.cols, dv = d.D / V;
    const float inv = 1.f / ((float)d.S * (float)d.D);
    const long total = d.N * d.tiles * d.splits;
    for (long id = blockIdx.x; id < total; id += gridDim.x) {
        const Tile k = tile_of<V>(d, id);
        const int P = lanes_per_group(k.gs), g = t / P;
        __syncthreads();
        if (g < k.gs) {
            float a = 0.f, q = 0.f;
            for (int e = t % P; e < d.D; e += P) {
                const int ch = (k.g0 + g) * d.D + e;
                const float w = d.w ? param(d.w, d.params_f32, ch, (const T*)nullptr) : 1.f;
                const float* ws = d.ws + k.n * d.splits * 2 * d.C + ch;
                for (int j = 0; j < d.splits; ++j) {
                    a = fmaf(w, ws[(long)j * 2 * d.C], a);
                    q = fmaf(w, ws[(long)j * 2 * d.C + d.C], q);
                }
            }
            for (int m = P >> 1; m; m >>= 1) {
                a += __shfl_xor(a, m);
                q += __shfl_xor(q, m);
            }
            if (t % P == 0) {
                sa[g] = a * inv;
                sq[g] = q * inv;
            }
        }
        __syncthreads();
        if (r < rows && c < k.cols) {
            const int ch = k.c0 + c * V, gi = d.pieces > 1 ? 0 : c / dv;
            const long ng = k.n * d.G + k.g0 + gi;
            const float mu = d.mean[ng], rs = d.rstd[ng], a = sa[gi], q = sq[gi];
            float w[V], b[V], h[V], dz[V];
            load_params<T, V>(d, ch, w, b);
            const T* x = static_cast<const T*>(d.x) + k.n * d.xs[0] + ch;
            const T* res = d.res ? static_cast<const T*>(d.res) + k.n * d.rs[0] + ch : nullptr;
            const T* dy = static_cast<const T*>(d.dy) + k.n * d.ds[0] + ch;
            const long out = k.n * d.S * d.C + ch;
            for (long p = k.s0 + r; p < k.s1; p += rows) {
                back_values<T, V>(d, x + p * d.xs[1], res ? res + p * d.rs[1] : nullptr, dy + p * d.ds[1], mu, rs, w, b, h, dz);
                if (d.dres) mz::store<T, V>(static_cast<T*>(d.dres) + out + p * d.C, dz);
                if (d.dx) {
#pragma unroll
                    for (int i = 0; i < V; ++i) dz[i] = rs * (fmaf(dz[i], w[i], -a) - h[i] * q);
                    mz::store<T, V>(static_cast<T*>(d.dx) + out + p * d.C, dz);
                }
            }
        }
    }
}

// dbias and dweight: the rows of ws summed over samples and chunks, 16 channels a workgroup, in 64 bits (a sum over every
// position of a batch that may cancel)
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_params_kernel(Norm d, long rows_total) {
    __shared__ double part[kThreads];
    const int t = threadIdx.x, c = blockIdx.x * 16 + t % 16, which = blockIdx.y;
    double s = 0.0;
    if (c < d.C)
        for (long r = t / 16; r < rows_total; r += kThreads / 16) s += d.ws[r * 2 * d.C + (long)which * d.C + c];
    part[t] = s;
    __syncthreads();
    if (t < 16 && c < d.C) {
        for (int j = 1; j < kThreads / 16; ++j) s += part[j * 16 + t];
        void* out = which ? d.dw : d.db;
        if (!out) return;
        if (d.params_f32) static_cast<float*>(out)[c] = (float)s;
        else static_cast<T*>(out)[c] = (T)(float)s;
    }
}

int vector_of(const mz_group_norm_t* c) {          // the widest access of at most 16 bytes that stays within a group
    int v = 16 / mz::dtype_size(c->dtype);
    while ((c->channels / c->groups) % v) v >>= 1;
    return v;
}

int check(const mz_group_norm_t* c) {
    MZ_REQUIRE(c != nullptr, "config is NULL");
    MZ_REQUIRE(c->batch >= 0 && c->positions >= 0 && c->channels >= 1 && c->channels <= 1 << 24, "bad sizes in mz_group_norm_t");
    MZ_REQUIRE(c->groups >= 1 && c->channels % c->groups == 0, "groups (%d) must divide channels (%d)", c->groups, c->channels);
    MZ_REQUIRE(mz::dtype_size(c->dtype), "dtype %d is not one of mz_dtype", c->dtype);
    MZ_REQUIRE(c->param_dtype == MZ_F32 || c->param_dtype == c->dtype, "param_dtype must be MZ_F32 or dtype");
    MZ_REQUIRE(c->activation >= MZ_ACT_NONE && c->activation <= MZ_ACT_TANH, "activation %d is not one of mz_activation", c->activation);
    MZ_REQUIRE(c->eps >= 0 && std::isfinite(c->eps), "eps must be finite and >= 0");
    MZ_REQUIRE(c->batch == 0 || c->positions <= (int64_t(1) << 48) / c->channels / c->batch, "the state has more than 2^48 elements");
    return MZ_OK;
}

Norm plan(const mz_group_norm_t* c) {
    Norm d = {};
    d.N = c->batch;
    d.S = c->positions;
    d.C = c->channels;
    d.G = c->groups;
    d.D = c->channels / c->groups;
    d.act = c->activation;
    d.params_f32 = c->param_dtype == MZ_F32;
    d.eps = (float)c->eps;
    for (int i = 0; i < 2; ++i) {
        d.xs[i] = c->x_strides[i];
        d.rs[i] = c->residual_strides[i];
        d.ds[i] = c->dy_strides[i];
    }
    const int dv = d.D / vector_of(c);
    if (dv > kThreads) {
        d.cols = kThreads;
        d.pieces = (dv + kThreads - 1) / kThreads;
        d.gs = 1;
        d.tiles = d.G * d.pieces;
    } else {
        d.gs = kThreads / dv < d.G ? kThreads / dv : d.G;
        d.cols = d.gs * dv;
        d.pieces = 1;
        d.tiles = (d.G + d.gs - 1) / d.gs;
    }
    const long rows = kThreads / d.cols;
    long splits = (2048 + d.N * d.tiles - 1) / (d.N * d.tiles > 0 ? d.N * d.tiles : 1);
    const long most = (d.S + rows * 8 - 1) / (rows * 8);       // at least eight vectors a thread
    if (splits > most) splits = most;
    if (splits > 64) splits = 64;
    if (splits < 1) splits = 1;
    d.chunk = (d.S + splits - 1) / splits;
    d.splits = d.chunk ? (int)((d.S + d.chunk - 1) / d.chunk) : 1;
    return d;
}

int64_t workspace_of(const Norm& d, bool backward) {
    if (d.N * d.S == 0) return 0;
    return backward ? d.N * d.splits * 2 * d.C * (int64_t)sizeof(float)
                    : d.N * d.G * d.splits * d.pieces * 3 * (int64_t)sizeof(float);
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return mz::fail(MZ_ERR_HIP, "%s launch failed: %s", what, hipGetErrorString(e));
    return MZ_OK;
}

template <typename F>
int with_type(int dtype, int v, F f) {
    if (dtype == MZ_F32) {
        if (v == 4) return f(float{}, std::integral_constant<int, 4>{});
        if (v == 2) return f(float{}, std::integral_constant<int, 2>{});
        return f(float{}, std::integral_constant<int, 1>{});
    }
    if (dtype == MZ_F16) {
        if (v == 8) return f(f16{}, std::integral_constant<int, 8>{});
        if (v == 4) return f(f16{}, std::integral_constant<int, 4>{});
        if (v == 2) return f(f16{}, std::integral_constant<int, 2>{});
        return f(f16{}, std::integral_constant<int, 1>{});
    }
    if (v == 8) return f(bf16{}, std::integral_constant<int, 8>{});
    if (v == 4) return f(bf16{}, std::integral_constant<int, 4>{});
    if (v == 2) return f(bf16{}, std::integral_constant<int, 2>{});
    return f(bf16{}, std::integral_constant<int, 1>{});
}

unsigned grid_of(long total) { return (unsigned)(total < (1L << 20) ? total : 1L << 20); }

}  // namespace

extern "C" {

int64_t mz_group_norm_workspace(const mz_group_norm_t* c, int32_t backward) {
    const int bad = check(c);
    return bad ? bad : workspace_of(plan(c), backward != 0);
}

int mz_group_norm_forward(void* stream, const mz_group_norm_t* c, const void* x, const void* residual, const void* weight,
                          const void* bias, void* out_y, float* out_mean, float* out_rstd, void* workspace,
                          int64_t workspace_bytes) {
    const int bad = check(c);
    if (bad) return bad;
    if (c->batch == 0 || c->positions == 0) return MZ_OK;
    MZ_REQUIRE(x && out_y, "x/out_y is NULL");
    MZ_REQUIRE(!out_mean == !out_rstd, "out_mean and out_rstd: both or neither");
    Norm d = plan(c);
    const int64_t need = workspace_of(d, false);
    MZ_REQUIRE(workspace_bytes >= need && (workspace || !need), "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    d.x = x;
    d.res = residual;
    d.w = weight;
    d.b = bias;
    d.y = out_y;
    d.mean = out_mean;
    d.rstd = out_rstd;
    d.ws = static_cast<float*>(workspace);
    const unsigned grid = grid_of(d.N * d.tiles * d.splits);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return with_type(c->dtype, vector_of(c), [&](auto t, auto v) {
        norm_stats_kernel<decltype(t), v.value><<<grid, kThreads, 0, st>>>(d);
        norm_apply_kernel<decltype(t), v.value><<<grid, kThreads, 0, st>>>(d);
        return launched("mz_group_norm_forward");
    });
}

int mz_group_norm_backward(void* stream, const mz_group_norm_t* c, const void* x, const void* residual, const void* weight,
                           const void* bias, const float* mean, const float* rstd, const void* dy, void* out_dx,
                           void* out_dresidual, void* out_dweight, void* out_dbias, void* workspace, int64_t workspace_bytes) {
    const int bad = check(c);
    if (bad) return bad;
    Norm d = plan(c);
    const int64_t need = workspace_of(d, true);
    const bool empty = c->batch == 0 || c->positions == 0;
    MZ_REQUIRE(empty || (x && mean && rstd && dy), "x/mean/rstd/dy is NULL");
    MZ_REQUIRE(workspace_bytes >= need && (workspace || !need), "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    d.x = x;
    d.res = residual;
    d.w = weight;
    d.b = bias;
    d.mean = const_cast<float*>(mean);
    d.rstd = const_cast<float*>(rstd);
    d.dy = dy;
    d.dx = out_dx;
    d.dres = out_dresidual;
    d.dw = out_dweight;
    d.db = out_dbias;
    d.ws = static_cast<float*>(workspace);
    const unsigned grid = grid_of(d.N * d.tiles * d.splits);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return with_type(c->dtype, vector_of(c), [&](auto t, auto v) {
        if (!empty) norm_back_sums_kernel<decltype(t), v.value><<<grid, kThreads, 0, st>>>(d);
        if (!empty && (d.dx || d.dres)) norm_back_apply_kernel<decltype(t), v.value><<<grid, kThreads, 0, st>>>(d);
        if (d.dw || d.db)       // of no rows: zeros
            norm_params_kernel<decltype(t)><<<dim3((d.C + 15) / 16, 2), kThreads, 0, st>>>(d, empty ? 0 : d.N * d.splits);
        return launched("mz_group_norm_backward");
    });
}

}  // extern "C"
