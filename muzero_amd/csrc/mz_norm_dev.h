// Device code of group norm with residual and activation over channels-last states, forward and backward (include/mzhip.h).
//
// Per sample n and group g of D = C / G channels, M = positions * D values:
//   mu = sum x / M, v = sum (x - mu)^2 / M, r = 1 / sqrt(v + eps), h = (x - mu) r, z = h w_c + b_c + residual, y = act(z)
//   dz = dy act'(z), db_c = sum dz, dw_c = sum dz h, a = sum_group dz w / M, q = sum_group dz w h / M,
//   dx = r (dz w - a - q h), dresidual = dz
// Bound by memory: forward reads x (and residual) and writes y, backward reads x, dy (and residual) and writes dx (and
// dresidual); 10 to 40 operations a value.
//
// A workgroup takes a tile of a sample: whole groups side by side, at least a 128-byte line of channels where there are as
// many.  A thread keeps one vector of V channels and walks down the positions, so consecutive lanes read consecutive
// addresses.  Vectors are as wide as an access can be (16 bytes) whatever D is: where D is no multiple of V, a group's last
// vector is moved back to end with the group, and its first `dup` channels, which are the vector's before it too, count
// nothing in the group's sums (they are stored twice, alike); where D is a smaller power of two, a vector holds Q = V / D
// groups with a sum of its own each, and a sample's last vector is moved back by whole groups (theirs is all stored twice,
// alike).  "Units" are what lanes share: a group, or the Q groups of a vector.  Vectors of a unit and units of
// a tile are padded to powers of two over the lanes: a lane's unit, vector and position come from bits of its number, and a
// unit's sums are a butterfly over the bits of its vectors and positions (group_sum), without index tables or divisions.  Two
// ways through:
//   resident  the tile's values stay in registers between the statistics and the result: one launch, every input read once.
//   split     samples too large for that (K vectors a thread do not hold the tile): positions are cut into chunks over
//             several workgroups; a first launch leaves each chunk's partial sums, a second adds them up and reads again.
// The variance is a sum of squared deviations from the mean (resident) or from the partial means, merged (split): no
// difference of large sums.  Every sum has one order, so results repeat bit for bit.
//
// Measured, with residual: 512 x 361 x 256 bf16, resident, forward 71 us (284 MB: 4.0 TB/s), backward 107 (473 MB: 4.4) and 5
// for the parameters' sums; a copy of 4 GB reaches 4.76.  24 x 9216 x 64 f16 without, split: forward 9.4 + 14.4 us (28 and
// 57 MB), backward 18.8 + 19.4 + 3.9 (57 and 85 MB), the inputs from the last-level cache.
#pragma once
#include "mz_vec.h"
#include <cmath>
#include <type_traits>

namespace mz_norm {

using mz::Vec;

constexpr int kSplitThreads = 256;
constexpr int kMostSplits = 64;

struct Norm {
    long N, S;
    int C, G, D, U, units, act, params_f32;   // U: channels of a unit, the last of `units` ends with the sample
    float eps;
    long xs[2], rs[2], ds[2];
    // lanes: bits [vector in unit : ldv][unit in tile : lgs][position : lrows][sample : the rest]
    int ldv, lgs, lrows, samples;
    int gs, tiles, pieces;                    // units of a tile, tiles of a sample, pieces of a unit wider than a workgroup
    int splits;                               // chunks of positions of a sample (split)
    long chunk, forward_blocks, blocks;       // positions of a chunk; workgroups of a tile (resident, forward and backward)
    const void *x, *res, *w, *b, *dy;
    void *y, *dx, *dres, *dw, *db;
    float *mean, *rstd, *ws;
};

struct Plan {
    Norm d;
    int v, q;                                 // channels of a vector, groups of it
    int threads, k;                           // of the resident kernels; k = 0: split
};

struct Lane {
    int vec, unit, row, sample;               // vector of its unit, unit of its tile, first position, sample
    int g, ch, dup;                           // unit and first channel within the sample, channels that are another lane's too
    int group;                                // first group of the unit
    int first, width;                         // this piece's first channel within its unit, and channels
    bool live;                                // not padding
};

template <int V, int Q>
__device__ Lane lane_of(const Norm& d, int tile) {
    Lane l;
    const int t = threadIdx.x;
    l.vec = t & ((1 << d.ldv) - 1);
    l.unit = (t >> d.ldv) & ((1 << d.lgs) - 1);
    l.row = (t >> (d.ldv + d.lgs)) & ((1 << d.lrows) - 1);
    l.sample = t >> (d.ldv + d.lgs + d.lrows);
    int gs = d.gs;
    l.first = 0;
    l.width = d.U;
    if (d.pieces > 1) {
        l.g = tile / d.pieces;
        l.first = ((tile - l.g * d.pieces) << d.ldv) * V;
        l.width = d.U - l.first < V << d.ldv ? d.U - l.first : V << d.ldv;
    } else {
        l.g = tile * d.gs;
        gs = d.units - l.g < gs ? d.units - l.g : gs;
    }
    l.live = l.vec * V < l.width && l.unit < gs && l.sample < d.samples;
    if (l.unit < gs) l.g += l.unit;           // padding reads what a live lane reads, and counts nothing
    const int in_unit = l.first + (l.live ? l.vec * V : 0), from = in_unit < d.U - V ? in_unit : d.U - V;
    l.dup = in_unit - from;
    const int begin = l.g * d.U;
    l.ch = (begin < d.C - d.U ? begin : d.C - d.U) + from;
    l.group = l.g * Q < d.G - Q ? l.g * Q : d.G - Q;
    return l;
}

// Sums of N values over the lanes of a unit (all its vectors and positions, of one sample), to every lane of it.
// `scratch`: TH * N floats that no thread still reads; an alternation of two needs no barrier in between.
template <int TH, int N>
__device__ inline void group_sum(float (&v)[N], const Norm& d, float* scratch) {
    const int dvp = 1 << d.ldv, pitch = 1 << (d.ldv + d.lgs);
    for (int m = 1; m < dvp && m < 64; m <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], m);
    for (int m = pitch; m < (pitch << d.lrows) && m < 64; m <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], m);
    if (TH == 64) return;
    // a unit's lanes differ in vector and position alone: wavefronts whose numbers differ in a unit's or a sample's bit stay apart
    const int t = threadIdx.x, sample = d.ldv + d.lgs + d.lrows, apart = ~((dvp - 1) | ((1 << d.lrows) - 1) * pitch) & ~63;
    // one slot for each unit and sample of a wavefront
    const int slot = ((t & 63 & (pitch - 1)) >> (d.ldv < 6 ? d.ldv : 6)) + (((t & 63) >> sample) << d.lgs);
#pragma unroll
    for (int k = 0; k < N; ++k) scratch[(t >> 6) * 64 * N + slot * N + k] = v[k];      // lanes of one slot hold the same value
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = 0.f;
    for (int w = 0; w < TH / 64; ++w)
        if ((((w << 6) ^ t) & apart) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += scratch[w * 64 * N + slot * N + k];
}

// Sums of V values over all positions and samples of the workgroup, to the lanes of its first row.  `scratch`: TH * V floats.
template <int TH, int V>
__device__ inline void column_sum(float (&v)[V], const Norm& d, float* scratch) {
    const int pitch = 1 << (d.ldv + d.lgs), t = threadIdx.x;
    for (int m = pitch; m < 64; m <<= 1)
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] += __shfl_xor(v[k], m);
    if (TH == 64) return;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) scratch[k * TH + t] = v[k];
    __syncthreads();
    if (t >= pitch) return;
    for (int w = 1; w < TH / 64; ++w)
        if (((w << 6) & (pitch - 1) & ~63) == 0)
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] += scratch[k * TH + (w << 6) + t];
}

template <typename T, int V>
__device__ inline void load_param(const void* p, int f32, int c, float missing, float (&v)[V]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = missing;
    } else if (f32) {
        const Vec<float, V> r = mz::load<float, V>(static_cast<const float*>(p) + c);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = r[i];
    } else {
        const Vec<T, V> r = mz::load<T, V>(static_cast<const T*>(p) + c);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = r[i];
    }
}
template <typename T, int V>
__device__ inline void load_params(const Norm& d, int c, float (&w)[V], float (&b)[V]) {
    load_param<T, V>(d.w, d.params_f32, c, 1.f, w);
    load_param<T, V>(d.b, d.params_f32, c, 0.f, b);
}

template <int Q>
__device__ inline void load_stats(const Norm& d, long at, float (&mu)[Q], float (&rs)[Q]) {
    const Vec<float, Q> m = mz::load<float, Q>(d.mean + at), r = mz::load<float, Q>(d.rstd + at);
#pragma unroll
    for (int q = 0; q < Q; ++q) mu[q] = m[q], rs[q] = r[q];
}

// No activation and relu share their code: a floor below which z is cut, and a threshold that z has to be above for its slope.
struct Cut {
    float floor, edge;
    __device__ explicit Cut(int act) : floor(act == MZ_ACT_RELU ? 0.f : -INFINITY), edge(act == MZ_ACT_RELU ? 0.f : NAN) {}
    __device__ float operator()(float z) const { return z < floor ? floor : z; }              // a NaN stays
    __device__ float slope(float z) const { return z <= edge ? 0.f : 1.f; }
};
// The others from one exponential and one reciprocal of the hardware (v_exp_f32, v_rcp_f32, one step each): with the library's
// exact division, erf and tanh the arithmetic took longer than the memory.  The exponent is a rounded product, so exp(x) is off
// by up to (1.3 |x| + 2) 2^-24 of itself: silu by up to (1.3 |z| + 8) 2^-24 of itself, tanh, whose exponential counts for less
// the farther out it is, by 12 2^-24.  A reciprocal below 2^-126 is 0: silu below -87.
__device__ inline float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950409f); }
__device__ inline float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

struct Silu {
    __device__ explicit Silu(int) {}
    __device__ static float sigmoid(float z) { return fast_rcp(1.f + fast_exp(-z)); }
    __device__ float operator()(float z) const { return z * sigmoid(z); }
    __device__ float slope(float z) const {
        const float s = sigmoid(z);
        return s * fmaf(z, 1.f - s, 1.f);
    }
};
// z times the normal distribution's integral, by the five-term approximation of Abramowitz and Stegun 7.1.26, with the
// exponential that the density needs too.  Off by 1.5e-7 / 2 at most and as much again or twice by f32's sums: 2.7e-7 |z|
// measured over [-10, 10].  That is absolute, as for 1 + erf: in the lower tail it is a growing part of the value (5e-4 at -4,
// 1.6e-3 at -5, 1e-2 at -8, where gelu is 5e-15).
struct Gelu {
    __device__ explicit Gelu(int) {}
    __device__ static float below(float z, float e) {          // e = exp(-z^2 / 2)
        const float t = fast_rcp(fmaf(fabsf(z), 0.3275911f * 0.70710678f, 1.f));
        const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f), 0.5f * 1.421413741f),
                                         0.5f * -0.284496736f), 0.5f * 0.254829592f);
        return z < 0.f ? p * e : fmaf(-p, e, 1.f);
    }
    __device__ float operator()(float z) const { return z * below(z, fast_exp(-0.5f * z * z)); }
    __device__ float slope(float z) const {
        const float e = fast_exp(-0.5f * z * z);
        return fmaf(z * 0.39894228f, e, below(z, e));
    }
};
// (1 - q) / (1 + q) with q = exp(-2 |z|); where 1 - q cancels, the first terms of the series of tanh
struct Tanh {
    __device__ explicit Tanh(int) {}
    __device__ float operator()(float z) const {
        const float q = fast_exp(-2.f * fabsf(z)), y = z * z;
        const float near = z * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
        return y < 0.0625f ? near : copysignf((1.f - q) * fast_rcp(1.f + q), z);
    }
    __device__ float slope(float z) const {
        const float q = fast_exp(-2.f * fabsf(z)), r = fast_rcp(1.f + q);
        return 4.f * q * r * r;
    }
};
template <typename F>
__device__ inline void with_activation(int act, F f) {       // the choice is outside the loops over values
    if (act == MZ_ACT_SILU) f(Silu(act));
    else if (act == MZ_ACT_GELU) f(Gelu(act));
    else if (act == MZ_ACT_TANH) f(Tanh(act));
    else f(Cut(act));
}

// sums over a vector's channels of f(value), for each of its Q groups
template <int Q, typename T, int V, typename F>
__device__ inline void sum_up(const Vec<T, V>& x, int dup, bool counts, F f, float (&sum)[Q]) {
    float p[Q] = {};
#pragma unroll
    for (int i = 0; i < V; ++i) p[i * Q / V] = f(x[i], i * Q / V, p[i * Q / V]);
    if (Q == 1 && dup) {                                    // once more without the other lane's
        p[0] = 0.f;
#pragma unroll
        for (int i = 1; i < V; ++i)
            if (i >= dup) p[0] = f(x[i], 0, p[0]);
    }
#pragma unroll
    for (int j = 0; j < Q; ++j) sum[j] += counts ? p[j] : 0.f;
}

template <int Q, typename T, int V, typename A>
__device__ inline void apply(const Vec<T, V>& x, const Vec<T, V>* res, const float (&mu)[Q], const float (&rs)[Q], const float (&w)[V],
                             const float (&b)[V], const A& act, T* y) {
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = fmaf((x[i] - mu[i * Q / V]) * rs[i * Q / V], w[i], b[i]);
    if (res)
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] += (*res)[i];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = act(f[i]);
    mz::store<T, V>(y, f);
}

// h and dz of V values
template <int Q, typename T, int V, typename A>
__device__ inline void back_values(const Vec<T, V>& x, const Vec<T, V>& dy, const Vec<T, V>* res, const float (&mu)[Q], const float (&rs)[Q],
                                   const float (&w)[V], const float (&b)[V], const A& act, float (&h)[V], float (&dz)[V]) {
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = (x[i] - mu[i * Q / V]) * rs[i * Q / V];
        z[i] = fmaf(h[i], w[i], b[i]);
    }
    if (res)
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] += (*res)[i];
#pragma unroll
    for (int i = 0; i < V; ++i) dz[i] = dy[i] * act.slope(z[i]);
}
template <int Q, typename T, int V>
__device__ inline void back_store(const Norm& d, long base, unsigned at, const float (&rs)[Q], const float (&aq)[2 * Q], const float (&w)[V],
                                  const float (&h)[V], float (&dz)[V], const T*) {
    if (d.dres) mz::store<T, V>(static_cast<T*>(d.dres) + base + at, dz);
    if (d.dx) {
#pragma unroll
        for (int i = 0; i < V; ++i) dz[i] = rs[i * Q / V] * (fmaf(dz[i], w[i], -aq[i * Q / V]) - h[i] * aq[Q + i * Q / V]);
        mz::store<T, V>(static_cast<T*>(d.dx) + base + at, dz);
    }
}

// dz, dz h into the channels' sums and, times the weight (0 for another lane's channels), into the groups' sums
template <int Q, int V>
__device__ inline void back_sum(const float (&h)[V], const float (&dz)[V], const float (&wq)[V], float (&s1)[V], float (&s2)[V], float (&aq)[2 * Q]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        s1[i] += dz[i];
        s2[i] = fmaf(dz[i], h[i], s2[i]);
        aq[i * Q / V] = fmaf(dz[i], wq[i], aq[i * Q / V]);
        aq[Q + i * Q / V] = fmaf(dz[i] * wq[i], h[i], aq[Q + i * Q / V]);
    }
}

// ---- resident ---------------------------------------------------------------------------------------------------------

// Up to K vectors a thread, positions row, row + step, ...: addresses are a workgroup's base and 32-bit byte offsets (the host
// checks that they suffice), a scalar base and one register a vector.
template <typename T, int V, int K>
__device__ inline void load_rows(Vec<T, V> (&v)[K], const T* base, int at, int stride, int row, int step, int S) {
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k * step < S) {                                 // the same for every thread
            const int s = row + k * step < S ? row + k * step : S - 1;      // past the end the last again, which counts nothing
            const unsigned bytes = (unsigned)(at + s * stride) * (unsigned)sizeof(T);
            v[k] = *reinterpret_cast<const Vec<T, V>*>(reinterpret_cast<const char*>(base) + bytes);
        }
}

// Ends what the compiler knows of loaded values, so that what is computed from them after the sums is computed anew: kept,
// the converted values, h and dz would take several times the registers of the vectors themselves.
template <typename T, int V, int K>
__device__ inline void forget(Vec<T, V> (&v)[K]) {
    if constexpr (sizeof(T) * V >= 4)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < Vec<T, V>::kWords; ++i) {
                uint32_t w = v[k].w[i];
                asm volatile("" : "+v"(w));
                v[k].w[i] = w;
            }
}

template <typename T, int V, int Q, int TH, int K>
__global__ void __launch_bounds__(TH) norm_forward_kernel(Norm d) {
    __shared__ float scratch[2][TH == 64 ? 1 : TH * Q];
    const int S = (int)d.S, step = 1 << d.lrows;
    const float inv = 1.f / ((float)d.S * (float)d.D);
    for (int tile = blockIdx.y; tile < d.tiles; tile += gridDim.y)
        for (long n0 = (long)blockIdx.x * d.samples; n0 < d.N; n0 += (long)gridDim.x * d.samples) {
            const Lane l = lane_of<V, Q>(d, tile);
            const int left = d.N - n0 < d.samples ? (int)(d.N - n0) : d.samples;       // samples of this workgroup
            const bool live = l.live && l.sample < left;
            const int j = live ? l.sample : 0;
            Vec<T, V> xv[K], rv[K];
            load_rows<T, V, K>(xv, static_cast<const T*>(d.x) + n0 * d.xs[0], j * (int)d.xs[0] + l.ch, (int)d.xs[1], l.row, step, S);
            if (d.res) load_rows<T, V, K>(rv, static_cast<const T*>(d.res) + n0 * d.rs[0], j * (int)d.rs[0] + l.ch, (int)d.rs[1], l.row, step, S);
            float w[V], b[V];
            load_params<T, V>(d, l.ch, w, b);
            float sum[Q] = {}, mu[Q], rs[Q];
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (k * step < S)
                    sum_up<Q>(xv[k], l.dup, live && l.row + k * step < S, [](float v, int, float p) { return p + v; }, sum);
            group_sum<TH>(sum, d, scratch[0]);
#pragma unroll
            for (int q = 0; q < Q; ++q) mu[q] = sum[q] * inv, sum[q] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (k * step < S)
                    sum_up<Q>(xv[k], l.dup, live && l.row + k * step < S,
                              [&](float v, int q, float p) { return fmaf(v - mu[q], v - mu[q], p); }, sum);
            group_sum<TH>(sum, d, scratch[1]);
#pragma unroll
            for (int q = 0; q < Q; ++q) rs[q] = 1.f / sqrtf(sum[q] * inv + d.eps);
            if (!live) continue;
            if (d.mean && l.vec == 0 && l.row == 0) {
                mz::store<float, Q>(d.mean + (n0 + j) * d.G + l.group, mu);
                mz::store<float, Q>(d.rstd + (n0 + j) * d.G + l.group, rs);
            }
            T* y = static_cast<T*>(d.y) + n0 * d.S * d.C;
            const int at = (j * S + l.row) * d.C + l.ch;
            with_activation(d.act, [&](auto act) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (l.row + k * step < S)
                        apply<Q>(xv[k], d.res ? &rv[k] : nullptr, mu, rs, w, b, act, y + (unsigned)(at + k * step * d.C));
            });
        }
}

// What a thread reads of one set of samples
template <typename T, int V, int K, int ARRAYS>
struct Held {
    Vec<T, V> v[ARRAYS][K];
};

// The same for wavefronts on their own with one or two vectors a thread: they stride over the samples and read the next set
// while they work on one, as too little of theirs would be under way otherwise.
template <typename T, int V, int Q, int K>
__global__ void __launch_bounds__(64) norm_forward_ahead_kernel(Norm d) {
    const int S = (int)d.S, step = 1 << d.lrows;
    const float inv = 1.f / ((float)d.S * (float)d.D);
    for (int tile = blockIdx.y; tile < d.tiles; tile += gridDim.y) {
        const Lane l = lane_of<V, Q>(d, tile);
        const auto left = [&](long n0) { return d.N - n0 < d.samples ? (int)(d.N - n0) : d.samples; };      // samples of a set
        const auto load = [&](Held<T, V, K, 2>& h, long n0) {
            const int j = l.live && l.sample < left(n0) ? l.sample : 0;
            load_rows<T, V, K>(h.v[0], static_cast<const T*>(d.x) + n0 * d.xs[0], j * (int)d.xs[0] + l.ch, (int)d.xs[1], l.row, step, S);
            if (d.res) load_rows<T, V, K>(h.v[1], static_cast<const T*>(d.res) + n0 * d.rs[0], j * (int)d.rs[0] + l.ch, (int)d.rs[1], l.row, step, S);
        };
        const long stride = (long)gridDim.x * d.samples;
        Held<T, V, K, 2> held, next;
        long n0 = (long)blockIdx.x * d.samples;
        if (n0 < d.N) load(held, n0);
        float w[V], b[V];
        load_params<T, V>(d, l.ch, w, b);
        for (; n0 < d.N; n0 += stride) {
            if (n0 + stride < d.N) load(next, n0 + stride);
            const bool live = l.live && l.sample < left(n0);
            const int j = live ? l.sample : 0;
            float sum[Q] = {}, mu[Q], rs[Q];
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (k * step < S)
                    sum_up<Q>(held.v[0][k], l.dup, live && l.row + k * step < S, [](float v, int, float p) { return p + v; }, sum);
            group_sum<64>(sum, d, nullptr);
#pragma unroll
            for (int q = 0; q < Q; ++q) mu[q] = sum[q] * inv, sum[q] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (k * step < S)
                    sum_up<Q>(held.v[0][k], l.dup, live && l.row + k * step < S,
                              [&](float v, int q, float p) { return fmaf(v - mu[q], v - mu[q], p); }, sum);
            group_sum<64>(sum, d, nullptr);
#pragma unroll
            for (int q = 0; q < Q; ++q) rs[q] = 1.f / sqrtf(sum[q] * inv + d.eps);
            if (live) {
                if (d.mean && l.vec == 0 && l.row == 0) {
                    mz::store<float, Q>(d.mean + (n0 + j) * d.G + l.group, mu);
                    mz::store<float, Q>(d.rstd + (n0 + j) * d.G + l.group, rs);
                }
                T* y = static_cast<T*>(d.y) + n0 * d.S * d.C;
                const int at = (j * S + l.row) * d.C + l.ch;
                with_activation(d.act, [&](auto act) {
#pragma unroll
                    for (int k = 0; k < K; ++k)
                        if (l.row + k * step < S)
                            apply<Q>(held.v[0][k], d.res ? &held.v[1][k] : nullptr, mu, rs, w, b, act, y + (unsigned)(at + k * step * d.C));
                });
            }
            held = next;
        }
    }
}

// A workgroup keeps its tile and strides over the samples: the channels' sums for dweight and dbias stay in registers and
// leave one row of ws [blocks][2][C] a workgroup.
template <typename T, int V, int Q, int TH, int K>
__global__ void __launch_bounds__(TH) norm_backward_kernel(Norm d) {
    __shared__ float scratch[TH == 64 ? 1 : TH * (2 * V > 4 * Q ? 2 * V : 4 * Q)];
    const int S = (int)d.S, step = 1 << d.lrows;
    const float inv = 1.f / ((float)d.S * (float)d.D);
    const long block = blockIdx.x;
    int turn = 0;
    for (int tile = blockIdx.y; tile < d.tiles; tile += gridDim.y) {
        const Lane l = lane_of<V, Q>(d, tile);
        float w[V], b[V], wq[V], s1[V] = {}, s2[V] = {};
        load_params<T, V>(d, l.ch, w, b);
#pragma unroll
        for (int i = 0; i < V; ++i) wq[i] = Q == 1 && i < l.dup ? 0.f : w[i];
        const auto left = [&](long n0) { return d.N - n0 < d.samples ? (int)(d.N - n0) : d.samples; };      // samples of a set
        const auto load = [&](Held<T, V, K, 3>& h, long n0) {
            const int j = l.live && l.sample < left(n0) ? l.sample : 0;
            load_rows<T, V, K>(h.v[0], static_cast<const T*>(d.x) + n0 * d.xs[0], j * (int)d.xs[0] + l.ch, (int)d.xs[1], l.row, step, S);
            load_rows<T, V, K>(h.v[1], static_cast<const T*>(d.dy) + n0 * d.ds[0], j * (int)d.ds[0] + l.ch, (int)d.ds[1], l.row, step, S);
            if (d.res) load_rows<T, V, K>(h.v[2], static_cast<const T*>(d.res) + n0 * d.rs[0], j * (int)d.rs[0] + l.ch, (int)d.rs[1], l.row, step, S);
        };
        constexpr bool AHEAD = TH == 64 && K <= 4;          // the next set is read while one is worked on
        const long stride = d.blocks * d.samples;
        Held<T, V, K, 3> held, next;
        long n0 = block * d.samples;
        if (AHEAD && n0 < d.N) load(held, n0);
        for (; n0 < d.N; n0 += stride, turn ^= 1) {
            if (!AHEAD) load(held, n0);
            else if (n0 + stride < d.N) load(next, n0 + stride);
            const bool live = l.live && l.sample < left(n0);
            const int j = live ? l.sample : 0;
            auto &xv = held.v[0], &gv = held.v[1], &rv = held.v[2];
            float mu[Q], rs[Q], aq[2 * Q] = {};
            load_stats(d, (n0 + j) * d.G + l.group, mu, rs);
            with_activation(d.act, [&](auto act) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (!live || l.row + k * step >= S) continue;
                    float h[V], dz[V];
                    back_values<Q>(xv[k], gv[k], d.res ? &rv[k] : nullptr, mu, rs, w, b, act, h, dz);
                    back_sum<Q>(h, dz, wq, s1, s2, aq);
                }
            });
            group_sum<TH>(aq, d, TH == 64 ? scratch : scratch + turn * 2 * Q * TH);
#pragma unroll
            for (int q = 0; q < 2 * Q; ++q) aq[q] *= inv;
            const long out = n0 * d.S * d.C;
            const int at = (j * S + l.row) * d.C + l.ch;
            forget(xv);
            forget(gv);
            forget(rv);
            with_activation(d.act, [&](auto act) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (!live || l.row + k * step >= S) continue;
                    float h[V], dz[V];
                    back_values<Q>(xv[k], gv[k], d.res ? &rv[k] : nullptr, mu, rs, w, b, act, h, dz);
                    back_store<Q>(d, out, (unsigned)(at + k * step * d.C), rs, aq, w, h, dz, (const T*)nullptr);
                }
            });
            if (AHEAD) held = next;
        }
        if (!d.dw && !d.db) continue;
        column_sum<TH>(s1, d, scratch);
        column_sum<TH>(s2, d, TH == 64 ? scratch : scratch + TH * V);
        if (TH > 64) __syncthreads();                       // before another tile's sums
        if (l.live && l.row == 0 && l.sample == 0) {
            mz::store<float, V>(d.ws + block * 2 * d.C + l.ch, s1);
            mz::store<float, V>(d.ws + block * 2 * d.C + d.C + l.ch, s2);
        }
    }
}

// ---- split ------------------------------------------------------------------------------------------------------------

// A grid of (chunks, tiles, samples); f(sample, its chunk's first and last position, lane) for each of a workgroup's parts.
struct Part {
    long n, s0, s1;
    int split, tile;
};
template <typename F>
__device__ inline void for_each_part(const Norm& d, F f) {
    for (long n = blockIdx.z; n < d.N; n += gridDim.z)
        for (int tile = blockIdx.y; tile < d.tiles; tile += gridDim.y) {
            const long s0 = blockIdx.x * d.chunk;
            f(Part{n, s0, s0 + d.chunk < d.S ? s0 + d.chunk : d.S, (int)blockIdx.x, tile});
        }
}
// where (split, piece) of a unit stands among its splits * pieces partial results
__device__ inline long part_at(const Norm& d, const Part& p, const Lane& l) {
    return ((p.n * d.units + l.g) * d.splits + p.split) * d.pieces + (d.pieces > 1 ? p.tile % d.pieces : 0);
}

constexpr int kBatch = 4;                       // vectors of a thread under way at once

// vectors of positions s, s + step, ...; past the end the first again, which counts nothing
template <typename T, int V>
__device__ inline void load_batch(Vec<T, V> (&v)[kBatch], const T* p, long stride, long s, int step, long end) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) v[k] = mz::load<T, V>(p + (s + k * step < end ? s + k * step : s) * stride);
}

// ws [N][units][splits][pieces][2][Q]: mean and sum of squared deviations of each part
template <typename T, int V, int Q>
__global__ void __launch_bounds__(kSplitThreads) norm_stats_kernel(Norm d) {
    __shared__ float scratch[2][kSplitThreads * Q];
    const int step = 1 << d.lrows;
    for_each_part(d, [&](const Part& p) {
        const Lane l = lane_of<V, Q>(d, p.tile);
        float count = 0.f, mean[Q] = {}, m2[Q] = {};
        if (l.live) {
            const T* x = static_cast<const T*>(d.x) + p.n * d.xs[0] + l.ch;
            for (long s = p.s0 + l.row; s < p.s1; s += kBatch * step) {     // a batch on its own, then merged
                Vec<T, V> v[kBatch];
                load_batch(v, x, d.xs[1], s, step, p.s1);
                float sum[Q] = {}, more = 0.f, m[Q], dev[Q] = {};
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    sum_up<Q>(v[k], l.dup, s + k * step < p.s1, [](float v, int, float p) { return p + v; }, sum);
                    more += s + k * step < p.s1 ? (float)(Q == 1 ? V - l.dup : V / Q) : 0.f;
                }
#pragma unroll
                for (int q = 0; q < Q; ++q) m[q] = sum[q] / more;
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    sum_up<Q>(v[k], l.dup, s + k * step < p.s1, [&](float v, int q, float p) { return fmaf(v - m[q], v - m[q], p); }, dev);
                const float f = more / (count + more);
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    const float e = m[q] - mean[q];
                    mean[q] = fmaf(e, f, mean[q]);
                    m2[q] += dev[q] + e * e * count * f;
                }
                count += more;
            }
        }
        const float all = (float)(p.s1 - p.s0) * (float)(Q == 1 ? l.width : V / Q);
        float v[Q], mu[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q) v[q] = count * mean[q];
        group_sum<kSplitThreads>(v, d, scratch[0]);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            mu[q] = v[q] / all;
            v[q] = count > 0.f ? fmaf(count * (mean[q] - mu[q]), mean[q] - mu[q], m2[q]) : 0.f;
        }
        group_sum<kSplitThreads>(v, d, scratch[1]);
        if (l.live && l.vec == 0 && l.row == 0) {
            float* ws = d.ws + 2 * Q * part_at(d, p, l);
            mz::store<float, Q>(ws, mu);
            mz::store<float, Q>(ws + Q, v);
        }
    });
}

template <typename T, int V, int Q>
__global__ void __launch_bounds__(kSplitThreads) norm_apply_kernel(Norm d) {
    __shared__ float scratch[2][kSplitThreads * Q];
    const int step = 1 << d.lrows;
    const float inv = 1.f / ((float)d.S * (float)d.D);
    for_each_part(d, [&](const Part& p) {
        const Lane l = lane_of<V, Q>(d, p.tile);
        const T* x = static_cast<const T*>(d.x) + p.n * d.xs[0] + l.ch;
        const T* res = d.res ? static_cast<const T*>(d.res) + p.n * d.rs[0] + l.ch : nullptr;
        // the unit's parts, over its lanes (a part's share of the values: its positions times its channels)
        const int parts = d.splits * d.pieces, lanes = 1 << (d.ldv + d.lrows), mine = (l.row << d.ldv) + l.vec;
        const float* ws = d.ws + 2 * Q * (p.n * d.units + l.g) * parts;
        const auto count = [&](int e) {
            const int split = d.pieces > 1 ? e / d.pieces : e, from = ((e - split * d.pieces) << d.ldv) * V;
            const long positions = split * d.chunk + d.chunk < d.S ? d.chunk : d.S - split * d.chunk;
            const int channels = Q > 1 ? V / Q : d.U - from < V << d.ldv ? d.U - from : V << d.ldv;
            return (float)positions * (float)channels;
        };
        float a[Q] = {}, mu[Q], rs[Q];
        if (l.unit < d.gs)
            for (int e = mine; e < parts; e += lanes) {
                const Vec<float, Q> m = mz::load<float, Q>(ws + 2 * Q * e);
#pragma unroll
                for (int q = 0; q < Q; ++q) a[q] = fmaf(count(e), m[q], a[q]);
            }
        group_sum<kSplitThreads>(a, d, scratch[0]);
#pragma unroll
        for (int q = 0; q < Q; ++q) mu[q] = a[q] * inv, a[q] = 0.f;
        if (l.unit < d.gs)
            for (int e = mine; e < parts; e += lanes) {
                const Vec<float, Q> m = mz::load<float, Q>(ws + 2 * Q * e), m2 = mz::load<float, Q>(ws + 2 * Q * e + Q);
#pragma unroll
                for (int q = 0; q < Q; ++q) a[q] += fmaf(count(e) * (m[q] - mu[q]), m[q] - mu[q], m2[q]);
            }
        group_sum<kSplitThreads>(a, d, scratch[1]);
#pragma unroll
        for (int q = 0; q < Q; ++q) rs[q] = 1.f / sqrtf(a[q] * inv + d.eps);
        if (!l.live) return;
        if (d.mean && p.split == 0 && l.vec == 0 && l.row == 0 && (d.pieces == 1 || p.tile % d.pieces == 0)) {
            mz::store<float, Q>(d.mean + p.n * d.G + l.group, mu);
            mz::store<float, Q>(d.rstd + p.n * d.G + l.group, rs);
        }
        float w[V], b[V];
        load_params<T, V>(d, l.ch, w, b);
        T* y = static_cast<T*>(d.y) + p.n * d.S * d.C + l.ch;
        with_activation(d.act, [&](auto act) {
            for (long s = p.s0 + l.row; s < p.s1; s += kBatch * step) {
                Vec<T, V> v[kBatch], r[kBatch];
                load_batch(v, x, d.xs[1], s, step, p.s1);
                if (res) load_batch(r, res, d.rs[1], s, step, p.s1);
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    if (s + k * step < p.s1) apply<Q>(v[k], res ? &r[k] : nullptr, mu, rs, w, b, act, y + (s + k * step) * d.C);
            }
        });
    });
}

// ws: sums of dz and dz h of a chunk's positions, [N * splits][2][C], then sums of dz w and dz w h of each part,
// [N][units][splits][pieces][2][Q]
template <typename T, int V, int Q>
__global__ void __launch_bounds__(kSplitThreads) norm_back_sums_kernel(Norm d) {
    __shared__ float scratch[2][kSplitThreads * (V > 2 * Q ? V : 2 * Q)];
    const int step = 1 << d.lrows;
    for_each_part(d, [&](const Part& p) {
        const Lane l = lane_of<V, Q>(d, p.tile);
        float s1[V] = {}, s2[V] = {}, w[V], b[V], wq[V], aq[2 * Q] = {};
        load_params<T, V>(d, l.ch, w, b);
#pragma unroll
        for (int i = 0; i < V; ++i) wq[i] = Q == 1 && i < l.dup ? 0.f : w[i];
        if (l.live) {
            float mu[Q], rs[Q];
            load_stats(d, p.n * d.G + l.group, mu, rs);
            const T* x = static_cast<const T*>(d.x) + p.n * d.xs[0] + l.ch;
            const T* res = d.res ? static_cast<const T*>(d.res) + p.n * d.rs[0] + l.ch : nullptr;
            const T* dy = static_cast<const T*>(d.dy) + p.n * d.ds[0] + l.ch;
            with_activation(d.act, [&](auto act) {
                for (long s = p.s0 + l.row; s < p.s1; s += kBatch * step) {
                    Vec<T, V> v[kBatch], g[kBatch], r[kBatch];
                    load_batch(v, x, d.xs[1], s, step, p.s1);
                    load_batch(g, dy, d.ds[1], s, step, p.s1);
                    if (res) load_batch(r, res, d.rs[1], s, step, p.s1);
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        if (s + k * step >= p.s1) continue;
                        float h[V], dz[V];
                        back_values<Q>(v[k], g[k], res ? &r[k] : nullptr, mu, rs, w, b, act, h, dz);
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            s1[i] += dz[i];
                            s2[i] = fmaf(dz[i], h[i], s2[i]);
                        }
                    }
                }
            });
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            aq[i * Q / V] = fmaf(s1[i], wq[i], aq[i * Q / V]);
            aq[Q + i * Q / V] = fmaf(s2[i], wq[i], aq[Q + i * Q / V]);
        }
        __syncthreads();
        group_sum<kSplitThreads>(aq, d, scratch[0]);
        column_sum<kSplitThreads>(s1, d, scratch[1]);
        column_sum<kSplitThreads>(s2, d, scratch[0]);
        if (l.live && l.row == 0) {
            float* ws = d.ws + (p.n * d.splits + p.split) * 2 * d.C + l.ch;
            mz::store<float, V>(ws, s1);
            mz::store<float, V>(ws + d.C, s2);
            if (l.vec == 0) mz::store<float, 2 * Q>(d.ws + d.N * d.splits * 2 * d.C + 2 * Q * part_at(d, p, l), aq);
        }
    });
}

template <typename T, int V, int Q>
__global__ void __launch_bounds__(kSplitThreads) norm_back_apply_kernel(Norm d) {
    __shared__ float scratch[2][2 * Q * kSplitThreads];
    const int step = 1 << d.lrows;
    const float inv = 1.f / ((float)d.S * (float)d.D);
    int turn = 0;
    for_each_part(d, [&](const Part& p) {
        const Lane l = lane_of<V, Q>(d, p.tile);
        const T* x = static_cast<const T*>(d.x) + p.n * d.xs[0] + l.ch;
        const T* res = d.res ? static_cast<const T*>(d.res) + p.n * d.rs[0] + l.ch : nullptr;
        const T* dy = static_cast<const T*>(d.dy) + p.n * d.ds[0] + l.ch;
        const int parts = d.splits * d.pieces;
        const float* ws = d.ws + d.N * d.splits * 2 * d.C + 2 * Q * (p.n * d.units + l.g) * parts;
        float aq[2 * Q] = {}, mu[Q], rs[Q];
        if (l.unit < d.gs)
            for (int e = (l.row << d.ldv) + l.vec; e < parts; e += 1 << (d.ldv + d.lrows)) {
                const Vec<float, 2 * Q> part = mz::load<float, 2 * Q>(ws + 2 * Q * e);
#pragma unroll
                for (int q = 0; q < 2 * Q; ++q) aq[q] += part[q];
            }
        group_sum<kSplitThreads>(aq, d, scratch[turn]);
        turn ^= 1;
        if (!l.live) return;
#pragma unroll
        for (int q = 0; q < 2 * Q; ++q) aq[q] *= inv;
        load_stats(d, p.n * d.G + l.group, mu, rs);
        float w[V], b[V];
        load_params<T, V>(d, l.ch, w, b);
        const long out = p.n * d.S * d.C + l.ch;
        with_activation(d.act, [&](auto act) {
            for (long s = p.s0 + l.row; s < p.s1; s += kBatch * step) {
                Vec<T, V> v[kBatch], g[kBatch], r[kBatch];
                load_batch(v, x, d.xs[1], s, step, p.s1);
                load_batch(g, dy, d.ds[1], s, step, p.s1);
                if (res) load_batch(r, res, d.rs[1], s, step, p.s1);
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    if (s + k * step >= p.s1) continue;
                    float h[V], dz[V];
                    back_values<Q>(v[k], g[k], res ? &r[k] : nullptr, mu, rs, w, b, act, h, dz);
                    back_store<Q>(d, out + (s + k * step) * d.C, 0, rs, aq, w, h, dz, (const T*)nullptr);
                }
            }
        });
    });
}

// ---- dweight, dbias ---------------------------------------------------------------------------------------------------

// ws [rows][2][C] summed over its rows: 8 columns a workgroup, 128 rows side by side, in 64 bits (sums over every position
// of a batch, which may cancel).  `first`: a launch's first column
template <typename T>
__global__ void __launch_bounds__(1024) norm_params_kernel(Norm d, long rows, int first) {
    __shared__ double part[16][8];
    const int t = threadIdx.x, c = first + blockIdx.x * 8 + (t & 7), column = c < 2 * d.C ? c : 2 * d.C - 1;
    double s = 0.0;
    for (long r = t >> 3; r < rows; r += 8 * 128) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = d.ws[(r + k * 128 < rows ? r + k * 128 : r) * 2 * d.C + column];
#pragma unroll
        for (int k = 0; k < 8; ++k) s += r + k * 128 < rows ? v[k] : 0.f;
    }
    for (int m = 8; m < 64; m <<= 1) s += __shfl_xor(s, m);
    if ((t & 63) < 8) part[t >> 6][t & 7] = s;
    __syncthreads();
    if (t < 8 && c < 2 * d.C) {
        for (int j = 1; j < 16; ++j) s += part[j][t];
        const bool which = c >= d.C;
        void* out = which ? d.dw : d.db;
        const int at = which ? c - d.C : c;
        if (!out) return;
        if (d.params_f32) static_cast<float*>(out)[at] = (float)s;
        else static_cast<T*>(out)[at] = (T)(float)s;
    }
}

// ---- launches, one file a type ----------------------------------------------------------------------------------------

template <int V>
using Int = std::integral_constant<int, V>;

template <typename T, typename F>
void with_vector(int v, int q, F f) {
    if constexpr (sizeof(T) == 2) {
        if (v == 8) return q == 8 ? f(Int<8>{}, Int<8>{}) : q == 4 ? f(Int<8>{}, Int<4>{}) : q == 2 ? f(Int<8>{}, Int<2>{}) : f(Int<8>{}, Int<1>{});
        if (v == 4) return f(Int<4>{}, Int<1>{});
    } else {
        if (v == 4) return q == 4 ? f(Int<4>{}, Int<4>{}) : q == 2 ? f(Int<4>{}, Int<2>{}) : f(Int<4>{}, Int<1>{});
    }
    if (v == 2) return q == 2 ? f(Int<2>{}, Int<2>{}) : f(Int<2>{}, Int<1>{});
    f(Int<1>{}, Int<1>{});
}
template <typename F>
void with_size(const Plan& p, F f) {                // threads, and vectors a thread, of the resident kernels
    if (p.threads == 64) {
        if (p.k <= 2) f(Int<64>{}, Int<2>{});
        else if (p.k <= 4) f(Int<64>{}, Int<4>{});
        else f(Int<64>{}, Int<8>{});
    } else if (p.threads == 256) {
        f(Int<256>{}, Int<8>{});
    } else {
        f(Int<512>{}, Int<8>{});
    }
}
inline unsigned grid_of(long total) { return (unsigned)(total < (1L << 22) ? total : 1L << 22); }

template <typename T>
void forward(const Plan& p, hipStream_t st) {
    const Norm& d = p.d;
    with_vector<T>(p.v, p.q, [&](auto v, auto q) {
        constexpr int V = v.value, Q = q.value;
        if (p.k) {
            const dim3 grid(grid_of(d.forward_blocks), d.tiles < 65535 ? d.tiles : 65535);
            with_size(p, [&](auto th, auto k) {
                if constexpr (th.value == 64 && k.value == 2) norm_forward_ahead_kernel<T, V, Q, 2><<<grid, 64, 0, st>>>(d);
                else norm_forward_kernel<T, V, Q, th.value, k.value><<<grid, th.value, 0, st>>>(d);
            });
        } else {
            const dim3 grid(d.splits, d.tiles < 65535 ? d.tiles : 65535, d.N < 65535 ? d.N : 65535);
            norm_stats_kernel<T, V, Q><<<grid, kSplitThreads, 0, st>>>(d);
            norm_apply_kernel<T, V, Q><<<grid, kSplitThreads, 0, st>>>(d);
        }
    });
}

template <typename T>
void backward(const Plan& p, hipStream_t st) {
    const Norm& d = p.d;
    const bool empty = d.N == 0 || d.S == 0;
    if (!empty)
        with_vector<T>(p.v, p.q, [&](auto v, auto q) {
            constexpr int V = v.value, Q = q.value;
            if (p.k) {
                const dim3 grid((unsigned)d.blocks, d.tiles < 65535 ? d.tiles : 65535);
                with_size(p, [&](auto th, auto k) { norm_backward_kernel<T, V, Q, th.value, k.value><<<grid, th.value, 0, st>>>(d); });
            } else {
                const dim3 grid(d.splits, d.tiles < 65535 ? d.tiles : 65535, d.N < 65535 ? d.N : 65535);
                norm_back_sums_kernel<T, V, Q><<<grid, kSplitThreads, 0, st>>>(d);
                if (d.dx || d.dres) norm_back_apply_kernel<T, V, Q><<<grid, kSplitThreads, 0, st>>>(d);
            }
        });
    const int most = 1 << 23;   // columns of a launch: a grid holds fewer than 2^32 threads side by side
    for (int c = 0; (d.dw || d.db) && c < 2 * d.C; c += most)          // of no rows: zeros
        norm_params_kernel<T><<<((2 * d.C - c < most ? 2 * d.C - c : most) + 7) / 8, 1024, 0, st>>>(d, empty ? 0 : p.k ? d.blocks : d.N * d.splits, c);
}

extern template void forward<float>(const Plan&, hipStream_t);
extern template void forward<mz::f16>(const Plan&, hipStream_t);
extern template void forward<mz::bf16>(const Plan&, hipStream_t);
extern template void backward<float>(const Plan&, hipStream_t);
extern template void backward<mz::f16>(const Plan&, hipStream_t);
extern template void backward<mz::bf16>(const Plan&, hipStream_t);

}  // namespace mz_norm
