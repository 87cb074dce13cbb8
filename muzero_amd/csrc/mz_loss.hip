// Cross entropy of unrolled logits against rows of the replay-target block, loss and gradient in one pass
// (include/mzhip.h).
//
// Per row, in f32, with m = max z, s = sum exp(z - m), T = sum t:
//   loss = w (sum over t != 0 of t (m - z) + T log s),   dz = w (T exp(z - m) / s - t)
// (both terms of the loss are sums of what is not negative: nothing cancels; exp(-d) from the hardware's exponential of a
// rounded product is off by (1.3 d + 2) 2^-24 of itself, at most 2^-23 of the largest).  The target row is found by the
// sample's (position + step, game): no gathered copy of the targets exists.
//
// Bound by memory: logits and targets are read once, the gradient is written once.  A row belongs to W lanes (a power of
// two), which hold all of it: up to K chunks of V adjacent classes each, read as one access a chunk, and two rounds of
// shuffles: the maximum, then the three sums together.  With K and what is asked for known to the compiler: at 552 vector
// operations a row, in loops up to the most chunks, arithmetic took 289 us where it now hides behind the memory.  6 x 16384
// rows of 601 classes, f16, against a block of 83 MB: 74 us (323 MB: 4.4 TB/s); 6 x 2048 rows of 362, bf16, loss alone and
// gradient alone, as autograd calls them: 9.2 and 9.8 us.
#include "mz_vec.h"
#include <cmath>

namespace {

using mz::bf16;
using mz::f16;
using mz::Vec;

constexpr int kThreads = 256;
constexpr int kMaxClasses = 4096;
constexpr float kLog2e = 1.4426950409f;

struct Loss {
    long U, B, P, G, u0;                // u0: first step of a launch
    int C, wide, lanes, last;           // wide: 8-byte indexes; lanes of a row, a lane's last chunk
    uint32_t block0;                    // workgroups of a step that earlier launches had
    long zs[2], ws[2], gs[2];
    const void* z;
    const float *t, *w, *g;
    const void *game, *position;
    float* loss;
    void* grad;
};

__device__ inline long index_at(const void* p, int wide, long i) {
    return wide ? (long)static_cast<const int64_t*>(p)[i] : (long)static_cast<const int32_t*>(p)[i];
}

// K chunks a lane: exactly K up to four, then up to K.
template <typename T, int V, int K, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(kThreads) categorical_kernel(Loss d) {
    const int lane = threadIdx.x & (d.lanes - 1), last = K <= 4 ? K - 1 : d.last;
    const long u = d.u0 + blockIdx.y, b = (d.block0 + blockIdx.x) * (long)(kThreads / d.lanes) + threadIdx.x / d.lanes;
    if (b >= d.B) return;                                    // all lanes of a row
    // The lane's chunk k.  One that would pass the row's end is moved back to end with it: of the last chunk, the first `twice`
    // classes belong to another lane (all V or more: the lane has no such chunk) and neither count nor are stored.
    const auto start = [&](int k) { return (lane + k * d.lanes) * V < d.C - V ? (lane + k * d.lanes) * V : d.C - V; };
    const int twice = (lane + last * d.lanes) * V - start(last);
    const T* z = static_cast<const T*>(d.z) + u * d.zs[0] + b * d.zs[1];
    Vec<T, V> zv[K];
    Vec<float, V> tv[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k <= last) zv[k] = mz::load<T, V>(z + start(k));
    const float w = d.w ? d.w[u * d.ws[0] + b * d.ws[1]] : 1.f;
    const long position = d.position ? index_at(d.position, d.wide, b) : 0, game = d.game ? index_at(d.game, d.wide, b) : b;
    const bool inside = position >= 0 && position < d.P - u && game >= 0 && game < d.G;
    if (inside) {
        const float* t = d.t + ((position + u) * d.G + game) * d.C;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k <= last) tv[k] = mz::load<float, V>(t + start(k));
    }
    float e[K][V], m = -INFINITY;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k <= last) {
#pragma unroll
            for (int i = 0; i < V; ++i) e[k][i] = zv[k][i];
            if (k == last)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    e[k][i] = i < twice ? -INFINITY : e[k][i];
                    tv[k].w[i] = i < twice ? 0 : tv[k].w[i];
                }
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmaxf(m, e[k][i]);
        }
    for (int k = d.lanes >> 1; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    bool empty = w == 0.f;
    if (m == -INFINITY) {                                    // nothing, or only NaN, above the lowest: a NaN is no empty row
        float nan = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k <= last)
#pragma unroll
                for (int i = 0; i < V; ++i) nan += e[k][i] != e[k][i] ? 1.f : 0.f;
        for (int k = d.lanes >> 1; k; k >>= 1) nan += __shfl_xor(nan, k);
        empty |= inside && nan == 0.f;
    }
    const bool live = inside && !empty;
    float s = 0.f, total = 0.f, l = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k <= last)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float below = m - e[k][i];             // before the factor, which the type's lowest value would overflow
                // a class without target adds nothing, also where its logit is -inf
                if (LOSS) l = fmaf(tv[k][i], tv[k][i] != 0.f ? below : 0.f, l);
                e[k][i] = __builtin_amdgcn_exp2f(below * -kLog2e);
                s += e[k][i];
                total += tv[k][i];
            }
    for (int k = d.lanes >> 1; k; k >>= 1) {
        s += __shfl_xor(s, k);
        total += __shfl_xor(total, k);
        if (LOSS) l += __shfl_xor(l, k);
    }
    const long row = u * d.B + b;
    if (LOSS && lane == 0) d.loss[row] = empty ? 0.f : inside ? w * fmaf(total, logf(s), l) : NAN;
    if (GRAD) {
        const float f = d.g ? w * d.g[u * d.gs[0] + b * d.gs[1]] : w, p = f * (total / s), dead = empty ? 0.f : NAN;
        T* out = static_cast<T*>(d.grad) + row * d.C;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k <= last) {
                float r[V];
#pragma unroll
                for (int i = 0; i < V; ++i) r[i] = live ? fmaf(p, e[k][i], -f * tv[k][i]) : dead;
                if (k < last || twice <= 0) mz::store<T, V>(out + start(k), r);
                else
#pragma unroll
                    for (int i = 1; i < V; ++i)
                        if (i >= twice) out[start(k) + i] = (T)r[i];
            }
    }
}

template <typename T, int V, int K>
void launch(const Loss& d, dim3 grid, hipStream_t st) {
    if (d.loss && d.grad) categorical_kernel<T, V, K, true, true><<<grid, kThreads, 0, st>>>(d);
    else if (d.loss) categorical_kernel<T, V, K, true, false><<<grid, kThreads, 0, st>>>(d);
    else categorical_kernel<T, V, K, false, true><<<grid, kThreads, 0, st>>>(d);
}

template <typename T>
void launch(Loss d, hipStream_t st) {
    // four classes a chunk, two chunks a lane; more chunks only where a wavefront's lanes are used up
    const int v = d.C >= 4 ? 4 : 1, chunks = (d.C + v - 1) / v;
    d.lanes = 1;
    while (d.lanes < 64 && d.lanes * 2 < chunks) d.lanes <<= 1;
    const int k = (chunks + d.lanes - 1) / d.lanes;
    d.last = k - 1;
    const long rows = kThreads / d.lanes;
    // what a grid may hold: fewer than 2^32 threads side by side, and 65535 steps
    const long blocks = (d.B + rows - 1) / rows, most_blocks = 1 << 23, most_steps = 65535;
    for (; d.u0 < d.U; d.u0 += most_steps)
        for (long first = 0; first < blocks; first += most_blocks) {
            d.block0 = (uint32_t)first;
            const dim3 grid((unsigned)(blocks - first < most_blocks ? blocks - first : most_blocks),
                            (unsigned)(d.U - d.u0 < most_steps ? d.U - d.u0 : most_steps));
            if (v == 1) k == 1 ? launch<T, 1, 1>(d, grid, st) : launch<T, 1, 2>(d, grid, st);
            else if (k == 1) launch<T, 4, 1>(d, grid, st);
            else if (k == 2) launch<T, 4, 2>(d, grid, st);
            else if (k == 3) launch<T, 4, 3>(d, grid, st);
            else if (k == 4) launch<T, 4, 4>(d, grid, st);
            else if (k <= 8) launch<T, 4, 8>(d, grid, st);
            else launch<T, 4, 16>(d, grid, st);
        }
}

}  // namespace

extern "C" int mz_categorical_loss(void* stream, const mz_categorical_t* c, const void* logits, const float* targets,
                                   const void* game, const void* position, const float* weights, const float* dloss,
                                   float* out_loss, void* out_dlogits) {
    MZ_REQUIRE(c != nullptr, "config is NULL");
    MZ_REQUIRE(c->unroll >= 0 && c->batch >= 0 && c->target_positions >= 0 && c->target_games >= 0, "bad sizes in mz_categorical_t");
    MZ_REQUIRE(c->classes >= 1 && c->classes <= kMaxClasses, "classes must be in [1, %d], got %d", kMaxClasses, c->classes);
    MZ_REQUIRE(mz::dtype_size(c->dtype), "dtype %d is not one of mz_dtype", c->dtype);
    MZ_REQUIRE(c->index_bytes == 4 || c->index_bytes == 8 || (!game && !position), "index_bytes must be 4 or 8");
    MZ_REQUIRE(c->batch == 0 || c->unroll <= (int64_t(1) << 48) / c->classes / c->batch, "the logits have more than 2^48 elements");
    MZ_REQUIRE(c->target_games == 0 || c->target_positions <= (int64_t(1) << 48) / c->classes / c->target_games,
               "the targets have more than 2^48 elements");
    if (c->unroll == 0 || c->batch == 0) return MZ_OK;
    MZ_REQUIRE(c->batch <= int64_t(1) << 31 && c->unroll <= int64_t(1) << 31, "more than 2^31 rows of a step, or steps");
    MZ_REQUIRE(logits && (targets || c->target_positions * c->target_games == 0), "logits/targets is NULL");
    MZ_REQUIRE(mz::aligned(mz::dtype_size(c->dtype), {logits, out_dlogits}) && mz::aligned(sizeof(float), {targets, weights, dloss, out_loss}) &&
                   (c->index_bytes == 0 || mz::aligned(c->index_bytes, {game, position})),
               "an array is not aligned to its type");
    if (!out_loss && !out_dlogits) return MZ_OK;
    Loss d = {};
    d.U = c->unroll;
    d.B = c->batch;
    d.P = c->target_positions;
    d.G = c->target_games;
    d.C = c->classes;
    d.wide = c->index_bytes == 8;
    for (int i = 0; i < 2; ++i) {
        d.zs[i] = c->logits_strides[i];
        d.ws[i] = c->weight_strides[i];
        d.gs[i] = c->dloss_strides[i];
    }
    d.z = logits;
    d.t = targets;
    d.w = weights;
    d.g = dloss;
    d.game = game;
    d.position = position;
    d.loss = out_loss;
    d.grad = out_dlogits;
    // rows that lie evenly behind one another, each with its own target row, are one long step
    const auto even = [&](const long* stride) { return stride[0] == d.B * stride[1]; };
    if (!game && !position && d.P == d.U && d.G == d.B && d.U * d.B <= 1L << 31 && even(d.zs) && (!d.w || even(d.ws)) && (!d.g || even(d.gs))) {
        d.B *= d.U;
        d.G = d.B;
        d.U = d.P = 1;
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (c->dtype == MZ_F32) launch<float>(d, st);
    else if (c->dtype == MZ_F16) launch<f16>(d, st);
    else launch<bf16>(d, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return mz::fail(MZ_ERR_HIP, "mz_categorical_loss launch failed: %s", hipGetErrorString(e));
    return MZ_OK;
}
