// Cross entropy of unrolled logits against rows of the replay-target block, loss and gradient in one pass
// (include/mzhip.h).
//
// Per row, in f32, with m = max z, s = sum exp(z - m), T = sum t:
//   loss = w (sum over t != 0 of t (m - z) + T log s),   dz = w (T exp(z - m) / s - t)
// (both terms of the loss are sums of what is not negative: nothing cancels).  The target row is found by the sample's
// (position + step, game): no gathered copy of the targets exists.
//
// Bound by memory: logits and targets are read once, the gradient is written once.  A row belongs to W lanes (a power of
// two), which hold all of it: up to K chunks of V adjacent classes each, read as one access a chunk, and two rounds of
// shuffles: the maximum, then the three sums together.  A last chunk that would pass the row's end is moved back to end
// with it; its first classes are its neighbour's too, which the sums leave out and the store writes a second time, alike.
#include "mz_vec.h"
#include <cmath>

namespace {

using mz::bf16;
using mz::f16;
using mz::Vec;

constexpr int kThreads = 256;
constexpr int kMaxClasses = 4096;

struct Loss {
    long U, B, P, G;
    int C, wide, lanes, chunks;         // wide: 8-byte indexes; lanes of a row, chunks of a row
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

template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads) categorical_kernel(Loss d) {
    const int lane = threadIdx.x & (d.lanes - 1);
    const long per_block = kThreads / d.lanes;
    for (long u = blockIdx.y; u < d.U; u += gridDim.y)
        for (long b = blockIdx.x * per_block + threadIdx.x / d.lanes; b < d.B; b += gridDim.x * per_block) {
            const T* z = static_cast<const T*>(d.z) + u * d.zs[0] + b * d.zs[1];
            const float w = d.w ? d.w[u * d.ws[0] + b * d.ws[1]] : 1.f;
            const long position = d.position ? index_at(d.position, d.wide, b) : 0, game = d.game ? index_at(d.game, d.wide, b) : b;
            const bool inside = position >= 0 && position < d.P - u && game >= 0 && game < d.G;
            const float* t = d.t + (inside ? ((position + u) * d.G + game) * d.C : 0);
            Vec<T, V> zv[K];
            Vec<float, V> tv[K];
            float e[K][V], m = -INFINITY, sums[3] = {0.f, 0.f, 0.f};
            if (w != 0.f && inside) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (k * d.lanes < d.chunks && lane + k * d.lanes < d.chunks) {
                        const int c = (lane + k * d.lanes) * V < d.C - V ? (lane + k * d.lanes) * V : d.C - V;
                        zv[k] = mz::load<T, V>(z + c);
                        tv[k] = mz::load<float, V>(t + c);
                    }
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (k * d.lanes < d.chunks && lane + k * d.lanes < d.chunks)
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            e[k][i] = zv[k][i];
                            m = fmaxf(m, e[k][i] != e[k][i] ? INFINITY : e[k][i]);      // a NaN ends in every sum
                        }
            }
            for (int k = d.lanes >> 1; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
            const bool empty = w == 0.f || (inside && m == -INFINITY), live = inside && !empty;
            if (live)
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (k * d.lanes < d.chunks && lane + k * d.lanes < d.chunks) {
                        const int twice = (lane + k * d.lanes) * V - (d.C - V);         // classes that the neighbour counts
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const float below = m - e[k][i], q = tv[k][i];
                            e[k][i] = __expf(-below);
                            if (i >= twice) {
                                sums[0] += e[k][i];
                                sums[1] += q;
                                if (q != 0.f) sums[2] = fmaf(q, below, sums[2]);
                            }
                        }
                    }
            for (int k = d.lanes >> 1; k; k >>= 1)
#pragma unroll
                for (int i = 0; i < 3; ++i) sums[i] += __shfl_xor(sums[i], k);
            const long row = u * d.B + b;
            if (d.loss && lane == 0) d.loss[row] = empty ? 0.f : inside ? w * fmaf(sums[1], logf(sums[0]), sums[2]) : NAN;
            if (d.grad) {
                const float f = d.g ? w * d.g[u * d.gs[0] + b * d.gs[1]] : w, p = sums[1] / sums[0];
                T* out = static_cast<T*>(d.grad) + row * d.C;
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (k * d.lanes < d.chunks && lane + k * d.lanes < d.chunks) {
                        const int c = (lane + k * d.lanes) * V < d.C - V ? (lane + k * d.lanes) * V : d.C - V;
                        float r[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) r[i] = empty ? 0.f : inside ? f * fmaf(p, e[k][i], -tv[k][i]) : NAN;
                        mz::store<T, V>(out + c, r);
                    }
            }
        }
}

template <typename T>
void launch(Loss d, hipStream_t st) {
    // four classes a chunk, two chunks a lane; more chunks only where a wavefront's lanes are used up
    const int v = d.C >= 4 ? 4 : 1;
    d.chunks = (d.C + v - 1) / v;
    d.lanes = 1;
    while (d.lanes < 64 && d.lanes * 2 < d.chunks) d.lanes <<= 1;
    const int k = (d.chunks + d.lanes - 1) / d.lanes;
    const long blocks = (d.B + kThreads / d.lanes - 1) / (kThreads / d.lanes);
    const dim3 grid((unsigned)(blocks < 1L << 20 ? blocks : 1L << 20), (unsigned)(d.U < 65535 ? d.U : 65535));
    if (v == 1) categorical_kernel<T, 1, 2><<<grid, kThreads, 0, st>>>(d);
    else if (k <= 2) categorical_kernel<T, 4, 2><<<grid, kThreads, 0, st>>>(d);
    else if (k <= 4) categorical_kernel<T, 4, 4><<<grid, kThreads, 0, st>>>(d);
    else if (k <= 8) categorical_kernel<T, 4, 8><<<grid, kThreads, 0, st>>>(d);
    else categorical_kernel<T, 4, 16><<<grid, kThreads, 0, st>>>(d);
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
    MZ_REQUIRE(logits && (targets || c->target_positions * c->target_games == 0), "logits/targets is NULL");
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
    if (!game && !position && d.P == d.U && d.G == d.B && even(d.zs) && (!d.w || even(d.ws)) && (!d.g || even(d.gs))) {
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
