// Cross entropy of unrolled logits against rows of the replay-target block, loss and gradient in one pass
// (include/mzhip.h).
//
// Per row, in f32:  m = max z, s = sum exp(z - m), loss = w sum_{t != 0} t (m - z + log s),
//                   dz = w (sum(t) exp(z - m) / s - t)
// The target row is found by the sample's (position + step, game): no gathered copy of the targets exists.
#include "mz_vec.h"
#include <cmath>

namespace {

using mz::bf16;
using mz::f16;

constexpr int kThreads = 256;
constexpr int kMaxClasses = 4096;

struct Loss {
    long U, B, P, G;
    int C, wide;                        // wide: 8-byte indexes
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

// one wavefront a row
template <typename T>
__global__ void __launch_bounds__(kThreads) categorical_kernel(Loss d) {
    const int lane = threadIdx.x & 63;
    const long rows = d.U * d.B, step = (long)gridDim.x * (kThreads / 64);
    for (long row = blockIdx.x * (long)(kThreads / 64) + (threadIdx.x >> 6); row < rows; row += step) {
        const long u = row / d.B, b = row - u * d.B;
        const float w = d.w ? d.w[u * d.ws[0] + b * d.ws[1]] : 1.f;
        const long position = d.position ? index_at(d.position, d.wide, b) : 0, game = d.game ? index_at(d.game, d.wide, b) : b;
        const bool inside = position >= 0 && position < d.P - u && game >= 0 && game < d.G;
        const T* z = static_cast<const T*>(d.z) + u * d.zs[0] + b * d.zs[1];
        const float* t = d.t + (inside ? ((position + u) * d.G + game) * d.C : 0);
        float m = -INFINITY, s = 0.f, l = 0.f, sum = 0.f;
        bool nan = !inside;
        if (w != 0.f && inside) {
            for (int c = lane; c < d.C; c += 64) {
                const float v = (float)z[c];
                nan |= v != v;
                m = fmaxf(m, v);
            }
            for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
            nan = __any(nan);
        }
        const bool empty = w == 0.f || (inside && !nan && m == -INFINITY);
        float log_s = 0.f;
        if (!empty && !nan) {
            for (int c = lane; c < d.C; c += 64) s += __expf((float)z[c] - m);
            s = mz::wave_sum(s);
            log_s = logf(s);
            for (int c = lane; c < d.C; c += 64) {
                const float q = t[c];
                sum += q;
                if (q != 0.f) l = fmaf(q, (m - (float)z[c]) + log_s, l);
            }
            l = mz::wave_sum(l);
            sum = mz::wave_sum(sum);
        }
        if (d.loss && lane == 0) d.loss[row] = empty ? 0.f : nan ? NAN : w * l;
        if (d.grad) {
            const float f = d.g ? w * d.g[u * d.gs[0] + b * d.gs[1]] : w, p = sum / s;
            T* out = static_cast<T*>(d.grad) + row * d.C;
            for (int c = lane; c < d.C; c += 64)
                out[c] = (T)(empty ? 0.f : nan ? NAN : f * (p * __expf((float)z[c] - m) - t[c]));
        }
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
    const long blocks = (d.U * d.B + kThreads / 64 - 1) / (kThreads / 64);
    const unsigned grid = (unsigned)(blocks < (1L << 20) ? blocks : 1L << 20);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (c->dtype == MZ_F32) categorical_kernel<float><<<grid, kThreads, 0, st>>>(d);
    else if (c->dtype == MZ_F16) categorical_kernel<f16><<<grid, kThreads, 0, st>>>(d);
    else categorical_kernel<bf16><<<grid, kThreads, 0, st>>>(d);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return mz::fail(MZ_ERR_HIP, "mz_categorical_loss launch failed: %s", hipGetErrorString(e));
    return MZ_OK;
}
