// The C entries of group norm: checks, and the choice of a way through (mz_norm_dev.h).
#include "mz_norm_dev.h"
#include <cmath>

namespace {

using mz_norm::kMostSplits;
using mz_norm::kSplitThreads;
using mz_norm::Norm;
using mz_norm::Plan;

// The widest vectors of at most 16 bytes.  A group of V channels or more is cut into such vectors, its last one moved back to
// end with it; smaller groups stand side by side in a vector where their size divides it, the last vector moved back to end
// with the sample (10958 x 25 x 146 bf16 in groups of 2: backward 199 us in vectors of 2, 120 in vectors of 8).
void choose_vector(const mz_group_norm_t* c, int* v, int* q) {
    const int most = 16 / mz::dtype_size(c->dtype), d = c->channels / c->groups;
    *q = 1;
    *v = most;
    if (d >= most) return;
    if ((d & (d - 1)) == 0 && c->channels >= most) *q = most / d;
    else if (d == 1 && c->channels > 1) *v = *q = 2;
    else
        while (*v > d) *v >>= 1;
}

int check(const mz_group_norm_t* c) {
    MZ_REQUIRE(c != nullptr, "config is NULL");
    MZ_REQUIRE(c->batch >= 0 && c->positions >= 0 && c->channels >= 1 && c->channels <= MZ_GROUP_NORM_MAX_CHANNELS, "bad sizes in mz_group_norm_t");
    MZ_REQUIRE(c->groups >= 1 && c->channels % c->groups == 0, "groups (%d) must divide channels (%d)", c->groups, c->channels);
    MZ_REQUIRE(mz::dtype_size(c->dtype), "dtype %d is not one of mz_dtype", c->dtype);
    MZ_REQUIRE(c->param_dtype == MZ_F32 || c->param_dtype == c->dtype, "param_dtype must be MZ_F32 or dtype");
    MZ_REQUIRE(c->activation >= MZ_ACT_NONE && c->activation <= MZ_ACT_TANH, "activation %d is not one of mz_activation", c->activation);
    MZ_REQUIRE(c->eps >= 0 && std::isfinite(c->eps), "eps must be finite and >= 0");
    MZ_REQUIRE(c->batch == 0 || c->positions <= (int64_t(1) << 48) / c->channels / c->batch, "the state has more than 2^48 elements");
    return MZ_OK;
}

int log2_up(long v) {
    int l = 0;
    while ((1L << l) < v) ++l;
    return l;
}

// Lanes of a workgroup of `threads`, and the vectors a thread then holds of a tile.  The split kernels take one sample a
// workgroup: with `several` false all lanes that units leave are positions, the ones past the last idle.
int lay_out(Norm& d, int v, int item, int threads, bool several) {
    const int dv = (d.U + v - 1) / v, lth = log2_up(threads), units = d.units;
    d.pieces = 1;
    d.samples = 1;
    d.ldv = log2_up(dv);
    if (d.ldv > lth) {                              // a unit wider than the workgroup: pieces of it
        d.ldv = lth;
        d.pieces = (dv + threads - 1) / threads;
        d.lgs = d.lrows = 0;
        d.gs = 1;
        d.tiles = units * d.pieces;
        return 0;
    }
    // Units of a tile and positions side by side: the units of a 128-byte line, or more, and as many positions as there are
    // lanes, or fewer beside more samples, whatever leaves fewest lanes idle over the positions, the padding of the tiles and
    // the samples -- unless there are too few workgroups to begin with, or a thread would then hold more vectors than the
    // kernels that read ahead do (nine positions on eight rows of lanes: two vectors a thread, nine sixteenths of them live; on
    // four rows three, three quarters).  The half a step is what sums over the lanes cost: they are shared by more vectors.
    // Backward: 34722 x 9 x 128 f32 in groups of 4 148 -> 116 us; 277777 x 9 x 16 bf16 137 -> 87; 104166 x 3 x 128 f32 179 -> 110.
    const int all = log2_up(units), room = lth - d.ldv, most = all < room ? all : room;
    const int line = log2_up((128 + (long)d.U * item - 1) / ((long)d.U * item)), least = line < most ? line : most, ls = log2_up(d.S);
    double best = INFINITY;
    long k = 0;
    for (int lgs = least; lgs <= most; ++lgs) {
        const int tiles = (units + (1 << lgs) - 1) >> lgs, widest = room - lgs < ls || !several ? room - lgs : ls;
        for (int lrows = widest; lrows >= (several ? 0 : widest); --lrows) {
            const long steps = (d.S + (1L << lrows) - 1) >> lrows, samples = 1L << (room - lgs - lrows);
            const double cost = (double)tiles * ((double)steps + 0.5) / (double)samples;
            const bool first = lgs == least && lrows == widest;
            if (!first && (cost >= best || steps > 4 || d.N * tiles < 2048 * (lrows < widest ? samples : 1))) continue;
            best = cost;
            k = steps;
            d.lgs = lgs;
            d.lrows = lrows;
        }
    }
    d.samples = 1 << (lth - d.ldv - d.lgs - d.lrows);
    d.tiles = (units + (1 << d.lgs) - 1) >> d.lgs;
    d.gs = (units + d.tiles - 1) / d.tiles;         // tiles of even size
    d.tiles = (units + d.gs - 1) / d.gs;
    return k < 1 << 20 ? (int)k : 1 << 20;
}

bool spans(int64_t stride, int64_t steps, int64_t most) { return steps == 0 || (stride >= 0 && stride <= most / steps); }

Plan plan(const mz_group_norm_t* c) {
    Plan p = {};
    Norm& d = p.d;
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
    choose_vector(c, &p.v, &p.q);
    d.U = p.q > 1 ? p.v : d.D;
    d.units = (d.C + d.U - 1) / d.U;
    const int v = p.v, item = mz::dtype_size(c->dtype);
    // the smallest workgroup whose registers hold a tile, one wavefront without barriers if it may be
    for (const int threads : {64, 256, 512}) {
        const int k = lay_out(d, v, item, threads, true);
        const int64_t reach = (int64_t(1) << 31) / item - d.C;                 // elements that a 32-bit byte offset spans
        bool near = true;
        const long last = (d.samples < d.N ? d.samples : d.N) - 1;             // of a workgroup's samples
        for (const long* s : {d.xs, d.rs, d.ds}) near &= spans(s[0], last, reach / 2) && spans(s[1], d.S - 1, reach / 2);
        near &= spans(d.S * d.C, d.samples, reach);
        if (k < 1 || k > 8 || !near) continue;
        p.threads = threads;
        p.k = k;
        const long sets = (d.N + d.samples - 1) / d.samples, fill = 2048 / (threads / 64) / d.tiles;
        d.blocks = sets < fill ? sets : fill > 1 ? fill : 1;                   // eight wavefronts a CU
        // twenty wavefronts a CU, which read ahead; 312500 x 128 bf16: 44 us, with a wavefront a set of samples 60
        const long ahead = 5120 / d.tiles;
        d.forward_blocks = threads > 64 || k > 2 || sets < ahead ? sets : ahead > 1 ? ahead : 1;
        d.splits = 1;
        return p;
    }
    lay_out(d, v, item, kSplitThreads, false);
    p.threads = kSplitThreads;
    p.k = 0;
    const long tiles = d.N * d.tiles > 0 ? d.N * d.tiles : 1, most = (d.S + (8L << d.lrows) - 1) / (8L << d.lrows);
    long splits = (2048 + tiles - 1) / tiles;                      // two thousand workgroups, eight vectors a thread or more
    if (splits > most) splits = most;
    if (splits > kMostSplits) splits = kMostSplits;
    if (splits < 1) splits = 1;
    d.chunk = (d.S + splits - 1) / splits;
    d.splits = d.chunk ? (int)((d.S + d.chunk - 1) / d.chunk) : 1;
    return p;
}

int64_t workspace_of(const Plan& p, bool backward) {
    const Norm& d = p.d;
    if (d.N == 0 || d.S == 0) return 0;
    const int64_t parts = p.k ? 0 : d.N * d.units * p.q * d.splits * d.pieces * 2;
    if (!backward) return parts * (int64_t)sizeof(float);
    return ((p.k ? d.blocks : d.N * d.splits) * 2 * d.C + parts) * (int64_t)sizeof(float);
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return mz::fail(MZ_ERR_HIP, "%s launch failed: %s", what, hipGetErrorString(e));
    return MZ_OK;
}

void run(int dtype, const Plan& p, bool backward, hipStream_t st) {
    if (dtype == MZ_F32) backward ? mz_norm::backward<float>(p, st) : mz_norm::forward<float>(p, st);
    else if (dtype == MZ_F16) backward ? mz_norm::backward<mz::f16>(p, st) : mz_norm::forward<mz::f16>(p, st);
    else backward ? mz_norm::backward<mz::bf16>(p, st) : mz_norm::forward<mz::bf16>(p, st);
}

}  // namespace

extern "C" {

int64_t mz_group_norm_workspace(const mz_group_norm_t* c, int32_t backward) {
    const int bad = check(c);
    return bad ? bad : workspace_of(plan(c), backward != 0);
}

int mz_debug_group_norm_layout(const mz_group_norm_t* c, int32_t* out8_host) {
    const int bad = check(c);
    if (bad) return bad;
    MZ_REQUIRE(out8_host, "out8_host is NULL");
    const Plan p = plan(c);
    const Norm& d = p.d;
    const int32_t out[8] = {p.threads, p.k, d.samples, 1 << d.lrows, 1 << d.lgs, 1 << d.ldv, d.pieces, d.splits};
    for (int i = 0; i < 8; ++i) out8_host[i] = out[i];
    return MZ_OK;
}

int mz_group_norm_forward(void* stream, const mz_group_norm_t* c, const void* x, const void* residual, const void* weight,
                          const void* bias, void* out_y, float* out_mean, float* out_rstd, void* workspace,
                          int64_t workspace_bytes) {
    const int bad = check(c);
    if (bad) return bad;
    if (c->batch == 0 || c->positions == 0) return MZ_OK;
    MZ_REQUIRE(x && out_y, "x/out_y is NULL");
    MZ_REQUIRE(!out_mean == !out_rstd, "out_mean and out_rstd: both or neither");
    Plan p = plan(c);
    const int64_t need = workspace_of(p, false);
    MZ_REQUIRE(workspace_bytes >= need && (workspace || !need), "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    MZ_REQUIRE(mz::aligned(mz::dtype_size(c->dtype), {x, residual, out_y}) && mz::aligned(mz::dtype_size(c->param_dtype), {weight, bias}) &&
                   mz::aligned(sizeof(float), {out_mean, out_rstd, workspace}),
               "an array is not aligned to its type");
    Norm& d = p.d;
    d.x = x;
    d.res = residual;
    d.w = weight;
    d.b = bias;
    d.y = out_y;
    d.mean = out_mean;
    d.rstd = out_rstd;
    d.ws = static_cast<float*>(workspace);
    run(c->dtype, p, false, static_cast<hipStream_t>(stream));
    return launched("mz_group_norm_forward");
}

int mz_group_norm_backward(void* stream, const mz_group_norm_t* c, const void* x, const void* residual, const void* weight,
                           const void* bias, const float* mean, const float* rstd, const void* dy, void* out_dx,
                           void* out_dresidual, void* out_dweight, void* out_dbias, void* workspace, int64_t workspace_bytes) {
    const int bad = check(c);
    if (bad) return bad;
    Plan p = plan(c);
    const int64_t need = workspace_of(p, true);
    const bool empty = c->batch == 0 || c->positions == 0;
    MZ_REQUIRE(empty || (x && mean && rstd && dy), "x/mean/rstd/dy is NULL");
    MZ_REQUIRE(workspace_bytes >= need && (workspace || !need), "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    MZ_REQUIRE(mz::aligned(mz::dtype_size(c->dtype), {x, residual, dy, out_dx, out_dresidual}) &&
                   mz::aligned(mz::dtype_size(c->param_dtype), {weight, bias, out_dweight, out_dbias}) &&
                   mz::aligned(sizeof(float), {mean, rstd, workspace}),
               "an array is not aligned to its type");
    Norm& d = p.d;
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
    run(c->dtype, p, true, static_cast<hipStream_t>(stream));
    return launched("mz_group_norm_backward");
}

}  // extern "C"
