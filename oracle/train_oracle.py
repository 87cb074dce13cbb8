"""Plain NumPy restatement in 64 bits of the training operators (muzero_amd/layers.py, muzero_amd/training.py), with bounds
on what rounding may do to a 32-bit evaluation of the same formulas."""
import math

import numpy as np

U32 = 2.0 ** -24                       # half a step of float32, relative


def _erf(z):
    return np.vectorize(math.erf, otypes=[np.float64])(z) if z.size else z


def act(z, activation):
    if activation == 'relu':
        return np.maximum(z, 0)
    if activation == 'silu':
        return z / (1 + np.exp(-z))
    if activation == 'gelu':
        return 0.5 * z * (1 + _erf(z / math.sqrt(2)))
    return np.tanh(z) if activation == 'tanh' else z


def act_slope(z, activation):
    if activation == 'relu':
        return (z > 0).astype(np.float64)
    if activation == 'silu':
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    if activation == 'gelu':
        return 0.5 * (1 + _erf(z / math.sqrt(2))) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return 1 - np.tanh(z) ** 2 if activation == 'tanh' else np.ones_like(z)


class GroupNormOracle:
    """x [N, S, C]; every attribute in 64 bits."""

    def __init__(self, x, groups, weight=None, bias=None, eps=1e-5, activation=None, residual=None):
        x = np.asarray(x, np.float64)
        N, S, C = x.shape
        self.shape, self.groups, self.activation = x.shape, groups, activation
        self.w = np.ones(C) if weight is None else np.asarray(weight, np.float64)
        self.b = np.zeros(C) if bias is None else np.asarray(bias, np.float64)
        self.res = np.zeros_like(x) if residual is None else np.asarray(residual, np.float64)
        g = x.reshape(N, S, groups, -1)
        mean = g.mean((1, 3), keepdims=True)
        var = ((g - mean) ** 2).mean((1, 3), keepdims=True)
        r = 1 / np.sqrt(var + eps)
        spread = lambda a: np.broadcast_to(a, g.shape).reshape(x.shape)
        self.h, self.r = spread((g - mean) * r), spread(r)
        self.z = self.h * self.w + self.b + self.res
        self.y = act(self.z, activation)
        # Rounding of a 32-bit evaluation, with up to `depth` additions behind one another: the mean is off by depth steps of
        # the largest value, the scale by depth + 8 relative steps, h by both.
        depth = 64
        top = np.abs(g).max((1, 3), keepdims=True) if S else np.abs(g)
        self.depth = depth
        off_var = 2 * depth * U32 * (var + top * np.sqrt(var) * U32)
        self.off_h = spread(r) * spread(depth * U32 * top) + np.abs(self.h) * (spread(off_var / (2 * (var + eps))) + 12 * U32)
        self.off_z = np.abs(self.w) * self.off_h + 4 * U32 * (np.abs(self.h * self.w) + np.abs(self.b) + np.abs(self.res))
        # no slope is above 1.13; exp, erf and tanh are within 8 steps of their terms' size
        self.off_y = 1.13 * self.off_z + 8 * U32 * (np.abs(self.z) if activation else 0)

    def backward(self, dy):
        N, S, C = self.shape
        n = S * (C // self.groups)
        dy = np.asarray(dy, np.float64)
        dz = dy * act_slope(self.z, self.activation)
        per = lambda a: a.reshape(N, S, self.groups, -1)
        mean = lambda a: np.broadcast_to(per(a).mean((1, 3), keepdims=True), per(a).shape).reshape(a.shape)
        g = dz * self.w
        a, q = mean(g), mean(g * self.h)
        out = dict(dresidual=dz, dbias=dz.sum((0, 1)), dweight=(dz * self.h).sum((0, 1)), dx=self.r * (g - a - q * self.h))
        # a slope is off by the argument's error times its own slope (at most 0.8), relu's not at all away from 0
        depth = self.depth
        off_dz = np.abs(dy) * ((0.8 * self.off_z if self.activation not in (None, 'relu') else 0) + 12 * U32)
        if self.activation is None:
            off_dz = np.zeros_like(dz)
        off_dzh = np.abs(self.h) * off_dz + np.abs(dz) * self.off_h
        off_g = np.abs(self.w) * off_dz
        off_a = mean(off_g) + depth * U32 * mean(np.abs(g))
        off_q = mean(np.abs(self.w) * off_dzh) + depth * U32 * mean(np.abs(g * self.h))
        size = np.abs(g) + np.abs(a) + np.abs(q * self.h)
        off_r = self.off_h / np.maximum(np.abs(self.h), 1)       # relative, of the scale
        off = dict(dresidual=off_dz, dbias=off_dz.sum((0, 1)) + 2 * depth * U32 * np.abs(dz).sum((0, 1)),
                   dweight=off_dzh.sum((0, 1)) + 2 * depth * U32 * np.abs(dz * self.h).sum((0, 1)),
                   dx=self.r * (off_g + off_a + np.abs(self.h) * off_q + np.abs(q) * self.off_h + size * (8 * U32 + off_r)))
        return out, off


def categorical(logits, targets, weights=None, dloss=None):
    """Rows [R, C] -> loss [R], gradient [R, C] of sum(dloss * loss) (dloss None = ones)."""
    z, t = np.asarray(logits, np.float64), np.asarray(targets, np.float64)
    w = np.ones(z.shape[0]) if weights is None else np.asarray(weights, np.float64)
    loss, grad = np.zeros(z.shape[0]), np.zeros_like(z)
    for i in range(z.shape[0]):
        if w[i] == 0 or (z[i] == -np.inf).all():
            continue
        if np.isnan(z[i]).any() or np.isposinf(z[i]).any():
            loss[i], grad[i] = np.nan, np.nan
            continue
        m = z[i].max()
        e = np.exp(z[i] - m)
        live = t[i] != 0
        with np.errstate(invalid='ignore'):
            loss[i] = w[i] * (t[i][live] * (m - z[i][live] + math.log(e.sum()))).sum()
        grad[i] = w[i] * (t[i].sum() * e / e.sum() - t[i]) * (1 if dloss is None else dloss[i])
    return loss, grad


def categorical_bounds(logits, targets, weights=None, dloss=None):
    """Bounds on the rounding of a 32-bit evaluation of categorical(): with m the maximum and d = m - z, exp(-d) is off by
    (d + 4) relative steps, the sum of C of them by depth more, its logarithm by as much absolutely."""
    z, t = np.asarray(logits, np.float64), np.abs(np.asarray(targets, np.float64))
    w = np.ones(z.shape[0]) if weights is None else np.abs(np.asarray(weights, np.float64))
    depth = 64 + 16                                # values of one lane behind one another, and the tree over the lanes
    m = z.max(-1, keepdims=True)
    with np.errstate(invalid='ignore'):
        d = np.where(np.isfinite(z), m - z, 0.0)
        e = np.where(np.isfinite(z), np.exp(z - m), 0.0)
        s = e.sum(-1, keepdims=True)
        off_s = ((d + 4) * e).sum(-1, keepdims=True) / s + depth                 # relative steps of s
        log_s = np.abs(np.log(s))
        loss = w * (t * ((d + off_s + 4 * log_s + 4) + depth * (d + log_s))).sum(-1) * U32
        T = t.sum(-1, keepdims=True)
        grad = (w * (1 if dloss is None else np.abs(dloss)))[:, None] * U32 * (T * e / s * (d + off_s + 2 * depth + 16) + 8 * t)
    return loss, grad


def clip(tensors, max_norm):
    """-> (norm, scale)"""
    norm = math.sqrt(math.fsum(float(v) ** 2 for t in tensors for v in np.asarray(t, np.float64).ravel()))
    return norm, (max_norm / norm if norm > max_norm else 1.0)
