"""Layers of networks composed outside the built-in kernels, next to network.py's state-action encoders: group norm with
an activation over channels-last states (csrc/mz_norm.hip), forward and backward."""
import functools
import math
import struct
from typing import Optional

import torch

from . import _lib
from ._launch import DTYPES, launch, refuse_capture_of_live_leaves, once, remember_leaves, require_hip, require_tensor
from .exceptions import MuZeroError

ACTIVATIONS = {None: _lib.MZ_ACT_NONE, 'relu': _lib.MZ_ACT_RELU, 'silu': _lib.MZ_ACT_SILU, 'gelu': _lib.MZ_ACT_GELU,
               'tanh': _lib.MZ_ACT_TANH}


# mz_group_norm_t up to its dy_strides, and those
_CONFIG, _DY = struct.Struct('=qqiiiiiidqqqq'), struct.Struct('=qq')


def _states(t):
    """-> (t or a dense copy of it, batch stride, position stride): the kernels walk a state as [batch][positions][C] with
    adjacent channels and one stride each for batch and positions."""
    shape = t.shape
    if not t.is_contiguous():
        stride = t.stride()
        if stride[-1] == 1 or shape[-1] == 1:
            step, span, ok = 0, 1, True
            for size, st in zip(reversed(shape[1:-1]), reversed(stride[1:-1])):
                if size == 1:
                    continue
                if span == 1:
                    step = st
                ok &= st == step * span
                span *= size
            if ok:
                return t, stride[0], step
        t = t.contiguous()
    return t, math.prod(shape[1:]), shape[-1]


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(config, backward):
    n = _lib.load().mz_group_norm_workspace(config, backward)
    if n < 0:
        _lib.check(n)
    return n


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(x, groups, weight, bias, eps, activation, residual, statistics):
    """-> y, mean and rstd [2, B, groups] or None, x and residual as the kernels read them, the configuration."""
    shape, dtype, device = x.shape, x.dtype, x.device
    x, xb, xp = _states(x)
    rb = rp = 0
    if residual is not None:
        residual, rb, rp = _states(residual)
    param = weight if weight is not None else bias
    config = _CONFIG.pack(shape[0], math.prod(shape[1:-1]), shape[-1], groups, DTYPES[dtype],
                          _lib.MZ_F32 if param is None else DTYPES[param.dtype], activation, 0, eps, xb, xp, rb, rp)
    y = torch.empty(shape, dtype=dtype, device=device)
    stats = mean = rstd = None
    if statistics:
        stats = torch.empty(2, shape[0], groups, dtype=torch.float32, device=device)
        mean = stats.data_ptr()
        rstd = mean + 4 * shape[0] * groups
    whole = config + _DY.pack(0, 0)
    n = _workspace_bytes(whole, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    launch(device, _lib.load().mz_group_norm_forward, whole, x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(bias), y.data_ptr(),
           mean, rstd, _ptr(ws), n)
    return y, stats, x, residual, config


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, groups, eps, activation):
        y, stats, x, residual, config = _forward(x, groups, weight, bias, eps, activation, residual, True)
        # the residual enters the gradients through the activation's argument alone
        ctx.save_for_backward(x, weight, bias, residual if activation else None, stats)
        ctx.config = config
        return y

    @staticmethod
    @once
    def backward(ctx, dy):
        x, weight, bias, residual, stats = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy, db, dp = _states(dy)
        config = ctx.config + _DY.pack(db, dp)
        device = x.device
        dx = torch.empty(x.shape, dtype=x.dtype, device=device) if need_x else None
        dres = torch.empty(x.shape, dtype=x.dtype, device=device) if need_r else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=device) if need_w else None
        dbias = torch.empty(bias.shape, dtype=bias.dtype, device=device) if need_b else None
        n = _workspace_bytes(config, 1)
        ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
        mean = stats.data_ptr()
        launch(device, _lib.load().mz_group_norm_backward, config, x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(bias), mean,
               mean + stats.numel() * 2, dy.data_ptr(), _ptr(dx), _ptr(dres), _ptr(dw), _ptr(dbias), _ptr(ws), n)
        return dx, dw, dbias, dres, None, None, None


def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """activation(normalised(x) * weight + bias + residual) of channels-last states x [B, ..., C] (float32, float16,
    bfloat16): every sample's C channels are normalised in `num_groups` groups of adjacent ones, over all positions, to
    mean 0 and (population) variance 1.

    weight, bias: [C], float32 or of x's type (both alike), or None.  activation: None, 'relu', 'silu', 'gelu' (by erf) or
    'tanh'.  residual: of x's shape and type.  Returns a dense tensor of x's shape and type; statistics are float32.
    Differentiable once with respect to all four tensors.  A state with one stride for its positions (a slice of the
    channels of a wider one, an NCHW tensor in channels-last memory, permuted) is read in place, others are copied first."""
    require_tensor('x', x, DTYPES)
    if x.dim() < 2:
        raise MuZeroError(f'x must be [B, ..., C], got shape {tuple(x.shape)}')
    device, channels = x.device, x.shape[-1]
    if num_groups < 1 or channels < 1 or channels % num_groups:
        raise MuZeroError(f'{channels} channels cannot be split into {num_groups} groups')
    if activation not in ACTIVATIONS:
        raise MuZeroError(f'activation {activation!r} is not one of {tuple(ACTIVATIONS)}')
    if not 0 <= eps < math.inf:
        raise MuZeroError(f'eps must be finite and >= 0, got {eps}')
    for name, p in (('weight', weight), ('bias', bias)):
        if p is not None:
            require_tensor(name, p, (torch.float32, x.dtype), device)
            if p.shape != (channels,):
                raise MuZeroError(f'{name} must have shape ({channels},), got {tuple(p.shape)}')
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise MuZeroError(f'weight is {weight.dtype}, bias {bias.dtype}: both must be of one type')
    if residual is not None:
        require_tensor('residual', residual, (x.dtype,), device)
        if residual.shape != x.shape:
            raise MuZeroError(f'residual has shape {tuple(residual.shape)}, x {tuple(x.shape)}')
    require_hip(device)
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    act = ACTIVATIONS[activation]
    if not torch.is_grad_enabled() or not (x.requires_grad or weight is not None and weight.requires_grad
                                           or bias is not None and bias.requires_grad
                                           or residual is not None and residual.requires_grad):
        return _forward(x, num_groups, weight, bias, eps, act, residual, False)[0]
    refuse_capture_of_live_leaves(device, (x, weight, bias, residual))
    return remember_leaves(device, _GroupNorm.apply(x, weight, bias, residual, num_groups, eps, act))
