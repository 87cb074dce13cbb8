"""Layers of networks composed outside the built-in kernels, next to network.py's state-action encoders: group norm with
an activation over channels-last states (csrc/mz_norm.hip), forward and backward."""
import ctypes
import math
from typing import Optional

import torch

from . import _lib
from ._launch import DTYPES, launch, refuse_capture_of_live_leaves, remember_leaves, require_hip, require_tensor
from .exceptions import MuZeroError

ACTIVATIONS = {None: _lib.MZ_ACT_NONE, 'relu': _lib.MZ_ACT_RELU, 'silu': _lib.MZ_ACT_SILU, 'gelu': _lib.MZ_ACT_GELU,
               'tanh': _lib.MZ_ACT_TANH}


def _states(t):
    """-> (t or a dense copy of it, batch stride, position stride): the kernels walk a state as [batch][positions][C] with
    adjacent channels and one stride each for batch and positions."""
    shape, stride = t.shape, t.stride()
    if t.is_contiguous():
        c = shape[-1]
        return t, t.numel() // max(shape[0], 1), c
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
    return t.contiguous(), math.prod(shape[1:]), shape[-1]


def _describe(x, groups, param_dtype, activation, eps, residual, dy=None):
    cfg = _lib.GroupNorm()
    cfg.batch, cfg.channels, cfg.groups = x.shape[0], x.shape[-1], groups
    cfg.positions = math.prod(x.shape[1:-1])
    cfg.dtype, cfg.param_dtype, cfg.activation, cfg.eps = DTYPES[x.dtype], DTYPES[param_dtype], activation, eps
    x, cfg.x_strides[0], cfg.x_strides[1] = _states(x)
    if residual is not None:
        residual, cfg.residual_strides[0], cfg.residual_strides[1] = _states(residual)
    if dy is not None:
        dy, cfg.dy_strides[0], cfg.dy_strides[1] = _states(dy)
    return cfg, x, residual, dy


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(lib, cfg, backward, device):
    n = lib.mz_group_norm_workspace(ctypes.byref(cfg), backward)
    if n < 0:
        _lib.check(n)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None, n


def _forward(x, groups, weight, bias, eps, activation, residual, statistics):
    lib = _lib.load()
    cfg, xs, rs, _ = _describe(x, groups, _param_dtype(x, weight, bias), activation, eps, residual)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if statistics:
        mean, rstd = torch.empty(2, x.shape[0], groups, dtype=torch.float32, device=x.device)
    ws, n = _workspace(lib, cfg, 0, x.device)
    launch(x.device, lib.mz_group_norm_forward, ctypes.byref(cfg), xs.data_ptr(), _ptr(rs), _ptr(weight), _ptr(bias),
           y.data_ptr(), _ptr(mean), _ptr(rstd), _ptr(ws), n)
    return y, mean, rstd


def _param_dtype(x, weight, bias):
    return weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, groups, eps, activation):
        y, mean, rstd = _forward(x, groups, weight, bias, eps, activation, residual, True)
        # the residual enters the gradients through the activation's argument alone
        ctx.save_for_backward(x, weight, bias, residual if activation else None, mean, rstd)
        ctx.rest = groups, eps, activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, residual, mean, rstd = ctx.saved_tensors
        groups, eps, activation = ctx.rest
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        lib = _lib.load()
        cfg, xs, rs, dys = _describe(x, groups, _param_dtype(x, weight, bias), activation, eps, residual, dy)
        new = lambda like: torch.empty(like.shape, dtype=like.dtype, device=like.device)
        dx = new(x) if need_x else None
        dres = new(x) if need_r else None
        dw = new(weight) if need_w else None
        db = new(bias) if need_b else None
        ws, n = _workspace(lib, cfg, 1, x.device)
        launch(x.device, lib.mz_group_norm_backward, ctypes.byref(cfg), xs.data_ptr(), _ptr(rs), _ptr(weight), _ptr(bias),
               mean.data_ptr(), rstd.data_ptr(), dys.data_ptr(), _ptr(dx), _ptr(dres), _ptr(dw), _ptr(db), _ptr(ws), n)
        return dx, dw, db, dres, None, None, None


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
    tensors = (x, weight, bias, residual)
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors):
        return _forward(x, num_groups, weight, bias, eps, act, residual, False)[0]
    refuse_capture_of_live_leaves(device, tensors)
    return remember_leaves(device, _GroupNorm.apply(x, weight, bias, residual, num_groups, eps, act))
