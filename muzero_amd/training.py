"""Operators of a training step on the targets of replay.py: the categorical loss with its gradient (csrc/mz_loss.hip), the
global gradient norm and clipping by it (csrc/mz_clip.hip).  The reference leaves them to Keras (training.py:13-51,157-204);
the names follow its framework."""
import ctypes
import math
import struct
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from ._launch import DTYPES, launch, once, refuse_capture_of_live_leaves, remember_leaves, require_hip, require_tensor
from .exceptions import MuZeroError

MAX_CLASSES = 4096


# ---- categorical loss ----------------------------------------------------------------------------------------------------
# mz_categorical_t up to its dloss_strides, and those
_CONFIG, _DLOSS = struct.Struct('=qqqqiiiiqqqq'), struct.Struct('=qq')


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """A tensor of the rows' shape -> (t or a dense copy of it, unroll stride, batch stride)."""
    if t.dim() == 2:
        return (t, *t.stride())
    return t.contiguous(), 0, 1


def _describe(logits, targets, game, position, weights):
    """Checks the arguments of a loss -> the tensors as the kernel reads them (logits, targets, game, position, weights) and
    the configuration without dloss_strides."""
    require_tensor('logits', logits, DTYPES)
    device, shape = logits.device, logits.shape
    if len(shape) < 2 or not 1 <= shape[-1] <= MAX_CLASSES:
        raise MuZeroError(f'logits must be [..., classes] with 1 to {MAX_CLASSES} classes, got {tuple(shape)}')
    require_tensor('targets', targets, (torch.float32,), device)
    if targets.requires_grad:
        raise MuZeroError('the loss is not differentiable with respect to targets')
    rows, classes = shape[:-1], shape[-1]
    index_bytes = 4
    if game is not None or position is not None:
        if len(shape) != 3:
            raise MuZeroError(f'with game and position, logits must be [unroll, batch, classes], got {tuple(shape)}')
        if game is None or position is None:
            raise MuZeroError('game and position: both or neither')
        if targets.dim() != 3 or targets.shape[-1] != classes:
            raise MuZeroError(f'targets must be [positions, games, {classes}], got {tuple(targets.shape)}')
        for name, t in (('game', game), ('position', position)):
            require_tensor(name, t, (torch.int32, torch.int64), device)
            if t.shape != rows[1:]:
                raise MuZeroError(f'{name} must have shape ({rows[1]},), got {tuple(t.shape)}')
        if game.dtype != position.dtype:
            raise MuZeroError(f'game is {game.dtype}, position {position.dtype}: both must be of one type')
        index_bytes = 4 if game.dtype == torch.int32 else 8
        game, position = game.contiguous(), position.contiguous()
        positions, games = targets.shape[:2]
    elif targets.shape != shape:
        raise MuZeroError(f'targets have shape {tuple(targets.shape)}, logits {tuple(shape)}')
    else:
        positions, games = rows if len(rows) == 2 else (1, math.prod(rows))
    wu = wb = 0
    if weights is not None:
        require_tensor('weights', weights, (torch.float32,), device)
        if weights.requires_grad:
            raise MuZeroError('the loss is not differentiable with respect to weights')
        if weights.shape != rows:
            try:
                weights = weights.expand(rows)
            except RuntimeError:
                raise MuZeroError(f'weights of shape {tuple(weights.shape)} do not broadcast to {tuple(rows)}') from None
        weights, wu, wb = _rows(weights)
    require_hip(device)
    if len(rows) == 2:
        if logits.stride(-1) != 1 and classes > 1:
            logits = logits.contiguous()
        (unroll, batch), (zu, zb, _) = rows, logits.stride()
    else:
        logits = logits.contiguous()
        unroll, batch, zu, zb = 1, math.prod(rows), 0, classes
    config = _CONFIG.pack(unroll, batch, positions, games, classes, DTYPES[logits.dtype], index_bytes, 0, zu, zb, wu, wb)
    return (logits, targets.contiguous(), game, position, weights), config


def _run(tensors, config, with_loss, with_grad, dloss=None):
    logits, targets, game, position, weights = tensors
    shape, device = logits.shape, logits.device
    gu = gb = 0
    if dloss is not None:
        dloss, gu, gb = _rows(dloss)
    loss = torch.empty(shape[:-1], dtype=torch.float32, device=device) if with_loss else None
    grad = torch.empty(shape, dtype=logits.dtype, device=device) if with_grad else None
    launch(device, _lib.load().mz_categorical_loss, config + _DLOSS.pack(gu, gb), logits.data_ptr(), targets.data_ptr(), _ptr(game),
           _ptr(position), _ptr(weights), _ptr(dloss), _ptr(loss), _ptr(grad))
    return loss, grad


class _CategoricalLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tensors, config):
        ctx.save_for_backward(*tensors)
        ctx.config = config
        return _run(tensors, config, True, False)[0]

    @staticmethod
    @once
    def backward(ctx, dloss):
        return _run(ctx.saved_tensors, ctx.config, False, True, dloss)[1], None, None


def categorical_loss(logits: torch.Tensor, targets: torch.Tensor, game: Optional[torch.Tensor] = None,
                     position: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cross entropy of the rows of `logits` [..., classes] (float32, float16, bfloat16; 1 to 4096 classes) against target
    distributions (float32): weights * sum over classes of -target * log_softmax(logits), float32 of shape [...].

    Without `game` and `position`, targets has the shape of logits.  With them, targets is a block [positions, games,
    classes] as replay.compute_targets returns it (policies, or values of a support), logits is [unroll, batch, classes], and
    row (u, b) meets targets[position[b] + u, game[b]]: no gathered copy.  An index outside the block gives NaN (the host
    does not look at them).  weights broadcast over the rows; rows of weight 0 are not read and give 0 whatever they hold.  A
    class with target 0 adds nothing, also where its logit is -inf (an illegal move); a row whose logits are all -inf gives 0.
    A row of zero targets (past the end of a game) gives 0.  Differentiable once with respect to logits alone."""
    tensors, config = _describe(logits, targets, game, position, weights)
    if not torch.is_grad_enabled() or not logits.requires_grad:
        return _run(tensors, config, True, False)[0]
    refuse_capture_of_live_leaves(logits.device, (logits,))
    return remember_leaves(logits.device, _CategoricalLoss.apply(logits, tensors, config))


def categorical_loss_and_grad(logits: torch.Tensor, targets: torch.Tensor, game: Optional[torch.Tensor] = None,
                              position: Optional[torch.Tensor] = None,
                              weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (categorical_loss(...), the gradient of its sum with respect to logits, of their shape and type), in one launch
    and outside autograd: for a step whose factors are all in `weights` (importance of the samples, scale of the unrolled
    steps), which passes the gradient on with logits.backward(grad)."""
    tensors, config = _describe(logits, targets, game, position, weights)
    return _run(tensors, config, True, True)


# ---- global norm and clipping --------------------------------------------------------------------------------------------
def _dense(t):
    """Every element of t's memory span once: contiguous in some order of its dimensions."""
    if t.is_contiguous():
        return True
    span = 1
    for st, size in sorted((st, size) for st, size in zip(t.stride(), t.shape) if size != 1):
        if st != span:
            return False
        span *= size
    return True


def _like(t, o):
    return isinstance(o, torch.Tensor) and o.dtype == t.dtype and o.device == t.device and o.shape == t.shape and \
        (o.is_contiguous() and t.is_contiguous() or o.stride() == t.stride())


def _describe_tensors(tensors, out):
    """Checks -> (device, mz_tensor_t array, output pointers or None)."""
    n = len(tensors)
    if not 1 <= n <= _lib.MZ_GLOBAL_NORM_MAX_TENSORS:
        raise MuZeroError(f'1 to {_lib.MZ_GLOBAL_NORM_MAX_TENSORS} tensors, got {n}')
    device = require_tensor('tensor 0', tensors[0], DTYPES).device
    table = bytearray()
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor) or t.dtype not in DTYPES or t.device != device:
            require_tensor(f'tensor {i}', t, DTYPES, device)
        if not _dense(t):
            raise MuZeroError(f'tensor {i} is not dense: shape {tuple(t.shape)}, strides {t.stride()}')
        table += _TENSOR.pack(t.data_ptr(), t.numel(), DTYPES[t.dtype])
    outputs = None
    if out is not None:
        if len(out) != n:
            raise MuZeroError(f'{n} tensors, {len(out)} outputs')
        for i, (t, o) in enumerate(zip(tensors, out)):
            if not _like(t, o):
                raise MuZeroError(f'output {i} must be like its tensor: {t.dtype} {tuple(t.shape)}, strides {t.stride()}, on {t.device}')
        outputs = struct.pack(f'={n}Q', *[o.data_ptr() for o in out])
    require_hip(device)
    return device, bytes(table), outputs


_TENSOR = struct.Struct('=Qqi4x')          # mz_tensor_t


def _call(device, fn, *args):
    """fn(stream, *args, workspace, its size, norm) -> norm"""
    workspace = torch.empty(_lib.MZ_GLOBAL_NORM_WORKSPACE, dtype=torch.uint8, device=device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    launch(device, fn, *args, workspace.data_ptr(), _lib.MZ_GLOBAL_NORM_WORKSPACE, norm.data_ptr())
    return norm


def _check_clip(max_norm, written):
    if not max_norm >= 0:
        raise MuZeroError(f'max_norm must be >= 0, got {max_norm}')
    for t in written:
        if t.requires_grad:
            raise MuZeroError('a tensor that requires grad cannot be written by clipping')


class GradientSet:
    """The gradients of a network whose buffers stay where they are from step to step (zeroed in place, or written by a
    captured graph): their table is checked once and kept on the device, and `global_norm()` and
    `clip_by_global_norm(max_norm)` cost two launches each, whatever the number of tensors.

    tensors: 1 to 8192 float32, float16 and bfloat16 tensors of one device, each dense in some order of its dimensions.
    out: the tensors that clipping writes, of the same shapes, strides and types; None = the tensors themselves.  The set
    keeps the tensors alive, and has to be kept as long as a graph with calls of it is replayed; it is made outside
    captures.  Results are ordered on the current stream; a set may be used on several streams at once."""

    def __init__(self, tensors: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]] = None) -> None:
        self.tensors: List[torch.Tensor] = list(tensors)
        self.out = None if out is None else list(out)
        self.device, described, outputs = _describe_tensors(self.tensors, self.out)
        if torch.cuda.is_current_stream_capturing():
            raise MuZeroError('a GradientSet uploads its table: make it before the capture')
        self._lib = _lib.load()
        n = len(self.tensors)
        host = bytearray(n * _lib.MZ_TENSOR_TABLE_ENTRY)
        self._table = _lib.TensorTable()
        _lib.check(self._lib.mz_tensor_table_build(n, described, outputs, (ctypes.c_char * len(host)).from_buffer(host),
                                                   ctypes.byref(self._table)))
        self._overlap = None if self._table.writable else self._lib.mz_last_error().decode('utf-8', 'replace')
        self._memory = torch.frombuffer(host, dtype=torch.uint8).to(self.device)
        self._stream = torch.cuda.current_stream(self.device)

    def _run(self, fn, *args):
        stream = torch.cuda.current_stream(self.device)
        if stream != self._stream and not torch.cuda.is_current_stream_capturing():
            self._memory.record_stream(stream)
        return _call(self.device, fn, ctypes.byref(self._table), self._memory.data_ptr(), *args)

    def global_norm(self) -> torch.Tensor:
        """sqrt of the sum of the squares of all elements of all tensors: a float32 scalar on the device."""
        return self._run(self._lib.mz_tensor_table_global_norm)

    def clip_by_global_norm(self, max_norm: float) -> torch.Tensor:
        """Writes every tensor times max_norm / global norm to its output where the norm is above max_norm, else unchanged,
        and returns the norm before clipping.  Where that is NaN every output is NaN; where it is infinite, finite elements
        become 0 and infinite ones NaN."""
        written = self.tensors if self.out is None else self.out
        _check_clip(max_norm, written)
        if self._overlap:
            raise MuZeroError(f'cannot clip: {self._overlap}')
        norm = self._run(self._lib.mz_tensor_table_clip, max_norm)
        torch.autograd.graph.increment_version(written)
        return norm


def global_norm(tensors: Sequence[torch.Tensor]) -> torch.Tensor:
    """GradientSet(tensors).global_norm() for tensors that are others in every step: their table travels with the launch, 112
    tensors each, and nothing is uploaded."""
    tensors = list(tensors)
    device, described, _ = _describe_tensors(tensors, None)
    return _call(device, _lib.load().mz_global_norm, len(tensors), described)


def clip_by_global_norm(tensors: Sequence[torch.Tensor], max_norm: float, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """GradientSet(tensors, out).clip_by_global_norm(max_norm) in the same way: in place, or into `out`; returns the norm
    before clipping.  Tensors that are written may not share memory with others of the list."""
    tensors, out = list(tensors), None if out is None else list(out)
    device, described, outputs = _describe_tensors(tensors, out)
    written = tensors if out is None else out
    _check_clip(max_norm, written)
    norm = _call(device, _lib.load().mz_clip_by_global_norm, len(tensors), described, outputs, max_norm)
    torch.autograd.graph.increment_version(written)
    return norm
