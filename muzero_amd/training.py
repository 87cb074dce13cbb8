"""Operators of a training step on the targets of replay.py: the categorical loss with its gradient (csrc/mz_loss.hip), the
global gradient norm and clipping by it (csrc/mz_clip.hip).  The reference leaves them to Keras (training.py:13-51,157-204);
the names follow its framework."""
import ctypes
import struct
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from ._launch import DTYPES, launch, require_hip, require_tensor
from .exceptions import MuZeroError


# ---- categorical loss ----------------------------------------------------------------------------------------------------
def _loss(fn, *tensors):
    try:
        return fn(*tensors)
    except TypeError:
        raise MuZeroError('logits, targets, game, position and weights are tensors (the last three may be None)') from None


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
    return _loss(_lib.native().categorical_loss, logits, targets, game, position, weights)


def categorical_loss_and_grad(logits: torch.Tensor, targets: torch.Tensor, game: Optional[torch.Tensor] = None,
                              position: Optional[torch.Tensor] = None,
                              weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (categorical_loss(...), the gradient of its sum with respect to logits, of their shape and type), in one launch
    and outside autograd: for a step whose factors are all in `weights` (importance of the samples, scale of the unrolled
    steps), which passes the gradient on with logits.backward(grad)."""
    return _loss(_lib.native().categorical_loss_and_grad, logits, targets, game, position, weights)


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
