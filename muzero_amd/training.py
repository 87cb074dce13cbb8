"""Operators of a training step on the targets of replay.py: the categorical loss with its gradient (csrc/mz_loss.hip), the
global gradient norm and clipping by it (csrc/mz_clip.hip).  The reference leaves them to Keras (training.py:13-51,157-204);
the names follow its framework.

A forward pass that is being captured into a graph is refused where its backward pass would reach an autograd node of a stream
outside the capture (an eager graph of the same leaves that is still alive).  Forward-mode derivatives, transforms of torch.func
and recordings of torch's operations (torch.jit.trace, torch.fx, torch.export, fake tensors) are refused."""
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
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
    does not look at them).  weights broadcast over the rows; rows of weight 0 give 0 whatever they hold.  A
    class with target 0 adds nothing, also where its logit is -inf (an illegal move); a row whose logits are all -inf gives 0.
    A row of zero targets (past the end of a game) gives 0, unless its logits are NaN or +inf.  Differentiable once, in reverse
    mode, with respect to logits alone."""
    return _loss(_lib.native().categorical_loss, logits, targets, game, position, weights)


def categorical_loss_and_grad(logits: torch.Tensor, targets: torch.Tensor, game: Optional[torch.Tensor] = None,
                              position: Optional[torch.Tensor] = None,
                              weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (categorical_loss(...), the gradient of its sum with respect to logits, of their shape and type), in one launch
    and outside autograd: for a step whose factors are all in `weights` (importance of the samples, scale of the unrolled
    steps), which passes the gradient on with logits.backward(grad)."""
    return _loss(_lib.native().categorical_loss_and_grad, logits, targets, game, position, weights)


# ---- global norm and clipping --------------------------------------------------------------------------------------------
def _list(fn, tensors, *args):
    try:
        return fn(list(tensors), *args)
    except TypeError:
        raise MuZeroError('tensors and out are lists of tensors (out may be None), max_norm is a number') from None


class GradientSet:
    """The gradients of a network whose buffers stay where they are from step to step (zeroed in place, or written by a
    captured graph): their table is checked once and kept on the device, and `global_norm()` and
    `clip_by_global_norm(max_norm)` cost two launches each, whatever the number of tensors.  With torch's optimisers that is
    optimizer.zero_grad(set_to_none=False): by default every backward pass makes new .grad tensors, of which the set knows
    nothing; clip_by_global_norm() below takes those.

    tensors: 1 to 8192 float32, float16 and bfloat16 tensors of one device, each dense in some order of its dimensions.
    out: the tensors that clipping writes, of the same shapes, strides and types; None = the tensors themselves.  The set
    keeps the tensors alive, and has to be kept as long as a graph with calls of it is replayed; it is made outside
    captures.  A tensor that was given other memory or another shape since is refused.  Results are ordered on the current stream; a set may be
    used on several streams at once."""

    def __init__(self, tensors: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]] = None) -> None:
        self._set = _list(_lib.native().GradientSet, tensors, out)

    def global_norm(self) -> torch.Tensor:
        """sqrt of the sum of the squares of all elements of all tensors: a float32 scalar on the device."""
        return self._set.global_norm()

    def clip_by_global_norm(self, max_norm: float) -> torch.Tensor:
        """Writes every tensor times max_norm / global norm to its output where the norm is above max_norm, else unchanged,
        and returns the norm before clipping.  Where that is NaN every output is NaN; where an element is infinite, finite ones
        become 0 and infinite ones NaN.  (A norm of finite elements above float32's range is returned as infinite, and clipped by
        all the same.)"""
        try:
            return self._set.clip_by_global_norm(max_norm)
        except TypeError:
            raise MuZeroError(f'max_norm must be a number, got {max_norm!r}') from None


def global_norm(tensors: Sequence[torch.Tensor]) -> torch.Tensor:
    """GradientSet(tensors).global_norm() for tensors that are others in every step: their table travels with the launch, 112
    tensors each, and nothing is uploaded.  Outside autograd: the norm has no gradient."""
    return _list(_lib.native().global_norm, tensors)


def clip_by_global_norm(tensors: Sequence[torch.Tensor], max_norm: float, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """GradientSet(tensors, out).clip_by_global_norm(max_norm) in the same way: in place, or into `out`; returns the norm
    before clipping.  Tensors that are written may not share memory with others of the list."""
    return _list(_lib.native().clip_by_global_norm, tensors, max_norm, out)
