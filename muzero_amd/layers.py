"""Layers of networks composed outside the built-in kernels, next to network.py's state-action encoders: group norm with
an activation over channels-last states (csrc/mz_norm.hip), forward and backward.  Under capture, see training.py."""
from typing import Optional

import torch

from . import _lib
from .exceptions import MuZeroError


def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """activation(normalised(x) * weight + bias + residual) of channels-last states x [B, ..., C] (float32, float16,
    bfloat16; at most 2^24 channels): every sample's C channels are normalised in `num_groups` groups of adjacent ones, over
    all positions, to mean 0 and (population) variance 1.

    weight, bias: [C], float32 or of x's type (both alike), or None.  activation: None, 'relu', 'silu', 'gelu' (by erf) or
    'tanh'.  residual: of x's shape and type.  Returns a dense tensor of x's shape and type; statistics are float32.
    Activations are float32 too: gelu within 3e-7 |z| of the exact one, silu and tanh within (1.3 |z| + 8) and 12 times 2^-24 of
    themselves.  A sample's result does not depend on what the others hold; the order of its sums may on the size of the batch.
    Differentiable once with respect to all four tensors, in reverse mode.  A state with one stride for its positions (a slice
    of the channels of a wider one, an NCHW tensor in channels-last memory, permuted) is read in place, others are copied."""
    try:
        return _lib.native().group_norm(x, num_groups, weight, bias, eps, activation, residual)
    except TypeError:
        raise MuZeroError('group_norm takes tensors (x, weight, bias, residual), an int (num_groups), a float (eps) and a name '
                          '(activation)') from None
