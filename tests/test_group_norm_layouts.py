"""How group norm shares a state among lanes (mz_debug_group_norm_layout), without a GPU: what the kernels rely on, and that the
cases of test_group_norm_layouts_gpu.py are laid out as they mean to be."""
import ctypes
import math
import random
from collections import namedtuple

import torch

from test_group_norm_layouts_gpu import FAR, SIDE_BY_SIDE

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
Layout = namedtuple('Layout', 'threads vectors samples positions units unit_vectors pieces splits')


def layout(N, S, C, groups, dtype, x=None, residual=None, dy=None):
    """x, residual, dy: batch and position strides, None = dense."""
    from muzero_amd import _lib
    config = _lib.GroupNorm(batch=N, positions=S, channels=C, groups=groups, dtype=dtype, param_dtype=0, activation=0, eps=1e-5)
    for field, strides in (('x_strides', x), ('residual_strides', residual), ('dy_strides', dy)):
        getattr(config, field)[:] = strides or (S * C, C)
    out = (ctypes.c_int32 * 8)()
    assert _lib.load().mz_debug_group_norm_layout(ctypes.byref(config), out) == 0
    return Layout(*out)


def test_lanes_fill_a_workgroup_and_split_positions_are_of_one_sample():
    rng = random.Random(4)
    log = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))
    split = wide = several = 0
    for _ in range(20000):
        groups, D, dtype = log(1, 300), log(1, 9000), rng.randrange(3)
        C, S = groups * D, log(1, 5000)
        N = log(1, min(100000, (1 << 48) // (C * S)))
        far = {k: (log(1, 1 << 34), log(1, 1 << 34)) for k in ('x', 'residual', 'dy') if rng.random() < 0.2}
        l = layout(N, S, C, groups, dtype, **far)
        case = N, S, C, groups, dtype, far, l
        assert l.threads in (64, 256, 512), case
        if l.pieces == 1:
            assert l.samples * l.positions * l.units * l.unit_vectors == l.threads, case
        if l.vectors == 0:
            assert l.samples == 1 and l.splits >= 1, case
        else:
            assert l.pieces == 1 and l.splits == 1 and 1 <= l.vectors <= 8 and l.positions * l.vectors >= S, case
        split += l.vectors == 0 and S * C < 1000
        wide += l.pieces > 1
        several += l.threads > 64 and l.samples > 1
    assert split and wide and several


def test_strides_that_no_second_sample_uses_change_nothing():
    for dtype in range(3):
        assert layout(1, 9, 128, 32, dtype, (1 << 40, 128), (0, 128), (1 << 33, 128)) == layout(1, 9, 128, 32, dtype)


def test_the_cases_of_the_gpu_tests_are_laid_out_as_they_say():
    for N, shape, C, groups, dtype, *_ in SIDE_BY_SIDE:
        l = layout(N, math.prod(shape), C, groups, DTYPES[dtype])
        assert l.threads == 256 and l.samples == 2 and l.vectors, (N, shape, C)
    for (N, (S,), C, groups, dtype, *_), batch, position in FAR:
        near, far = layout(N, S, C, groups, DTYPES[dtype]), (batch, position or C)
        assert near.vectors and near.samples > 1, (N, S, C)
        for which in ('x', 'residual', 'dy'):
            assert layout(N, S, C, groups, DTYPES[dtype], **{which: far}).vectors == 0, (N, S, C, which)
