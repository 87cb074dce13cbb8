"""muzero_amd.layers.group_norm where lanes of one workgroup belong to several samples, and where they may not: the oracle's
values, and a sample's results beside other samples."""
import pytest
import torch

from test_group_norm_gpu import BF16, F16, F32, check, make, oracle, rows, run_and_check

pytestmark = pytest.mark.gpu

# batch, positions, channels, groups, type, activation, residual, parameters: groups of 65 to 128 vectors, at one position for any
# batch and at two to four for large ones, are where a workgroup of four wavefronts holds two samples
SIDE_BY_SIDE = [
    (2, (), 257, 1, F32, 'relu', True, 'f32'), (5, (), 300, 1, F32, None, False, 'f32'), (5, (), 512, 1, F32, 'silu', True, 'f32'),
    (4, (), 768, 2, F32, 'gelu', False, 'f32'), (7, (1,), 1024, 2, F32, 'tanh', True, 'f32'), (3, (), 1536, 3, F32, None, True, None),
    (2, (), 513, 1, F16, 'silu', True, 'same'), (5, (), 768, 1, F16, 'relu', False, 'f32'), (6, (1, 1), 1024, 1, BF16, 'gelu', True, 'f32'),
    (5, (), 2048, 2, BF16, None, True, 'same'), (1, (), 512, 1, F32, 'silu', True, 'f32'),
    (4099, (), 512, 1, F32, 'silu', True, 'f32'), (4099, (), 600, 1, BF16, 'relu', True, 'f32'), (4099, (), 768, 2, F32, None, False, 'f32'),
    (4099, (2,), 512, 1, F32, 'relu', True, 'f32'), (4099, (3,), 384, 1, F32, 'gelu', False, 'f32'), (4099, (4,), 512, 1, F32, 'tanh', True, 'f32'),
    (4099, (2,), 1024, 1, F16, 'silu', False, 'same'), (4099, (3,), 1026, 2, BF16, 'relu', True, 'f32'),
]


def name_of(case):
    return '-'.join(str(v).replace('torch.', '').replace(' ', '') for v in case)


@pytest.mark.parametrize('case', SIDE_BY_SIDE, ids=name_of)
def test_samples_side_by_side_against_the_oracle(case):
    run_and_check(*make(case, 11))


def results(x, G, w, b, activation, res, dy):
    from muzero_amd.layers import group_norm
    leaves = [t.detach().requires_grad_() for t in (x, res)]
    y = group_norm(leaves[0], G, w, b, activation=activation, residual=leaves[1])
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


# every layout: one wavefront and more, samples side by side in a wavefront and across, wide units, positions split
LAYOUTS = [
    (33, (3, 3), 128, 32, BF16), (5, (), 512, 1, F32), (4099, (3,), 384, 1, F32), (64, (2,), 32, 8, F32), (2500, (9,), 16, 4, BF16),
    (6, (19, 19), 64, 4, F32), (5, (25,), 146, 73, F32), (3, (2500,), 16, 4, F16), (4, (), 4100, 1, BF16), (700, (2,), 10, 5, F16),
    (3, (101,), 520, 40, F32),
]


@pytest.mark.parametrize('case', LAYOUTS, ids=name_of)
def test_a_sample_does_not_see_the_others(case):
    x, G, w, b, activation, res, dy = make((*case, 'silu', True, 'f32'), 5)
    N = x.shape[0]
    whole = results(x, G, w, b, activation, res, dy)
    for i in {0, N // 2, N - 1}:
        # others in their place, in a batch of the same size: not a bit of it changes
        other = [torch.randn_like(t) * 50 for t in (x, res, dy)]
        for o, t in zip(other, (x, res, dy)):
            o[i] = t[i]
        for got, want in zip(results(other[0], G, w, b, activation, other[1], other[2]), whole):
            assert torch.equal(got[i], want[i]), i
        # on its own the order of the sums may be another: held to the oracle
        one = slice(i, i + 1)
        o = oracle(x[one], G, w, b, activation, res[one])
        want, off = o.backward(rows(dy[one]))
        for got in (results(x[one], G, w, b, activation, res[one], dy[one]), [t[one] for t in whole]):
            check('y', got[0], o.y, o.off_y, x.dtype)
            check('dx', got[1], want['dx'], off['dx'], x.dtype)
            check('dresidual', got[2], want['dresidual'], off['dresidual'], x.dtype)


def spread(t, batch_stride, position_stride=None):
    """t [N, S, C], its samples (and positions) that many elements apart."""
    N, S, C = t.shape
    position_stride = position_stride or C
    memory = torch.empty((N - 1) * batch_stride + (S - 1) * position_stride + C, dtype=t.dtype, device='cuda')
    return memory.as_strided(t.shape, (batch_stride, position_stride, 1)).copy_(t)


# small samples that lie farther apart than 32-bit offsets reach from the first of a workgroup to its last: a step of each game
# out of a large buffer, or positions on the far side of one
FAR = [
    ((3, (4,), 16, 4, F32, 'silu', True, 'f32'), 200_000_000, None), ((20, (1,), 16, 4, F32, 'tanh', True, 'f32'), 20_000_000, None),
    ((3, (9,), 16, 4, BF16, 'gelu', True, 'f32'), 600_000_000, None), ((7, (1,), 24, 24, F16, 'silu', True, 'same'), 100_000_001, None),
    ((2, (1,), 300, 1, F32, None, True, 'f32'), 300_000_000, None), ((3, (5,), 20, 10, BF16, 'silu', True, 'f32'), 600_000_000, None),
    ((70, (2,), 8, 2, F32, 'silu', True, 'f32'), 40_000_001, None),
    ((3, (3,), 64, 16, F16, 'gelu', True, 'f32'), 64, 400_000_000), ((2, (2,), 37, 37, BF16, 'tanh', True, 'same'), 37, 700_000_001),
]


@pytest.mark.parametrize('which', ['x', 'residual', 'dy', 'all'])
@pytest.mark.parametrize('case', FAR, ids=lambda c: name_of(c[0]) + f'-{c[1]}-{c[2]}')
def test_samples_and_positions_far_apart(case, which):
    shape, batch_stride, position_stride = case
    x, G, w, b, activation, res, dy = make(shape, 23)
    if which in ('x', 'all'):
        x = spread(x, batch_stride, position_stride)
    if which in ('residual', 'all'):
        res = spread(res, batch_stride, position_stride)
    if which in ('dy', 'all'):
        dy = spread(dy, batch_stride, position_stride)
    run_and_check(x, G, w, b, activation, res, dy)


# 2^25 sums of dweight and dbias: eight columns a workgroup of 1024 threads are 2^32 threads, more than one grid holds
@pytest.mark.parametrize('case', [(1, (), 2 ** 24, 2 ** 21, F16, None, False, 'f32'), (2, (), 2 ** 23 + 4, 1, F32, None, False, 'f32'),
                                  (1, (), 2 ** 24, 2 ** 24, BF16, None, True, 'same')], ids=name_of)
def test_as_many_channels_as_there_may_be(case):
    run_and_check(*make(case, 3))
