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
