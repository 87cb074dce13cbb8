"""Calls of the training operators that would return results without what belongs to them (a derivative, a recorded operation, a
sign) or read other memory than they were given: refused, before anything is launched and whatever the device."""
import pytest
import torch
from torch.autograd import forward_ad

from muzero_amd.exceptions import MuZeroError


def calls(wrap=lambda t: t):
    """name -> a call of each operator, one of its tensors wrapped."""
    from muzero_amd.layers import group_norm
    from muzero_amd.training import GradientSet, categorical_loss, categorical_loss_and_grad, clip_by_global_norm, global_norm
    x, w, z, t = torch.zeros(2, 3, 8), torch.ones(8), torch.zeros(4, 5), torch.ones(4, 5)
    return {'x': lambda: group_norm(wrap(x), 2), 'weight': lambda: group_norm(x, 2, wrap(w)), 'bias': lambda: group_norm(x, 2, w, wrap(w)),
            'residual': lambda: group_norm(x, 2, residual=wrap(x)), 'logits': lambda: categorical_loss(wrap(z), t),
            'targets': lambda: categorical_loss(z, wrap(t)), 'weights': lambda: categorical_loss(z, t, weights=wrap(torch.ones(4))),
            'both': lambda: categorical_loss_and_grad(wrap(z), t), 'norm': lambda: global_norm([x, wrap(w)]),
            'clip': lambda: clip_by_global_norm([wrap(x), w], 1.0), 'out': lambda: clip_by_global_norm([x], 1.0, [wrap(x.clone())]),
            'set': lambda: GradientSet([x, wrap(w)])}


@pytest.mark.parametrize('name', calls())
def test_forward_mode_derivatives(name):
    with forward_ad.dual_level():
        with pytest.raises(MuZeroError, match='forward-mode'):
            calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))[name]()


@pytest.mark.parametrize('name', calls())
def test_tensors_without_memory_of_their_own(name):
    for transform in (lambda f: torch.func.vmap(f)(torch.zeros(3)), lambda f: torch.func.grad(f)(torch.tensor(0.0)),
                      lambda f: torch.func.jvp(f, (torch.tensor(0.0),), (torch.tensor(1.0),))):
        with pytest.raises(MuZeroError, match='torch.func'):
            transform(lambda s: calls(lambda t: t + s)[name]())
    with pytest.raises(MuZeroError, match='strided'):
        calls(lambda t: t.to_sparse())[name]()


@pytest.mark.gpu
def test_forward_mode_derivatives_on_the_device():
    from muzero_amd.layers import group_norm
    from muzero_amd.training import categorical_loss
    x, z = torch.randn(2, 3, 8, device='cuda', requires_grad=True), torch.randn(4, 5, device='cuda', requires_grad=True)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t.detach(), torch.ones_like(t))
        for call in (lambda: group_norm(dual(x), 2), lambda: categorical_loss(dual(z), torch.ones_like(z))):
            with pytest.raises(MuZeroError, match='forward-mode'):
                call()
        for y, leaf in ((group_norm(x, 2), x), (categorical_loss(z, torch.ones(4, 5, device='cuda')), z)):
            with pytest.raises(RuntimeError, match='forward-mode'):        # a tangent of the gradient
                torch.autograd.grad(y, leaf, dual(y))
        assert torch.isfinite(group_norm(forward_ad.unpack_dual(dual(x)).primal, 2)).all()


def recordings(call):
    """The call under everything that records torch's operations."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    s = torch.zeros(())
    yield lambda: torch.jit.trace(call, (s,), check_trace=False)
    yield lambda: make_fx(call)(s)
    yield lambda: make_fx(call, tracing_mode='fake')(s)

    def fake():
        with FakeTensorMode(allow_non_fake_inputs=True):
            call(s)
    yield fake


@pytest.mark.parametrize('name', calls())
def test_recorded_calls(name):
    for record in recordings(lambda s: calls()[name]()):
        with pytest.raises(MuZeroError, match='cannot be recorded'):
            record()


@pytest.mark.gpu
def test_recorded_calls_on_the_device():
    from torch.fx.experimental.proxy_tensor import make_fx
    from muzero_amd.layers import group_norm
    from muzero_amd.training import GradientSet, categorical_loss, clip_by_global_norm
    x, z = torch.randn(2, 3, 8, device='cuda'), torch.randn(4, 5, device='cuda')
    t, kept = torch.ones_like(z), GradientSet([x.clone()])
    for call in (lambda x, z: group_norm(x, 2), lambda x, z: categorical_loss(z, t), lambda x, z: clip_by_global_norm([x], 1.0),
                 lambda x, z: kept.global_norm(), lambda x, z: kept.clip_by_global_norm(1.0)):
        for record in (lambda: torch.jit.trace(call, (x, z), check_trace=False), lambda: make_fx(call)(x, z)):
            with pytest.raises(MuZeroError, match='cannot be recorded'):
                record()
        assert torch.isfinite(call(x.clone(), z)).all()                    # and not refused any longer


@pytest.mark.parametrize('channels', [2 ** 24 + 1, 2 ** 32 + 8, 2 ** 40])
def test_more_channels_than_the_kernels_count(channels):
    from muzero_amd.layers import group_norm
    for groups in (1, channels // 8 if channels % 8 == 0 else channels):
        with pytest.raises(MuZeroError, match='at most 16777216 channels'):
            group_norm(torch.zeros(1, 1, 1).expand(2, 3, channels), groups)


def negatives(t):
    """Tensors of t's values whose memory holds them negated: as a view of nothing else, and as a conjugate's imaginary part."""
    return [torch._neg_view(-t)] + ([torch.complex(t, -t).conj().imag] if t.dtype == torch.float32 else [])


def test_lazy_negatives_in_lists():
    from muzero_amd.training import GradientSet, clip_by_global_norm, global_norm
    a = torch.ones(5)
    for n in negatives(a):
        assert n.is_neg() and torch.equal(n, a)
        for call in (lambda: GradientSet([a, n]), lambda: global_norm([n]), lambda: clip_by_global_norm([n], 1.0)):
            with pytest.raises(MuZeroError, match='negative'):
                call()
    with pytest.raises(MuZeroError, match='negative'):
        clip_by_global_norm([a], 1.0, [torch._neg_view(a.clone())])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
def test_lazy_negatives_are_read_with_their_sign(dtype):
    from muzero_amd.layers import group_norm
    from muzero_amd.training import categorical_loss, categorical_loss_and_grad
    gen = torch.Generator(device='cuda').manual_seed(2)
    noise = lambda *s: torch.randn(*s, generator=gen, device='cuda')
    x, res, dy, w, b = noise(3, 4, 8).to(dtype), noise(3, 4, 8).to(dtype), noise(3, 4, 8).to(dtype), noise(8).to(dtype), noise(8).to(dtype)
    z, t, weights, up = noise(2, 3, 5).to(dtype), noise(2, 3, 5).abs(), noise(2, 3).abs(), noise(2, 3)

    def run(x, w, b, res, dy, z, t, weights, up):
        leaves = [v.detach().requires_grad_() for v in (x, w, b, res, z)]
        y = group_norm(leaves[0], 2, leaves[1], leaves[2], activation='silu', residual=leaves[3])
        loss = categorical_loss(leaves[4], t, weights=weights)
        return [y, loss, *torch.autograd.grad(y, leaves[:4], dy), *torch.autograd.grad(loss, leaves[4], up), group_norm(x, 2, w, b, residual=res),
                *categorical_loss_and_grad(z, t, weights=weights)]

    args = [x, w, b, res, dy, z, t, weights, up]
    want = run(*args)
    for i, arg in enumerate(args):
        for n in negatives(arg):
            assert n.is_neg()
            assert all(torch.equal(p, q) for p, q in zip(run(*args[:i], n, *args[i + 1:]), want)), i


class Wrapper(torch.Tensor):
    """A tensor that stands for another one: of its shape and type, with no memory."""
    @staticmethod
    def __new__(cls, inner):
        self = torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)
        self.inner = inner
        return self

    @classmethod
    def __torch_dispatch__(cls, fn, types, args=(), kwargs=None):
        return fn(*(a.inner if isinstance(a, cls) else a for a in args), **(kwargs or {}))


@pytest.mark.parametrize('name', calls())
def test_tensors_that_wrap_others(name):
    with pytest.raises(MuZeroError, match='memory of its own'):
        calls(Wrapper)[name]()


def test_zeros_without_memory_in_lists():
    from muzero_amd.training import GradientSet, clip_by_global_norm
    a, zeros = torch.ones(5), torch._efficientzerotensor(5)
    for call in (lambda: GradientSet([a, zeros]), lambda: clip_by_global_norm([a], 1.0, [zeros])):
        with pytest.raises(MuZeroError, match='zeros without any'):
            call()


@pytest.mark.gpu
def test_wrappers_and_zeros_without_memory_on_the_device():
    from muzero_amd.layers import group_norm
    from muzero_amd.training import categorical_loss
    x, w = torch.randn(2, 3, 8, device='cuda', requires_grad=True), torch.full((8,), 2.0, device='cuda')
    z, t = torch.randn(4, 5, device='cuda', requires_grad=True), torch.ones(4, 5, device='cuda')
    weights, index = torch.ones(4, device='cuda'), torch.zeros(4, dtype=torch.int64, device='cuda')
    for call in (lambda: group_norm(x, 2, Wrapper(w)), lambda: group_norm(x, 2, w, Wrapper(w)), lambda: group_norm(x, 2, residual=Wrapper(x.detach())),
                 lambda: categorical_loss(z, t, weights=Wrapper(weights)), lambda: categorical_loss(z[None], t[None], Wrapper(index), index),
                 lambda: categorical_loss(z[None], t[None], index, Wrapper(index))):
        with pytest.raises(MuZeroError, match='memory of its own'):
            call()
    none = lambda like: torch._efficientzerotensor(like.shape, device='cuda')
    y, loss = group_norm(x, 2, none(w), none(w), residual=none(x)), categorical_loss(z, none(t), weights=weights)
    assert (y == 0).all() and (loss == 0).all() and (categorical_loss(z, t, weights=none(weights)) == 0).all()
    assert (torch.autograd.grad(group_norm(x, 2), x, none(x))[0] == 0).all()
    assert (torch.autograd.grad(categorical_loss(z, t), z, none(loss))[0] == 0).all()
