"""oracle/train_oracle.py against central differences and against torch's autograd in 64 bits (CPU), and the refusals of
the training operators that need no GPU: argument checks of the Python entries, and of the C entries before any launch."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import train_oracle as to

NORM_CASES = [(2, 5, 6, 3, 'relu', True), (2, 1, 8, 8, None, False), (3, 4, 12, 1, 'silu', False), (2, 9, 4, 2, 'gelu', True),
              (2, 3, 6, 2, 'tanh', True)]


@pytest.mark.parametrize('N,S,C,G,activation,residual', NORM_CASES)
def test_group_norm_oracle_against_differences_and_autograd(N, S, C, G, activation, residual):
    rng = np.random.default_rng(N * 100 + C)
    x, dy, res = rng.standard_normal((3, N, S, C))
    w, b = 1 + 0.3 * rng.standard_normal(C), 0.3 * rng.standard_normal(C)
    res = res if residual else None
    o = to.GroupNormOracle(x, G, w, b, 1e-5, activation, res)
    got, _ = o.backward(dy)
    f = lambda **k: (to.GroupNormOracle(**{**dict(x=x, groups=G, weight=w, bias=b, eps=1e-5, activation=activation, residual=res), **k}).y * dy).sum()
    step = 1e-6
    for name, key, base in (('dx', 'x', x), ('dweight', 'weight', w), ('dbias', 'bias', b), ('dresidual', 'residual', res)):
        if base is None:
            continue
        for at in rng.integers(0, base.size, 6):
            e = np.zeros(base.size)
            e[at] = step
            e = e.reshape(base.shape)
            diff = (f(**{key: base + e}) - f(**{key: base - e})) / (2 * step)
            assert abs(diff - got[name].ravel()[at]) < 1e-6 * max(1, np.abs(dy).sum() / 10)
    t = lambda a: torch.tensor(a, dtype=torch.float64, requires_grad=True)
    X, W, B = t(x), t(w), t(b)
    y = torch.nn.functional.group_norm(X.permute(0, 2, 1), G, W, B, 1e-5).permute(0, 2, 1)
    y = y + (torch.tensor(res) if residual else 0)
    y = {'relu': torch.relu, 'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu, 'tanh': torch.tanh, None: lambda v: v}[activation](y)
    np.testing.assert_allclose(o.y, y.detach().numpy(), rtol=1e-10, atol=1e-12)
    for a, g in zip(torch.autograd.grad(y, [X, W, B], torch.tensor(dy)), (got['dx'], got['dweight'], got['dbias'])):
        np.testing.assert_allclose(g, a.numpy(), rtol=1e-7, atol=1e-9)


def test_categorical_oracle_against_differences():
    rng = np.random.default_rng(5)
    z, t, w = 3 * rng.standard_normal((4, 7)), rng.random((4, 7)), rng.random(4)
    t[1] = 0
    z[2, 3], t[2, 3] = -np.inf, 0
    loss, grad = to.categorical(z, t, w)
    step = 1e-6
    for i in range(4):
        for c in range(7):
            if not np.isfinite(z[i, c]):
                assert grad[i, c] == 0
                continue
            e = np.zeros_like(z)
            e[i, c] = step
            diff = (to.categorical(z + e, t, w)[0] - to.categorical(z - e, t, w)[0]).sum() / (2 * step)
            assert abs(diff - grad[i, c]) < 1e-7
    assert loss[1] == 0 and (grad[1] == 0).all()


# ---- refusals ------------------------------------------------------------------------------------------------------------
def test_group_norm_refuses():
    from muzero_amd.exceptions import MuZeroError
    from muzero_amd.layers import group_norm
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    for kw in (dict(num_groups=3), dict(num_groups=0), dict(num_groups=2, activation='elu'), dict(num_groups=2, eps=-1.0),
               dict(num_groups=2, eps=math.inf), dict(num_groups=2, weight=torch.ones(7)), dict(num_groups=2, weight=w.double()),
               dict(num_groups=2, weight=w, bias=torch.ones(1)), dict(num_groups=2, residual=torch.zeros(2, 3, 4)),
               dict(num_groups=2, residual=torch.zeros(2, 3, 8, dtype=torch.float16)), dict(num_groups=2, weight=[1.0] * 8)):
        with pytest.raises(MuZeroError):
            group_norm(x, **kw)
    for bad in (torch.zeros(8), torch.zeros(2, 3, 8, dtype=torch.float64), torch.zeros(2, 8, dtype=torch.int32), None, torch.zeros(2, 3, 0)):
        with pytest.raises(MuZeroError):
            group_norm(bad, 2)
    with pytest.raises(MuZeroError, match='one type'):
        group_norm(x.half(), 2, w, w.half())
    with pytest.raises(MuZeroError, match='HIP device'):
        group_norm(x, 2, w, w)


def test_categorical_loss_refuses():
    from muzero_amd.exceptions import MuZeroError
    from muzero_amd.training import categorical_loss, categorical_loss_and_grad
    z, block, i = torch.zeros(3, 4, 5), torch.zeros(9, 6, 5), torch.zeros(4, dtype=torch.int32)
    bad = [dict(targets=block), dict(targets=block, game=i), dict(targets=block, game=i, position=i.long()),
           dict(targets=block, game=i, position=i[:3]), dict(targets=block[..., :4], game=i, position=i),
           dict(targets=block.double(), game=i, position=i), dict(targets=block, game=i.float(), position=i),
           dict(targets=torch.zeros(3, 4, 5), weights=torch.ones(3)), dict(targets=torch.zeros(3, 4, 5), weights=torch.ones(4).half()),
           dict(targets=torch.zeros(3, 4, 5, requires_grad=True)), dict(targets=torch.zeros(3, 4, 5), weights=torch.ones(4, requires_grad=True)),
           dict(targets=None)]
    for fn in (categorical_loss, categorical_loss_and_grad):
        for kw in bad:
            with pytest.raises(MuZeroError):
                fn(z, **kw)
        with pytest.raises(MuZeroError):
            fn(torch.zeros(5), torch.zeros(5))
        with pytest.raises(MuZeroError):
            fn(torch.zeros(2, 4097), torch.zeros(2, 4097))
        with pytest.raises(MuZeroError):
            fn(torch.zeros(2, 0), torch.zeros(2, 0))
        with pytest.raises(MuZeroError):
            fn([0.0], torch.zeros(1))
        with pytest.raises(MuZeroError, match='unroll'):
            fn(torch.zeros(4, 5), block, game=i, position=i)
        with pytest.raises(MuZeroError, match='HIP device'):
            fn(z, block, game=i, position=i, weights=torch.ones(4))


def test_gradient_set_refuses():
    from muzero_amd.exceptions import MuZeroError
    from muzero_amd.training import GradientSet, clip_by_global_norm, global_norm
    a, b = torch.zeros(3, 4), torch.zeros(5)
    for tensors, out in (([], None), (None, None), (a.numel(), None), ([a], 3), ([a], [1.0]), ([a.double()], None),
                         ([a, 1.0], None), ([a[:, :2]], None), ([a, b], [a]), ([a], [b]), ([a], [a.half()]), ([torch.zeros(4).expand(3, 4)], None), ([a], [torch.zeros(4, 3).t()])):
        with pytest.raises(MuZeroError):
            GradientSet(tensors, out)
    with pytest.raises(MuZeroError):
        global_norm([torch.zeros(1)] * 8193)
    with pytest.raises(MuZeroError, match='HIP device'):
        clip_by_global_norm([a, b], 1.0)


def _lib():
    from muzero_amd import _lib
    return _lib, _lib.load()


def test_c_entries_refuse_before_any_launch():
    L, lib = _lib()
    INVALID, fake = -1, 0x10000
    norm = L.GroupNorm(batch=2, positions=3, channels=8, groups=2, dtype=0, param_dtype=0, activation=1, eps=1e-5)
    assert lib.mz_group_norm_workspace(ctypes.byref(norm), 0) >= 0
    assert lib.mz_group_norm_workspace(None, 0) == INVALID
    for field, value in (('groups', 3), ('groups', 0), ('batch', -1), ('positions', -1), ('channels', 0), ('dtype', 3), ('dtype', -1),
                         ('param_dtype', 2), ('activation', 5), ('eps', float('nan')), ('eps', -1.0), ('positions', 1 << 47)):
        other = L.GroupNorm.from_buffer_copy(norm)
        setattr(other, field, value)
        assert lib.mz_group_norm_workspace(ctypes.byref(other), 1) == INVALID, field
        assert lib.mz_group_norm_forward(None, ctypes.byref(other), fake, None, None, None, fake, None, None, fake, 1 << 30) == INVALID
    assert lib.mz_group_norm_forward(None, ctypes.byref(norm), None, None, None, None, fake, None, None, fake, 1 << 20) == INVALID
    assert lib.mz_group_norm_forward(None, ctypes.byref(norm), fake, None, None, None, fake, fake, None, fake, 1 << 20) == INVALID
    need = lib.mz_group_norm_workspace(ctypes.byref(norm), 1)
    if need:
        assert lib.mz_group_norm_backward(None, ctypes.byref(norm), fake, None, None, None, fake, fake, fake, fake, None, fake, fake,
                                          fake, need - 1) == INVALID
    loss = L.Categorical(unroll=2, batch=3, target_positions=2, target_games=3, classes=5, dtype=0, index_bytes=4)
    for field, value in (('classes', 0), ('classes', 4097), ('unroll', -1), ('dtype', 7), ('index_bytes', 2), ('batch', 1 << 48)):
        other = L.Categorical.from_buffer_copy(loss)
        setattr(other, field, value)
        assert lib.mz_categorical_loss(None, ctypes.byref(other), fake, fake, fake, fake, None, None, fake, fake) == INVALID, field
    assert lib.mz_categorical_loss(None, ctypes.byref(loss), None, fake, None, None, None, None, fake, None) == INVALID
    assert lib.mz_categorical_loss(None, ctypes.byref(loss), fake, None, None, None, None, None, fake, None) == INVALID


def test_clip_refuses_overlap_before_any_launch():
    L, lib = _lib()
    ws = L.MZ_GLOBAL_NORM_WORKSPACE

    def clip(tensors, outputs=None, max_norm=1.0, workspace_bytes=ws):
        table = (L.Tensor * len(tensors))(*[L.Tensor(data=p, elements=n, dtype=k) for p, n, k in tensors])
        out = None if outputs is None else (ctypes.c_void_p * len(outputs))(*outputs)
        return lib.mz_clip_by_global_norm(None, len(tensors), table, out, max_norm, 0x100, workspace_bytes, 0x100)

    A, B = 0x100000, 0x200000
    refused = [dict(tensors=[(A, 16, 0), (A, 16, 0)]),                          # the same tensor twice, in place
               dict(tensors=[(A, 16, 0), (A + 60, 16, 0)]), dict(tensors=[(A + 2, 16, 2), (A, 2, 2)]),
               dict(tensors=[(A, 16, 0), (B, 16, 0)], outputs=[B, A]),          # swapped
               dict(tensors=[(A, 16, 0)], outputs=[A + 4]),                     # shifted
               dict(tensors=[(A, 16, 0), (B, 1, 0)], outputs=[B + 64, A + 60]),
               dict(tensors=[(A, 4, 0)], outputs=[None]), dict(tensors=[(A + 2, 4, 0)]), dict(tensors=[(A, 4, 0)], outputs=[B + 2]),
               dict(tensors=[(None, 4, 0)]), dict(tensors=[(A, -1, 0)]), dict(tensors=[(A, 4, 5)]), dict(tensors=[(A, 4, 0)], max_norm=-1.0),
               dict(tensors=[(A, 4, 0)], max_norm=float('nan')), dict(tensors=[(A, 4, 0)], workspace_bytes=ws - 1), dict(tensors=[]),
               dict(tensors=[(A, 1 << 42, 0), (A + (1 << 44), 1 << 42, 0), (A + (1 << 45), 1, 0)])]
    for kw in refused:
        assert clip(**kw) == -1, kw


def test_tensor_tables_are_checked_where_they_are_built():
    L, lib = _lib()
    A = 0x100000
    build = lambda table, n, host, out: lib.mz_tensor_table_build(n, (L.Tensor * len(table))(*table), None, host, ctypes.byref(out) if out else None)
    two = [L.Tensor(data=A, elements=5000, dtype=0), L.Tensor(data=A + (1 << 20), elements=0, dtype=1), L.Tensor(data=A + (1 << 20), elements=1, dtype=2)]
    host, info = (ctypes.c_char * (3 * L.MZ_TENSOR_TABLE_ENTRY))(), L.TensorTable()
    assert build(two, 3, host, info) == 0
    assert (info.entries, info.writable) == (2, 1) and info.chunks == -(-5000 // info.chunk) + 1       # empty tensors are left out
    assert build(two, 3, None, info) == -1 and build(two, 0, host, info) == -1
    assert build([L.Tensor(data=None, elements=1, dtype=0)], 1, host, info) == -1
    assert build([two[0], two[0]], 2, host, info) == 0 and info.writable == 0
    args = (0x100, L.MZ_GLOBAL_NORM_WORKSPACE, 0x100)
    assert lib.mz_tensor_table_clip(None, ctypes.byref(info), 0x100, 1.0, *args) == -1                  # overlapping tensors
    assert build(two, 3, host, info) == 0
    assert lib.mz_tensor_table_clip(None, ctypes.byref(info), 0x100, -1.0, *args) == -1
    assert lib.mz_tensor_table_clip(None, ctypes.byref(info), None, 1.0, *args) == -1
    assert lib.mz_tensor_table_clip(None, ctypes.byref(L.TensorTable(entries=-1)), 0x100, 1.0, *args) == -1
    assert lib.mz_tensor_table_global_norm(None, None, 0x100, *args) == -1
    assert lib.mz_tensor_table_global_norm(None, ctypes.byref(info), 0x100, 0x100, L.MZ_GLOBAL_NORM_WORKSPACE - 1, 0x100) == -1
    assert lib.mz_tensor_table_global_norm(None, ctypes.byref(info), 0x100, 0x100, L.MZ_GLOBAL_NORM_WORKSPACE, None) == -1


def test_c_entries_refuse_arrays_that_are_not_aligned_to_their_type():
    L, lib = _lib()
    A, ws = 0x100000, L.MZ_GLOBAL_NORM_WORKSPACE
    norm = L.GroupNorm(batch=2, positions=3, channels=8, groups=2, dtype=2, param_dtype=0, activation=1, eps=1e-5)
    good = [A, A, A, A, A, A, A, A]                                    # x, residual, weight, bias, y, mean, rstd, workspace
    for i, off in ((0, 1), (1, 1), (2, 2), (3, 2), (4, 1), (5, 2), (6, 2), (7, 2)):
        args = list(good)
        args[i] += off
        assert lib.mz_group_norm_forward(None, ctypes.byref(norm), *args, 1 << 20) == -1, i
    for i, off in enumerate((1, 1, 2, 2, 2, 2, 1, 1, 1, 2, 2, 2)):     # x, residual, weight, bias, mean, rstd, dy, dx, dres, dw, db, ws
        args = [A] * 12
        args[i] += off
        assert lib.mz_group_norm_backward(None, ctypes.byref(norm), *args, 1 << 20) == -1, i
    loss = L.Categorical(unroll=2, batch=3, target_positions=2, target_games=3, classes=5, dtype=1, index_bytes=8)
    for i, off in enumerate((1, 2, 4, 4, 2, 2, 2, 1)):                 # logits, targets, game, position, weights, dloss, loss, dlogits
        args = [A] * 8
        args[i] += off
        assert lib.mz_categorical_loss(None, ctypes.byref(loss), *args) == -1, i
    table = (L.Tensor * 1)(L.Tensor(data=A, elements=4, dtype=0))
    assert lib.mz_global_norm(None, 1, table, 0x1004, ws, A) == -1 and lib.mz_global_norm(None, 1, table, 0x1000, ws, A + 2) == -1
