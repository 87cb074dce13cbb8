"""Cases, plain forms and 64-bit values of the operators a training step of a composed network consists of besides its
products: group norm with an activation over channels-last states, the categorical loss against the replay targets with
its gradient, and the global gradient norm with clipping.

`run` computes them with elementary torch operations in 32 bits, or with muzero_amd's operators where `own` is true.
"""
import math
import random

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
ITEM = {'f32': 4, 'f16': 2, 'bf16': 2}

# tensors of the CartPole network in weight order (kernel, bias per layer)
CARTPOLE_SIZES = [51712, 128, 16384, 128, 32768, 128, 16384, 128, 16384, 128, 128, 1, 16384, 128, 16384, 128, 12928, 101,
                  256, 2]

MOST_NORM = 512 * 361 * 256          # elements of the largest listed case of each operator
MOST_LOSS = 6 * 16384 * 601
MOST_CLIP = 250_000_123


def _norm(name, batch, positions, channels, groups, dtype, activation, residual, train, extra=0):
    return dict(name=name, op='group_norm', batch=batch, positions=positions, channels=channels, groups=groups, dtype=dtype,
                activation=activation, residual=residual, train=train, extra=extra)


def _loss(name, unroll, batch, classes, dtype, indexed, masked, autograd, games=0, moves=0):
    return dict(name=name, op='loss', unroll=unroll, batch=batch, classes=classes, dtype=dtype, indexed=indexed,
                masked=masked, autograd=autograd, games=games, moves=moves)


def _clip(name, net, tensors, elements, split, dtype, clip, kept):
    return dict(name=name, op='clip', net=net, tensors=tensors, elements=elements, split=split, dtype=dtype, clip=clip,
                kept=kept)


def listed():
    return [
        # one game's 3x3x128 state in a search of a single tree: nothing but latency
        _norm('norm one board', 1, 9, 128, 32, 'f32', 'relu', False, False),
        # the two-position states of a lockstep search over 16384 games: inference at full width
        _norm('norm 16384 states', 16384, 2, 128, 16, 'f32', 'relu', True, False),
        # residual block of a 3x3 board network in training, one batch of 4096 positions
        _norm('norm 3x3 train', 4096, 9, 128, 32, 'bf16', 'relu', True, True),
        # residual block of a 19x19 board network in training
        _norm('norm 19x19 train', 512, 361, 256, 16, 'bf16', 'relu', True, True),
        # first block over 96x96 frames in training: samples far larger than a workgroup's registers
        _norm('norm 96x96 train', 24, 9216, 64, 8, 'f16', 'silu', False, True),
        # a state with one-hot action planes behind it (128 + 18 channels), normalised in pairs: odd widths
        _norm('norm 146 channels', 777, 25, 146, 73, 'f32', 'gelu', False, True),
        # the value support of 101 bins, three unrolled steps of a small batch, straight from the replay targets
        _loss('loss 101 bins', 3, 128, 101, 'f32', True, False, False, 64, 160),
        # the policy over a 19x19 board with its pass move: illegal moves masked, loss.backward() as a trainer calls it
        _loss('loss 362 moves', 6, 2048, 362, 'bf16', True, True, True, 1024, 60),
        # reanalysed batch with a 601-bin value support
        _loss('loss 601 bins', 6, 16384, 601, 'f16', True, False, False, 512, 64),
        # the gradients of the CartPole network, clipped into the flat buffer that its weights are handed over in
        _clip('clip cartpole', True, 20, sum(CARTPOLE_SIZES), 0, 'f32', True, False),
        # a network of many tensors of all sizes, in two types
        _clip('clip 161 tensors', False, 161, 23_456_789, 5, 'mixed', True, True),
        # gradients far larger than the caches
        _clip('clip 250M', False, 7, MOST_CLIP, 3, 'f32', True, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['group_norm', 'group_norm', 'loss', 'loss', 'clip'])
    if op == 'group_norm':
        groups = rng.choice([1, 2, 4, 8, 16, 32, rng.randrange(1, 40)])
        channels = groups * max(1, _log(rng, 1, 512) // groups)
        # from eight values a group: of two, nothing is left of a gradient once mean and scale are taken out
        positions = max(_log(rng, 1, 9216), -(-8 * groups // channels))
        batch = min(_log(rng, 1, 16384), max(1, MOST_NORM // (positions * channels)))
        train = rng.random() < 0.6
        return dict(op=op, batch=batch, positions=positions, channels=channels, groups=groups,
                    dtype=rng.choice(['f32', 'f16', 'bf16', 'bf16']), activation=rng.choice(['none', 'relu', 'silu', 'gelu', 'tanh']),
                    residual=rng.random() < 0.5, train=train, extra=rng.choice([0, 0, 0, 2, 18]))
    if op == 'loss':
        unroll, classes = rng.randrange(1, 7), _log(rng, 2, 4096)
        batch = min(_log(rng, 1, 16384), max(1, MOST_LOSS // (unroll * classes)))
        games, moves = _log(rng, 1, 512), _log(rng, 1, 60)
        games = min(games, max(1, MOST_LOSS // ((moves + unroll) * classes)))
        return dict(op=op, unroll=unroll, batch=batch, classes=classes, dtype=rng.choice(['f32', 'f16', 'bf16']),
                    indexed=rng.random() < 0.6, masked=rng.random() < 0.5, autograd=rng.random() < 0.4, games=games, moves=moves)
    elements = _log(rng, 1000, MOST_CLIP)
    return dict(op=op, net=False, tensors=_log(rng, 1, 300), elements=elements, split=rng.randrange(1 << 20),
                dtype=rng.choice(['f32', 'bf16', 'mixed']), clip=rng.random() < 0.6, kept=rng.random() < 0.5)


# ---- group norm ------------------------------------------------------------------------------------------------------

EPS = 1e-5


def _prepare_norm(case, gen):
    N, S, C, dtype = case['batch'], case['positions'], case['channels'], DTYPES[case['dtype']]
    noise = lambda *shape: torch.randn(*shape, generator=gen, device='cuda')
    # a convolution's outputs: every channel with an offset and a scale of its own
    x = noise(N, S, C + case['extra']) * (1 + 0.5 * noise(C + case['extra']).abs()) + noise(C + case['extra'])
    state = dict(case, x=x.to(dtype)[..., :C], weight=1 + 0.2 * noise(C), bias=0.2 * noise(C),
                 res=noise(N, S, C).to(dtype) if case['residual'] else None)
    del x
    if case['train']:
        dy = noise(N, S, C).to(dtype)
        if case['activation'] == 'relu':         # no gradient where the argument is at the kink: it has none there
            dy[_affine(state, torch.float64)[0].abs() < 1e-4] = 0
        state['dy'] = dy
        state['leaves'] = [t.detach().requires_grad_() for t in (state['x'], state['weight'], state['bias'])]
        if case['residual']:
            state['leaves'].append(state['res'].detach().requires_grad_())
    return state


def _affine(s, at):
    N, S, C, G = s['batch'], s['positions'], s['channels'], s['groups']
    x = s['x'].to(at).reshape(N, S, G, C // G)
    d = x - x.sum((1, 3), keepdim=True) / (S * (C // G))
    rstd = torch.rsqrt((d * d).sum((1, 3), keepdim=True) / (S * (C // G)) + EPS)
    xhat = (d * rstd).reshape(N, S, C)
    z = xhat * s['weight'].to(at) + s['bias'].to(at)
    if s['res'] is not None:
        z = z + s['res'].to(at)
    return z, xhat, rstd


def _act(z, activation):
    if activation == 'relu':
        return torch.where(z > 0, z, torch.zeros_like(z))
    if activation == 'silu':
        return z / (1 + torch.exp(-z))
    if activation == 'gelu':
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return torch.tanh(z) if activation == 'tanh' else z


def _act_slope(z, activation):
    if activation == 'relu':
        return (z > 0).to(z.dtype)
    if activation == 'silu':
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 + z * (1 - sig))
    if activation == 'gelu':
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return 1 - torch.tanh(z) ** 2 if activation == 'tanh' else torch.ones_like(z)


def _run_norm(s):
    activation = None if s['activation'] == 'none' else s['activation']
    if own:
        from muzero_amd.layers import group_norm
        if not s['train']:
            return group_norm(s['x'], s['groups'], s['weight'], s['bias'], eps=EPS, activation=activation, residual=s['res'])
        leaves = s['leaves']
        y = group_norm(leaves[0], s['groups'], leaves[1], leaves[2], eps=EPS, activation=activation,
                       residual=leaves[3] if s['residual'] else None)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, s['dy']))
    N, S, C, G, dtype = s['batch'], s['positions'], s['channels'], s['groups'], s['x'].dtype
    z, xhat, rstd = _affine(s, torch.float32)
    y = _act(z, activation).to(dtype)
    if not s['train']:
        return y
    dz = s['dy'].float() * _act_slope(z, activation)
    dbias, dweight = dz.sum((0, 1)), (dz * xhat).sum((0, 1))
    g = (dz * s['weight']).reshape(N, S, G, C // G)
    h = xhat.reshape(N, S, G, C // G)
    n = S * (C // G)
    dx = rstd * (g - g.sum((1, 3), keepdim=True) / n - h * ((g * h).sum((1, 3), keepdim=True) / n))
    return [y, dx.reshape(N, S, C).to(dtype), dweight, dbias] + ([dz.to(dtype)] if s['residual'] else [])


def _exact_norm(s):
    N, S, C, G = s['batch'], s['positions'], s['channels'], s['groups']
    x, w, b = (t.double().requires_grad_(s['train']) for t in (s['x'], s['weight'], s['bias']))
    res = s['res'].double().requires_grad_(s['train']) if s['res'] is not None else None
    grouped = x.reshape(N, S, G, C // G).transpose(1, 2).reshape(N, G, -1)
    var, mean = torch.var_mean(grouped, dim=2, correction=0, keepdim=True)
    z = ((grouped - mean) / torch.sqrt(var + EPS)).reshape(N, G, S, C // G).transpose(1, 2).reshape(N, S, C)
    z = z * w + b + (res if res is not None else 0)
    y = {'none': lambda t: t, 'relu': lambda t: t.clamp(min=0), 'silu': lambda t: t * torch.sigmoid(t),
         'gelu': lambda t: t * 0.5 * torch.erfc(-t / math.sqrt(2)), 'tanh': torch.tanh}[s['activation']](z)
    if not s['train']:
        return y
    return [y.detach()] + list(torch.autograd.grad(y, [x, w, b] + ([res] if res is not None else []), s['dy'].double()))


def _work_norm(c):
    n, passes = c['batch'] * c['positions'] * c['channels'], 1 + (1 if c['residual'] else 0) + 1
    if c['train']:        # the forward's inputs are the backward's too: once; its outputs and gradients once each
        passes += 1 + 1 + (1 if c['residual'] else 0)
    return {'bytes': n * ITEM[c['dtype']] * passes + 8 * c['channels'] * (2 if c['train'] else 1), 'flops': n * (30 if c['train'] else 10)}


# ---- categorical loss ------------------------------------------------------------------------------------------------

def _prepare_loss(case, gen):
    U, B, C = case['unroll'], case['batch'], case['classes']
    noise = lambda *shape: torch.randn(*shape, generator=gen, device='cuda')
    uniform = lambda *shape: torch.rand(*shape, generator=gen, device='cuda')
    logits = 2 * noise(U, B, C)
    rows = (case['moves'] + U, case['games']) if case['indexed'] else (U, B)
    legal = (uniform(C) < 0.7) if case['masked'] else None
    if legal is not None:
        legal[0] = True
    # visit distributions or two-hot supports; a tenth of the rows lie past the end of their game and are zero
    if case['masked'] or C < 64:
        targets = torch.exp(2 * noise(*rows, C))
        if legal is not None:
            targets = targets * legal
            logits = torch.where(legal, logits, torch.full_like(logits, -math.inf))
        targets /= targets.sum(-1, keepdim=True)
    else:
        at = uniform(*rows, 1) * (C - 1)
        low = at.floor()
        targets = torch.zeros(*rows, C, device='cuda')
        targets.scatter_(-1, low.long(), 1 - (at - low))
        targets.scatter_add_(-1, (low.long() + 1).clamp(max=C - 1), at - low)
    targets *= (uniform(*rows, 1) < 0.9)
    # importance weights of the samples, the unrolled steps sharing their gradient
    weights = (0.2 + uniform(B)) * torch.tensor([1.0] + [1.0 / max(1, U - 1)] * (U - 1), device='cuda')[:, None]
    state = dict(case, logits=logits.to(DTYPES[case['dtype']]), targets=targets, weights=weights, game=None, position=None)
    if case['indexed']:
        state['game'] = torch.randint(0, case['games'], (B,), generator=gen, device='cuda', dtype=torch.int32)
        state['position'] = torch.randint(0, case['moves'] + 1, (B,), generator=gen, device='cuda', dtype=torch.int32)
    state['leaf'] = state['logits'].detach().requires_grad_()
    return state


def _target_rows(s):
    if s['game'] is None:
        return s['targets']
    steps = torch.arange(s['unroll'], device='cuda')[:, None]
    return s['targets'][s['position'].long() + steps, s['game'].long()]


def _run_loss(s):
    if own:
        from muzero_amd.training import categorical_loss, categorical_loss_and_grad
        if not s['autograd']:
            return list(categorical_loss_and_grad(s['logits'], s['targets'], game=s['game'], position=s['position'],
                                                  weights=s['weights']))
        loss = categorical_loss(s['leaf'], s['targets'], game=s['game'], position=s['position'], weights=s['weights'])
        return [loss.detach()] + list(torch.autograd.grad(loss.sum(), s['leaf']))
    z, t = s['logits'].float(), _target_rows(s)
    top = z.max(-1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    loss = torch.where(t != 0, t * (top - z + torch.log(total)), torch.zeros_like(t)).sum(-1)
    grad = t.sum(-1, keepdim=True) * (e / total) - t
    return [s['weights'] * loss, (s['weights'][..., None] * grad).to(s['logits'].dtype)]


def _exact_loss(s):
    z, t, w = s['logits'].double(), _target_rows(s).double(), s['weights'].double()
    log_p = z - torch.logsumexp(z, -1, keepdim=True)
    loss = -w * (t * log_p.masked_fill(t == 0, 0.0)).sum(-1)
    return [loss, w[..., None] * (t.sum(-1, keepdim=True) * torch.exp(log_p) - t)]


def _work_loss(c):
    rows = c['unroll'] * c['batch']
    block = min(rows, (c['moves'] + c['unroll']) * c['games']) if c['indexed'] else rows
    n = c['classes']
    return {'bytes': 2 * rows * n * ITEM[c['dtype']] + block * n * 4 + rows * 8 + (8 * c['batch'] if c['indexed'] else 0),
            'flops': 12 * rows * n}


# ---- global norm and clipping ----------------------------------------------------------------------------------------

def _sizes(case):
    if case['net']:
        return CARTPOLE_SIZES
    rng = random.Random(case['split'])
    share = [math.exp(rng.uniform(0, 9)) for _ in range(case['tensors'])]
    return [max(1, int(case['elements'] * s / sum(share))) for s in share]


def _kinds(case):
    n = len(_sizes(case))
    return [('bf16' if i % 3 else 'f32') if case['dtype'] == 'mixed' else case['dtype'] for i in range(n)]


def _prepare_clip(case, gen):
    sizes, kinds = _sizes(case), _kinds(case)
    # gradients of layers differ by orders of magnitude
    grads = [(torch.randn(n, generator=gen, device='cuda').mul_(10.0 ** (-(i % 5)))).to(DTYPES[k])
             for i, (n, k) in enumerate(zip(sizes, kinds))]
    state = dict(case, grads=grads, limit=0.5, flat={}, out=None, kept_set=None)
    if case['clip']:      # one flat buffer per type, tensor behind tensor
        state['flat'] = {k: torch.zeros(sum(n for n, j in zip(sizes, kinds) if j == k), dtype=DTYPES[k], device='cuda')
                         for k in sorted(set(kinds))}
        at = dict.fromkeys(state['flat'], 0)
        state['out'] = []
        for n, k in zip(sizes, kinds):
            state['out'].append(state['flat'][k][at[k]:at[k] + n])
            at[k] += n
    if own:
        if case['kept']:          # a trainer whose gradient buffers live as long as it does keeps their table
            from muzero_amd.training import GradientSet
            state['kept_set'] = GradientSet(grads, out=state['out'])
    return state


def _run_clip(s):
    if own:
        from muzero_amd.training import clip_by_global_norm, global_norm
        if s['kept_set'] is not None:
            norm = s['kept_set'].clip_by_global_norm(s['limit']) if s['clip'] else s['kept_set'].global_norm()
        else:
            norm = clip_by_global_norm(s['grads'], s['limit'], out=s['out']) if s['clip'] else global_norm(s['grads'])
        return {'norm': norm, **s['flat']}
    norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s['grads']]).sum().sqrt()
    if s['clip']:
        scale = torch.where(norm > s['limit'], s['limit'] / norm, torch.ones_like(norm)).float()
        [o.copy_(g.float() * scale) for g, o in zip(s['grads'], s['out'])]
    return {'norm': norm.float(), **s['flat']}


def _exact_clip(s):
    norm = math.sqrt(math.fsum(float(torch.dot(g.double(), g.double())) for g in s['grads']))
    flat = {k: torch.cat([g for g in s['grads'] if g.dtype == DTYPES[k]]).double().mul_(min(1.0, s['limit'] / norm) if norm else 1.0)
            for k in s['flat']}
    return {'norm': torch.tensor(norm, dtype=torch.float64), **flat}


def _work_clip(c):
    total = sum(n * ITEM[k] for n, k in zip(_sizes(c), _kinds(c)))
    return {'bytes': total * (2 if c['clip'] else 1) + 4, 'flops': sum(_sizes(c)) * (3 if c['clip'] else 2)}


# ---- what is called --------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return {'group_norm': _prepare_norm, 'loss': _prepare_loss, 'clip': _prepare_clip}[case['op']](case, gen)


def run(state):
    return {'group_norm': _run_norm, 'loss': _run_loss, 'clip': _run_clip}[state['op']](state)


def exact(case, seed):
    return {'group_norm': _exact_norm, 'loss': _exact_loss, 'clip': _exact_clip}[case['op']](prepare(case, seed))


def work(case):
    return {'group_norm': _work_norm, 'loss': _work_loss, 'clip': _work_clip}[case['op']](case)
