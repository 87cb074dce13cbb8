"""What the training operators (layers.py, training.py) share: argument checks, launches, captures of autograd graphs."""
import torch

from . import _lib
from .exceptions import MuZeroError

DTYPES = {torch.float32: _lib.MZ_F32, torch.float16: _lib.MZ_F16, torch.bfloat16: _lib.MZ_BF16}

# the current stream's handle; the call behind torch.cuda.current_stream, which takes 25 times as long to wrap it
_current_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)

_ACCUMULATE = type(torch.autograd.graph.get_gradient_edge(torch.zeros((), requires_grad=True)).node)


def require_tensor(name, t, dtypes, device=None):
    """A tensor of one of `dtypes` (on `device` if given); returns it."""
    if not isinstance(t, torch.Tensor):
        raise MuZeroError(f'{name} must be a tensor, got {type(t).__name__}')
    if t.dtype not in dtypes:
        raise MuZeroError(f'{name}: expected one of {tuple(dtypes)}, got {t.dtype}')
    if device is not None and t.device != device:
        raise MuZeroError(f'{name} is on {t.device}, expected {device}')
    return t


def require_hip(device):
    if device.type != 'cuda':
        raise MuZeroError(f'the tensors must be on a HIP device, not {device}; muzero_amd has no CPU fallback')


def launch(device, fn, *args):
    """fn(stream, *args) of libmzhip.so on `device`'s current stream, with that device current."""
    index = device.index
    if index == torch.cuda.current_device():
        status = fn(_current_stream(index), *args)
    else:
        with torch.cuda.device(device):
            status = fn(_current_stream(index), *args)
    if status < 0:
        _lib.check(status)


def once(backward):
    """backward of an autograd.Function that is differentiable once: the usual pass runs with gradients off and goes straight
    through; under create_graph=True its results refuse to be differentiated again."""
    refusing = torch.autograd.function.once_differentiable(backward)
    return lambda ctx, *grads: (refusing if torch.is_grad_enabled() else backward)(ctx, *grads)


def refuse_capture_of_live_leaves(device, tensors):
    """A leaf's gradient is accumulated on the stream its accumulation node was made on, and the node lives as long as any
    autograd graph that holds it.  A backward pass captured while such a graph of another stream lives would leave the
    capture, which ends the process: refused here, before anything is captured."""
    if not torch.cuda.is_current_stream_capturing():
        return
    stream = _current_stream(device.index)
    for t in tensors:
        if t is not None and t.requires_grad and t.is_leaf:
            made_on = torch.autograd.graph.get_gradient_edge(t).node.metadata.get('mzhip_stream', stream)
            if made_on != stream:
                raise MuZeroError('this forward pass is being captured while an autograd graph of the same leaf tensor from '
                                  'another stream is alive: delete its outputs (the loss among them) before capturing')


def remember_leaves(device, output):
    """Notes the stream on the accumulation nodes of `output`'s leaves, for refuse_capture_of_live_leaves."""
    for node, _ in output.grad_fn.next_functions:
        if type(node) is _ACCUMULATE and 'mzhip_stream' not in node.metadata:
            node.metadata['mzhip_stream'] = _current_stream(device.index)
    return output
