"""Argument checks and launches of operators that are bound with ctypes."""
import torch

from . import _lib
from .exceptions import MuZeroError

DTYPES = {torch.float32: _lib.MZ_F32, torch.float16: _lib.MZ_F16, torch.bfloat16: _lib.MZ_BF16}

# the current stream's handle; the call behind torch.cuda.current_stream, which takes 25 times as long to wrap it
_current_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


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
