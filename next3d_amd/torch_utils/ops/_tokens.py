"""What the token operators (layer_norm, rotary, attention) share: element types, argument checks, the device their launches go to."""
import contextlib

import torch

from ... import _lib

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}           # N3D_F32 / N3D_F16 / N3D_BF16


def require_tensor(op, name, t, dtypes, ndim=None):
    """RuntimeError unless `t` is a dense tensor of one of `dtypes` (and of `ndim` dimensions)."""
    if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
        raise RuntimeError(f'{op}: {name} must be a (dense) tensor')
    if t.dtype not in dtypes:
        raise RuntimeError(f'{op}: {name} must be {" or ".join(str(d).replace("torch.", "") for d in dtypes)} (got {t.dtype})')
    if ndim is not None and t.ndim != ndim:
        raise RuntimeError(f'{op}: {name} must have {ndim} dimensions (got {t.ndim})')


def require_same_device(op, *tensors):
    _lib.require_device(*tensors)
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        raise RuntimeError(f'{op}: all tensors must be on one device (got {", ".join(sorted(str(d) for d in devices))})')


def on_device(t):
    """Launches inside go to the device of `t` and to torch's current stream there, whatever the current device is."""
    if t.device.index is None or t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
