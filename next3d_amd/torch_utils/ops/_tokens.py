"""What the token operators (layer_norm, rotary, attention) share: element types and argument checks.  Buffers, launches and autograd nodes are in
csrc/token_ext.cpp, which also refuses the calls that torch's tracers and forward-mode derivatives make: neither sees into the library."""
import torch

from ... import _lib

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}           # N3D_F32 / N3D_F16 / N3D_BF16


def require_tensor(op, name, t, dtypes, ndim=None):
    """RuntimeError unless `t` is a dense tensor (whose memory holds its values: no lazy negation) of one of `dtypes` (and of `ndim` dimensions)."""
    if not isinstance(t, torch.Tensor) or t.layout != torch.strided or t.is_neg():
        raise RuntimeError(f'{op}: {name} must be a (dense) tensor')
    if t.dtype not in dtypes:
        raise RuntimeError(f'{op}: {name} must be {" or ".join(str(d).replace("torch.", "") for d in dtypes)} (got {t.dtype})')
    if ndim is not None and t.ndim != ndim:
        raise RuntimeError(f'{op}: {name} must have {ndim} dimensions (got {t.ndim})')


def require_sizes(op, *sizes):
    """RuntimeError unless all sizes fit the kernels' 31 bits."""
    if max(sizes) >= 1 << 31:
        raise RuntimeError(f'{op}: a size of 2^31 or more ({max(sizes)})')


def require_same_device(op, first, *others):
    """RuntimeError unless all (that are not None) lie on one HIP device."""
    device = first.device
    if device.type != 'cuda':
        _lib.require_device(first)
    for t in others:
        if t is not None and t.device != device:
            _lib.require_device(t)
            raise RuntimeError(f'{op}: all tensors must be on one device (got {device} and {t.device})')
