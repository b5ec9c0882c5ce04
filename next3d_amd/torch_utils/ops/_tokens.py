"""What the token operators (layer_norm, rotary, attention) share: element types, argument checks, the device their launches go to.

A call's host time matters here — a block runs these operators on small tensors too, and a Python autograd node already costs some 20 us — so the checks are
flat, buffers are allocated together, and the descriptors are packed in one call."""
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


def require_same_device(op, first, *others):
    """RuntimeError unless all (that are not None) lie on one HIP device."""
    device = first.device
    if device.type != 'cuda':
        _lib.require_device(first)
    for t in others:
        if t is not None and t.device != device:
            _lib.require_device(t)
            raise RuntimeError(f'{op}: all tensors must be on one device (got {device} and {t.device})')


def launch(t, fn, *args):
    """fn(*args, stream) on the device of `t`, on torch's current stream there, whatever the current device is.  The caller's locals keep every tensor of the
    call alive until it returns: by then the work is enqueued, and the allocator's stream order protects the memory."""
    if t.get_device() == _lib._get_device():
        rc = fn(*args, _lib._stream_handle())
    else:
        with torch.cuda.device(t.device):
            rc = fn(*args, _lib._stream_handle())
    if rc != 0:
        _lib.check(rc)


def pointer(t):
    return 0 if t is None else t.data_ptr()


def wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def once(backward):
    """Marks a Function's `backward` as differentiable once: under create_graph its results refuse a second derivative (torch's once_differentiable); without
    it — every ordinary step — the wrapper's bookkeeping is skipped."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return staticmethod(run)
