"""layer_norm — normalisation of every row of channels, forward and backward, on libn3d.so (csrc/layer_norm.hip).

Not an operator of the reference's layer (whose only norm is `normalize_2nd_moment`): it stands beside the others for models over tokens — w vectors,
tri-plane texels, frames — together with `rotary` and `attention`."""
import functools

import torch

from ... import _lib
from ._tokens import DTYPES, launch, once, pointer, require_same_device, require_tensor, wants_grad


def _rows(x):
    """[rows, C] with dense channels: a view where the strides allow it."""
    c = x.shape[-1]
    if x.ndim != 2:
        x = x.reshape(x.numel() // c, c)
    return x if c == 1 or x.stride(1) == 1 else x.contiguous()


def _new(x):
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


@functools.lru_cache(maxsize=1024)
def _workspace(rows, c, dtype):
    return _lib.lib().n3d_layer_norm_bwd_workspace(rows, c, dtype)


def _forward(x, weight, bias, eps, want_stats):
    x2 = _rows(x)
    rows, c = x2.shape
    y = _new(x)
    affine = bias if weight is None else weight
    stats, at = None, 0
    if want_stats:
        stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)                 # mean, rstd
        at = stats.data_ptr()
    launch(x, _lib.lib().n3d_layer_norm, x2.data_ptr(), pointer(weight), pointer(bias), y.data_ptr(), at, at and at + 4 * rows, rows, c, x2.stride(0), DTYPES[x.dtype],
           0 if affine is None else DTYPES[affine.dtype], eps)
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @once
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        x2, dy2 = _rows(x), _rows(dy)
        rows, c = x2.shape
        dtype = DTYPES[x.dtype]
        affine = ctx.bias_dtype if weight is None else weight.dtype
        dx = _new(x) if want_x else None
        make = torch.empty if rows else torch.zeros
        dw = make(c, dtype=affine, device=x.device) if want_w else None
        db = make(c, dtype=affine, device=x.device) if want_b else None
        if rows:
            ws = torch.empty(_workspace(rows, c, dtype), dtype=torch.float32, device=x.device) if want_w or want_b else None
            at = stats.data_ptr()
            launch(x, _lib.lib().n3d_layer_norm_bwd, dy2.data_ptr(), x2.data_ptr(), pointer(weight), at, at + 4 * rows, pointer(dx), pointer(dw), pointer(db),
                   pointer(ws), rows, c, x2.stride(0), dy2.stride(0), dtype, 0 if affine is None else DTYPES[affine])
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x (float32, float16 or bfloat16; any leading dimensions and strides).

    weight / bias: [C], either may be None, both float32 or both of x's type.  Mean and variance are float32 sums of centred values; y has x's type, rounded
    once.  Differentiable (once) in x, weight and bias; the gradients are bitwise reproducible."""
    require_tensor('layer_norm', 'x', x, DTYPES)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise RuntimeError('layer_norm: x needs a last dimension of at least one channel')
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None:
            require_tensor('layer_norm', name, t, (torch.float32, x.dtype), 1)
            if t.shape[0] != x.shape[-1]:
                raise RuntimeError(f'layer_norm: {name} has {t.shape[0]} elements for {x.shape[-1]} channels')
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError('layer_norm: weight and bias must have one dtype')
    eps = float(eps)
    if not 0 <= eps < float('inf'):
        raise RuntimeError('layer_norm: eps must be a finite number that is not negative')
    require_same_device('layer_norm', x, weight, bias)
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    if wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]
