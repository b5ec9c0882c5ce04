"""layer_norm — normalisation of every row of channels, forward and backward, on libn3d.so (csrc/layer_norm.hip).

Not an operator of the reference's layer (whose only norm is `normalize_2nd_moment`): it stands beside the others for models over tokens — w vectors,
tri-plane texels, frames — together with `rotary` and `attention`."""
import math

import torch

from ... import _lib
from ._tokens import DTYPES, on_device, require_same_device, require_tensor, wants_grad


def _rows(x):
    """[rows, C] with dense channels: a view where the strides allow it."""
    c = x.shape[-1]
    x = x.reshape(x.numel() // c, c)
    return x if c == 1 or x.stride(1) == 1 else x.contiguous()


def _affine_dtype(x, weight, bias):
    return next((t.dtype for t in (weight, bias) if t is not None), torch.float32 if x is None else x.dtype)


def _forward(x, weight, bias, eps, want_stats):
    x2 = _rows(x)
    rows, c = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device) if want_stats else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if want_stats else None
    with on_device(x):
        _lib.check(_lib.lib().n3d_layer_norm(_lib.ptr(x2), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(y), _lib.ptr(mean), _lib.ptr(rstd), rows, c, x2.stride(0),
                                             DTYPES[x.dtype], DTYPES[_affine_dtype(x, weight, bias)], eps, _lib.stream()))
    return y, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.affine_dtype = _affine_dtype(x, weight, bias)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        x2, dy2 = _rows(x), _rows(dy)
        rows, c = x2.shape
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_x else None
        make = torch.empty if rows else torch.zeros
        dw = make(c, dtype=ctx.affine_dtype, device=x.device) if want_w else None
        db = make(c, dtype=ctx.affine_dtype, device=x.device) if want_b else None
        if rows:
            lib, code = _lib.lib(), DTYPES[x.dtype]
            with on_device(x):
                ws = torch.empty(lib.n3d_layer_norm_bwd_workspace(rows, c, code), dtype=torch.float32, device=x.device) if want_w or want_b else None
                _lib.check(lib.n3d_layer_norm_bwd(_lib.ptr(dy2), _lib.ptr(x2), _lib.ptr(weight), _lib.ptr(mean), _lib.ptr(rstd), _lib.ptr(dx), _lib.ptr(dw),
                                                  _lib.ptr(db), _lib.ptr(ws), rows, c, x2.stride(0), dy2.stride(0), code, DTYPES[ctx.affine_dtype], _lib.stream()))
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
    if not (eps >= 0 and math.isfinite(eps)):
        raise RuntimeError('layer_norm: eps must be a finite number that is not negative')
    require_same_device('layer_norm', x, weight, bias)
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    if wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]
