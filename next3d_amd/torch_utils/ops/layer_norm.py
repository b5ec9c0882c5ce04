"""layer_norm — normalisation of every row of channels, forward and backward, on libn3d.so (csrc/layer_norm.hip).

Not an operator of the reference's layer (whose only norm is `normalize_2nd_moment`): it stands beside the others for models over tokens — w vectors,
tri-plane texels, frames — together with `rotary` and `attention`."""
import torch

from ... import _lib
from ._tokens import DTYPES, require_same_device, require_sizes, require_tensor


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x (float32, float16 or bfloat16; any leading dimensions and strides).

    weight / bias: [C], either may be None, both float32 or both of x's type.  Mean and variance are float32 sums of centred values; y has x's type, rounded
    once.  Differentiable (once) in x, weight and bias; the gradients are bitwise reproducible."""
    require_tensor('layer_norm', 'x', x, DTYPES)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise RuntimeError('layer_norm: x needs a last dimension of at least one channel')
    require_sizes('layer_norm', x.shape[-1])
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
    return _lib.token_ext().layer_norm(x, weight, bias, eps)
