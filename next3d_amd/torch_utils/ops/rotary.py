"""rotary — rotary positions with several axes (time, height, width) for tokens of images and videos, on libn3d.so (csrc/rotary.hip).

Not an operator of the reference's layer; it turns the queries and keys of `attention`."""
import operator

import torch

from ... import _lib
from ._tokens import DTYPES, require_same_device, require_sizes, require_tensor

_POSITIONS = (torch.float32, torch.int32, torch.int64)


def rotary(q, positions, sections, k=None, base=10000.0, pairing='interleaved', ladder='axis'):
    """q [B, L, Hq, D] — and k [B, L, Hk, D], in the same launch — with every pair of channels turned by its axis's position.

    positions: [L, A], or [B, L, A], float32 / int32 / int64, A = 1..4 axes (time, height, width, ...).  sections: A even numbers of channels, one per
    axis, in order; channels behind their sum pass through.  Pair i of an axis of s channels turns by position * base**(-2 i / s) (ladder='axis'); with
    ladder='shared' pair p of all P pairs turns by its axis's position * base**(-p / P).  pairing='interleaved': a pair is two neighbouring channels;
    pairing='half': channels i and i + half, the halves of the axis's section (ladder='axis') or of all rotated channels (ladder='shared').
    q and k: float32, float16 or bfloat16, any strides.  Angles are taken in 64 bits; results are rounded once.  Returns the turned q, or (q, k);
    differentiable (once) in q and k."""
    require_tensor('rotary', 'q', q, DTYPES, 4)
    if k is not None:
        require_tensor('rotary', 'k', k, (q.dtype,), 4)
        if k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
            raise RuntimeError(f'rotary: k {tuple(k.shape)} does not have the batch, tokens and channels of q {tuple(q.shape)}')
    require_tensor('rotary', 'positions', positions, _POSITIONS)
    b, l, _, d = q.shape
    require_sizes('rotary', b * l)
    try:
        sections = tuple(operator.index(s) for s in sections)
    except TypeError:
        raise RuntimeError(f'rotary: sections must be whole numbers (got {sections!r})') from None
    if not 1 <= len(sections) <= 4 or any(s < 0 or s % 2 for s in sections) or not 0 < sum(sections) <= d:
        raise RuntimeError(f'rotary: sections must be 1 to 4 even numbers of channels that add up to 2..{d} (got {sections})')
    if d > 1024:
        raise RuntimeError(f'rotary: more than 1024 channels (got {d})')
    if q.shape[2] + (0 if k is None else k.shape[2]) > 4096:
        raise RuntimeError('rotary: more than 4096 heads')
    if tuple(positions.shape) not in ((l, len(sections)), (1, l, len(sections)), (b, l, len(sections))):
        raise RuntimeError(f'rotary: positions must be [{l}, {len(sections)}] or [{b}, {l}, {len(sections)}] (got {tuple(positions.shape)})')
    if pairing not in ('interleaved', 'half') or ladder not in ('axis', 'shared'):
        raise RuntimeError(f"rotary: pairing is 'interleaved' or 'half', ladder 'axis' or 'shared' (got {pairing!r}, {ladder!r})")
    base = float(base)
    if not 0 < base < float('inf'):
        raise RuntimeError('rotary: base must be a positive finite number')
    if positions.requires_grad:
        raise RuntimeError('rotary: positions have no gradient')
    require_same_device('rotary', q, k, positions)
    yq, yk = _lib.token_ext().rotary(q, k, positions, sections, base, pairing == 'interleaved', ladder == 'shared')
    return yq if k is None else (yq, yk)
