"""rotary — rotary positions with several axes (time, height, width) for tokens of images and videos, on libn3d.so (csrc/rotary.hip).

Not an operator of the reference's layer; it turns the queries and keys of `attention`."""
import struct

import torch

from ... import _lib
from ._tokens import DTYPES, launch, once, pointer, require_same_device, require_tensor, wants_grad

_POSITIONS = {torch.float32: 0, torch.int32: 1, torch.int64: 2}
_PACK = struct.Struct('=5Q8qd15i4x')                                     # n3d_rotary_desc, field by field


def _turn(q, k, positions, plan, inverse):
    sections, base, interleaved, shared = plan
    first = k if q is None else q
    b, l, _, d = first.shape
    yq = yk = None
    q_strides = k_strides = (0, 0, 0)
    if q is not None:
        if q.stride(3) != 1:
            q = q.contiguous()
        yq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        q_strides = q.stride()[:3]
    if k is not None:
        if k.stride(3) != 1:
            k = k.contiguous()
        yk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        k_strides = k.stride()[:3]
    desc = _lib.RotaryDesc.from_buffer_copy(_PACK.pack(
        pointer(q), pointer(k), positions.data_ptr(), pointer(yq), pointer(yk), *q_strides, *k_strides,
        positions.stride(0) if positions.ndim == 3 and positions.shape[0] > 1 else 0, positions.stride(-2), base, b, l, 0 if q is None else q.shape[2],
        0 if k is None else k.shape[2], d, len(sections), *sections, *(0,) * (4 - len(sections)), DTYPES[first.dtype], _POSITIONS[positions.dtype], interleaved,
        shared, inverse))
    launch(first, _lib.lib().n3d_rotary, desc)
    return yq, yk


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, plan):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.plan = plan
        yq, yk = _turn(q, k, positions, plan, False)
        return yq if k is None else (yq, yk)

    @once
    def backward(ctx, dq, dk=None):
        positions, = ctx.saved_tensors
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is None and dk is None:
            return None, None, None, None
        return (*_turn(dq, dk, positions, ctx.plan, True), None, None)


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
    sections = tuple(int(s) for s in sections)
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
    if positions.stride(-1) != 1:
        positions = positions.contiguous()
    plan = (sections, base, pairing == 'interleaved', ladder == 'shared')
    if wants_grad(q, k):
        return _Rotary.apply(q, k, positions, plan)
    yq, yk = _turn(q, k, positions, plan, False)
    return yq if k is None else (yq, yk)
