"""attention — softmax attention over tokens, forward and backward, on libn3d.so (csrc/attention_fwd.hip, csrc/attention_bwd.hip).

Not an operator of the reference's layer; with `layer_norm` and `rotary` it makes the block of a model over w vectors, tri-plane texels or frames.  One call
serves training (with gradients), prompts and single tokens over a cache (few queries, many keys: the keys are split over the chip)."""
import math
import struct

import torch

from ... import _lib
from ._tokens import DTYPES, launch, once, pointer, require_same_device, require_tensor, wants_grad

_PACK = struct.Struct('=15Q15q2f8i')                                     # n3d_attention_desc, field by field


def _operand(t):
    """`t` [B, L, H, D] itself if the kernels can read it where it lies — dense channels, strides of whole 16-byte units, 16-byte aligned — or a dense copy;
    with its (batch, token, head) strides."""
    strides = [s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape)]
    if t.stride(3) != 1 or (strides[0] | strides[1] | strides[2]) & 7 or strides[1] > 1 << 23 or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = t.stride()[:3]
    return t, strides


def _call(q, k, v, opts, out, lse, dout=None, dq=None, dk=None, dv=None):
    """One call of the library: n3d_attention, or with `dout` n3d_attention_bwd."""
    scale, causal, prefix, documents, key_documents, lengths, softcap, slopes = opts
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1:3]
    q_, q_strides = _operand(q)
    k_, k_strides = _operand(k)
    v_, v_strides = _operand(v)
    lib = _lib.lib()
    if dout is None:
        size, run, do_, do_strides = lib.n3d_attention_workspace, lib.n3d_attention, None, (0, 0, 0)
    else:
        size, run = lib.n3d_attention_bwd_workspace, lib.n3d_attention_bwd
        do_, do_strides = _operand(dout)
    desc = _lib.AttentionDesc.from_buffer_copy(_PACK.pack(
        q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), out.data_ptr(), pointer(lse), pointer(prefix), pointer(lengths), pointer(documents), pointer(key_documents),
        pointer(slopes), 0, pointer(do_), pointer(dq), pointer(dk), pointer(dv), *q_strides, *k_strides, *v_strides, *do_strides,
        0 if documents is None else documents.stride(0), 0 if documents is None else key_documents.stride(0), 0, scale, softcap, b, lq, lk, hq, hk, d,
        DTYPES[q.dtype], causal))
    need = size(desc)
    if need:
        if need < 0:
            _lib.check(-1)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        desc.workspace, desc.workspace_bytes = ws.data_ptr(), need
    launch(q, run, desc)


def _forward(q, k, v, opts, want_lse):
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device) if want_lse else None
    if out.numel():
        _call(q, k, v, opts, out, lse)
    return out, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, opts):
        out, lse = _forward(q, k, v, opts, True)
        scale, causal, prefix, documents, key_documents, lengths, softcap, slopes = opts
        ctx.save_for_backward(q, k, v, out, lse, prefix, documents, key_documents, lengths, slopes)
        ctx.numbers = scale, causal, softcap
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @once
    def backward(ctx, dout, _):
        if dout is None:
            return None, None, None, None
        q, k, v, out, lse, prefix, documents, key_documents, lengths, slopes = ctx.saved_tensors
        scale, causal, softcap = ctx.numbers
        want_q, want_k, want_v, _ = ctx.needs_input_grad
        make = torch.empty if q.numel() else torch.zeros                                        # (no queries: nothing flows)
        dq = make(q.shape, dtype=q.dtype, device=q.device) if want_q else None
        dk = dv = None
        if want_k or want_v:
            dk = make(k.shape, dtype=k.dtype, device=k.device)
            dv = make(v.shape, dtype=v.dtype, device=v.device)
        if q.numel():
            _call(q, k, v, (scale, causal, prefix, documents, key_documents, lengths, softcap, slopes), out, lse, dout, dq, dk, dv)
        return dq, dk if want_k else None, dv if want_v else None, None


def _mask_input(name, t, shape):
    require_tensor('attention', name, t, (torch.int32,), len(shape))
    if tuple(t.shape) != shape:
        raise RuntimeError(f'attention: {name} must be {list(shape)} (got {list(t.shape)})')
    return t if t.numel() == 0 or t.stride(-1) == 1 else t.contiguous()


def attention(q, k, v, scale=None, causal=False, prefix=None, documents=None, key_documents=None, lengths=None, softcap=0.0, slopes=None, return_lse=False):
    """softmax(scores) v for q [B, Lq, Hq, D] and k, v [B, Lk, Hk, D] (float16 or bfloat16, any strides; D a multiple of 8 up to 128; Hq a multiple of Hk,
    query head h reads key head h // (Hq // Hk)).  Returns [B, Lq, Hq, D], and with return_lse also the logarithm of each row's sum, [B, Hq, Lq] float32.

    Scores: t = scale * q.k (scale defaults to D ** -0.5);  softcap > 0: t = softcap * tanh(t / softcap);  slopes [Hq] float32: t -= slope * distance.
    lengths [B] int32: only the first n = lengths[b] keys are in use (default: all of them; the others are never read) — a cache that is filled up to
    there.  Query i stands at position i + n - Lq: the last query beside the last key; its distance to key j is |position - j|.
    causal: key j is visible up to the query's position;  prefix [B] int32 (with causal): and every key j < prefix[b].
    documents [B, Lq] / key_documents [B, Lk] int32 (key_documents defaults to documents where Lq == Lk): a query sees the keys of its own document only; a
    negative number belongs to none (padding).  Rows that see nothing are 0, with lse -inf, and have no gradient.  What a row does not see does not reach
    it, not even NaN or infinity.

    Softmax statistics and sums are float32; weights (and in the backward pass dscores) are rounded to the inputs' type for the matrix cores.
    Differentiable (once) in q, k and v; results and gradients are bitwise reproducible."""
    types = (torch.float16, torch.bfloat16)
    require_tensor('attention', 'q', q, types, 4)
    for name, t in (('k', k), ('v', v)):
        require_tensor('attention', name, t, (q.dtype,), 4)
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1:3]
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise RuntimeError(f'attention: k {tuple(k.shape)} and v {tuple(v.shape)} do not match q {tuple(q.shape)}')
    if hk < 1 or hq < 1 or hq % hk:
        raise RuntimeError(f'attention: {hq} query heads are not a multiple of {hk} key heads')
    if not 8 <= d <= 128 or d % 8:
        raise RuntimeError(f'attention: head sizes are multiples of 8 from 8 to 128 (got {d})')
    scale = d ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    if not math.isfinite(scale) or not (softcap >= 0 and math.isfinite(softcap)):
        raise RuntimeError('attention: scale and softcap must be finite numbers, softcap not negative')
    if prefix is not None:
        if not causal:
            raise RuntimeError('attention: a prefix needs causal=True')
        prefix = _mask_input('prefix', prefix, (b,))
    if lengths is not None:
        lengths = _mask_input('lengths', lengths, (b,))
    if documents is None and key_documents is not None:
        raise RuntimeError('attention: key_documents need documents')
    if documents is not None:
        if key_documents is None and lq != lk:
            raise RuntimeError(f'attention: {lq} queries and {lk} keys need key_documents too')
        documents = _mask_input('documents', documents, (b, lq))
        key_documents = documents if key_documents is None else _mask_input('key_documents', key_documents, (b, lk))
    if slopes is not None:
        require_tensor('attention', 'slopes', slopes, (torch.float32,), 1)
        if slopes.shape[0] != hq:
            raise RuntimeError(f'attention: {slopes.shape[0]} slopes for {hq} query heads')
        if slopes.requires_grad:
            raise RuntimeError('attention: slopes have no gradient')
        slopes = slopes.contiguous()
    require_same_device('attention', q, k, v, prefix, documents, key_documents, lengths, slopes)
    opts = (scale, bool(causal), prefix, documents, key_documents, lengths, softcap, slopes)
    if wants_grad(q, k, v):
        out, lse = _Attention.apply(q, k, v, opts)
    else:
        out, lse = _forward(q, k, v, opts, return_lse)
    return (out, lse) if return_lse else out
