"""attention — softmax attention over tokens, forward and backward, on libn3d.so (csrc/attention_fwd.hip, csrc/attention_bwd.hip).

Not an operator of the reference's layer; with `layer_norm` and `rotary` it makes the block of a model over w vectors, tri-plane texels or frames.  One call
serves training (with gradients), prompts and single tokens over a cache (few queries, many keys: the keys are split over the chip)."""
import torch

from ... import _lib
from ._tokens import require_same_device, require_sizes, require_tensor


def _mask_input(name, t, shape):
    require_tensor('attention', name, t, (torch.int32,), len(shape))
    if tuple(t.shape) != shape:
        raise RuntimeError(f'attention: {name} must be {list(shape)} (got {list(t.shape)})')
    return t if t.numel() == 0 or t.stride(-1) == 1 else t.contiguous()


def attention(q, k, v, scale=None, causal=False, prefix=None, documents=None, key_documents=None, lengths=None, softcap=0.0, slopes=None, return_lse=False):
    """softmax(scores) v for q [B, Lq, Hq, D] and k, v [B, Lk, Hk, D] (float16 or bfloat16, any strides; D a multiple of 8 up to 128; Hq a multiple of Hk,
    query head h reads key head h // (Hq // Hk)).  Returns [B, Lq, Hq, D], and with return_lse also the logarithm of each row's sum, [B, Hq, Lq] float32.

    Scores: t = scale * q.k (scale defaults to D ** -0.5);  softcap > 0 (to 4096): t = softcap * tanh(t / softcap), off by 2^-22 softcap;  slopes [Hq] float32: t -= slope * distance.
    lengths [B] int32: only the first n = lengths[b] keys are in use (default: all of them; the others are never read) — a cache that is filled up to
    there.  Query i stands at position i + n - Lq: the last query beside the last key; its distance to key j is |position - j|.
    causal: key j is visible up to the query's position;  prefix [B] int32 (with causal): and every key j < prefix[b].
    documents [B, Lq] / key_documents [B, Lk] int32 (key_documents defaults to documents where Lq == Lk): a query sees the keys of its own document only; a
    negative number belongs to none (padding).  Rows that see nothing are 0, with lse -inf, and have no gradient.  What a row does not see does not reach
    it, not even NaN or infinity.

    Softmax statistics and sums are float32; weights (and in the backward pass dscores) are rounded to the inputs' type for the matrix cores.  float16
    dscores take a power of two of each query's own (of each key's own for dk), so gradients of any size keep their digits.  Differentiable (once) in q, k and v, not through the logarithms; results and gradients are bitwise reproducible, results also
    with and without gradients being recorded.  Refused: 2^24 blocks of rows (128 queries of a head, or 32 queries and heads where there are few) or more."""
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
    require_sizes('attention', b, lq, lk, hq)
    scale = d ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    if not abs(scale) <= 2.0 ** 100 or not (softcap == 0 or 2.0 ** -100 <= softcap <= 4096):
        raise RuntimeError('attention: scale must be finite (within 2^100), softcap 0 (none) or between 2^-100 and 4096')
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
    out, lse = _lib.token_ext().attention(q, k, v, scale, bool(causal), prefix, documents, key_documents, lengths, softcap, slopes, bool(return_lse))
    return (out, lse) if return_lse else out
