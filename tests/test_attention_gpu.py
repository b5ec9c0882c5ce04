"""-m gpu tests of `attention` against its definition in float64 (tests/_token_ref.py, bounds derived there)."""
import pytest
import torch

import _token_ref as R

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _randn(shape, seed, dtype, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _inputs(b, lq, lk, hq, hk, d, dtype, seed=0):
    return (_randn((b, lq, hq, d), seed, dtype), _randn((b, lk, hk, d), seed + 1, dtype), _randn((b, lk, hk, d), seed + 2, dtype),
            _randn((b, lq, hq, d), seed + 3, dtype))


def _docs(b, n, count, seed=0, pad=0):
    cuts = torch.randint(0, max(n - pad, 1), (b, count - 1), generator=torch.Generator().manual_seed(seed)).sort(dim=1).values
    ids = (torch.arange(n)[None, :, None] >= cuts[:, None, :]).sum(2).to(torch.int32)
    if pad:
        ids[:, n - pad:] = -1
    return ids


def _to(dev, kw):
    return {name: t.to(dev) if isinstance(t, torch.Tensor) else t for name, t in kw.items()}


def _check(dev, q, k, v, do=None, what='', **kw):
    """Forward (with lse) and, with `do`, the gradients; returns what came out."""
    from next3d_amd.torch_utils.ops import attention
    leaves = [t.to(dev).requires_grad_(do is not None) for t in (q, k, v)]
    out, lse = attention.attention(*leaves, return_lse=True, **_to(dev, kw))
    got = dict(out=out, lse=lse)
    if do is not None:
        got.update(zip(('dq', 'dk', 'dv'), torch.autograd.grad(out, leaves, do.to(dev))))
    vals, tols = R.attention(q, k, v, do, **kw)
    for name, t in got.items():
        want, tol = vals[name], tols[name]
        if name == 'lse':
            empty = want == float('-inf')
            assert torch.equal(t.cpu() == float('-inf'), empty), what
            t, want, tol = t.cpu()[~empty], want[~empty], tol[~empty]
        R.assert_within(t, want, tol, f'{what} {name}')
    return {name: t.detach() for name, t in got.items()}


SIZES = [  # B, Lq, Lk, Hq, Hk, D
    (1, 1, 1, 1, 1, 64), (2, 1, 77, 4, 2, 128), (1, 3, 200, 2, 2, 32), (2, 65, 65, 2, 1, 64), (1, 129, 300, 3, 3, 72), (1, 300, 129, 4, 1, 128), (2, 128, 128, 2, 2, 96),
    (1, 257, 191, 2, 1, 8), (1, 66, 1000, 1, 1, 80), (1, 200, 64, 6, 2, 40)]


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('size', SIZES, ids=str)
def test_attention(dev, size, dtype, causal):
    q, k, v, do = _inputs(*size, dtype)
    _check(dev, q, k, v, do, causal=causal)


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('d', [64, 128])
def test_attention_score_forms(dev, d, dtype):
    b, n, hq, hk = 2, 150, 4, 2
    q, k, v, do = _inputs(b, n, n, hq, hk, d, dtype, 7)
    slopes = 2.0 ** -torch.arange(1.0, hq + 1)
    prefix = torch.tensor([0, 70], dtype=torch.int32)
    docs = _docs(b, n, 5, 1, pad=20)
    for kw in (dict(softcap=4.0), dict(slopes=slopes), dict(causal=True, prefix=prefix), dict(documents=docs), dict(documents=docs, causal=True),
               dict(causal=True, prefix=prefix, documents=docs, softcap=10.0, slopes=slopes), dict(scale=0.0), dict(scale=-0.3), dict(scale=0.7, softcap=1.0)):
        _check(dev, q, k, v, do, what=str(sorted(kw)), **kw)


@pytest.mark.parametrize('dtype', [F16, BF16])
def test_attention_lengths(dev, dtype):
    """A cache filled to different lengths, zero and full among them: few queries (keys split over the chip), and many."""
    lengths = torch.tensor([0, 1, 63, 64, 65, 700, 1500, 5000], dtype=torch.int32)         # (5000: more than there are, all 1500)
    for lq, hq, hk, d in ((1, 4, 1, 128), (5, 2, 2, 64), (40, 2, 1, 80), (100, 1, 1, 64)):
        q, k, v, do = _inputs(8, lq, 1500, hq, hk, d, dtype, 3)
        for kw in (dict(), dict(causal=True), dict(causal=True, prefix=torch.tensor([9, 0, 100, 3, 65, 1, 1500, 2000], dtype=torch.int32))):
            _check(dev, q, k, v, do if lq in (5, 100) else None, what=f'{lq} {sorted(kw)}', lengths=lengths, **kw)
    q, k, v, do = _inputs(1, 3, 9, 1, 1, 16, dtype, 3)
    _check(dev, q, k, v, do, lengths=torch.tensor([-4], dtype=torch.int32))


@pytest.mark.parametrize('dtype', [F16, BF16])
def test_attention_few_queries_of_large_groups(dev, dtype):
    lengths = torch.tensor([700, 0, 333], dtype=torch.int32)
    for lq, hq, hk, d in ((5, 32, 2, 128), (32, 6, 1, 64), (33, 6, 1, 64), (1, 71, 1, 80), (17, 12, 2, 40)):
        q, k, v, do = _inputs(3, lq, 700, hq, hk, d, dtype, 79)
        _check(dev, q, k, v, what=f'{lq}', causal=True, lengths=lengths, softcap=9.0)
        _check(dev, q, k, v, do, what=f'{lq}', documents=_docs(3, lq, 3, 8), key_documents=_docs(3, 700, 3, 9))


def test_attention_never_reads_behind_the_length(dev):
    """NaN behind the last key in use reaches nothing, and the gradients there are zero."""
    for lq in (1, 33, 200):
        q, k, v, do = _inputs(2, lq, 300, 2, 1, 64, BF16, 5)
        k[:, 250:], v[:, 250:] = float('nan'), float('inf')
        got = _check(dev, q, k, v, do, lengths=torch.tensor([250, 100], dtype=torch.int32))
        assert int(got['dk'][:, 250:].abs().sum()) == 0 and int(got['dv'][1, 100:].abs().sum()) == 0


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_attention_masked_nonfinite_stays_away(dev, bad):
    """NaN or infinity in tokens of another document, behind the diagonal or in padding does not reach the rows that do not see them — forward (tiles with
    matrix products over masked keys) and in every gradient."""
    b, n, d = 1, 190, 64
    for dtype, hq, hk in ((F16, 2, 2), (BF16, 4, 1)):
        q, k, v, do = _inputs(b, n, n, hq, hk, d, dtype, 11)
        docs = _docs(b, n, 3, 2, pad=30)
        pad = docs[0] < 0
        for t in (q, k, v, do):                                             # padding: seen by nobody, sees nothing
            t[:, pad] = bad
        _check(dev, q, k, v, do, what='padding', documents=docs)
        q, k, v, do = _inputs(b, n, n, hq, hk, d, dtype, 12)
        docs = _docs(b, n, 2, 3)
        cut = int((docs[0] == 0).sum())
        for t, name in ((k, 'k'), (v, 'v'), (q, 'q'), (do, 'do')):
            spoiled = dict(q=q, k=k, v=v, do=do)
            spoiled[name] = t.clone()
            spoiled[name][:, cut + 5] = bad                                 # in the second document: the first must not notice
            clean = _run(dev, q, k, v, do, documents=docs)
            got = _run(dev, *(spoiled[x] for x in ('q', 'k', 'v', 'do')), documents=docs)
            for key in ('out', 'dq', 'dk', 'dv'):
                assert bool(torch.isfinite(got[key][:, :cut]).all()), (name, key)
                assert float((got[key][:, :cut].float() - clean[key][:, :cut].float()).abs().max()) <= 0.05, (name, key)
        q, k, v, do = _inputs(b, n, n, hq, hk, d, dtype, 13)
        v[:, 100] = bad                                                     # causal: queries before 100 do not see it
        got = _run(dev, q, k, v, do, causal=True)
        vals, tols = R.attention(q[:, :100], k[:, :100], v[:, :100], do[:, :100], causal=True)
        R.assert_within(got['out'][:, :100], vals['out'], tols['out'], 'before the bad key')
        R.assert_within(got['dq'][:, :100], vals['dq'], tols['dq'], 'before the bad key')
        assert not bool(torch.isfinite(got['out'][:, 100:]).any())
        for lq in (1, 4):                                                   # few queries over a cache
            q, k, v, _ = _inputs(2, lq, 600, hq, hk, d, dtype, 14)
            kd = _docs(2, 600, 2, 4)
            qd = torch.zeros(2, lq, dtype=torch.int32)
            for x in range(2):
                v[x, kd[x] == 1], k[x, kd[x] == 1] = bad, bad
            _check(dev, q, k, v, what='cache', documents=qd, key_documents=kd)


def _run(dev, q, k, v, do, **kw):
    from next3d_amd.torch_utils.ops import attention
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    out = attention.attention(*leaves, **_to(dev, kw))
    return dict(zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *torch.autograd.grad(out, leaves, do.to(dev)))))


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('size', [(1, 1100, 1200, 1, 1, 64), (1, 2100, 1030, 2, 1, 128), (2, 1031, 2500, 2, 2, 72), (1, 130, 4100, 2, 1, 32), (1, 4100, 70, 3, 1, 96)], ids=str)
def test_attention_few_heads_of_long_sequences(dev, size, dtype):
    """Few workgroups' worth of rows: the long axis is split as well, also where runs of it are empty, masked or hold NaN behind the mask."""
    b, lq, lk, hq, hk, d = size
    q, k, v, do = _inputs(*size, dtype, 17)
    prefix, lengths = torch.full((b,), lk // 3, dtype=torch.int32), torch.full((b,), lk - 37, dtype=torch.int32)
    _check(dev, q, k, v, do, what='plain')
    _check(dev, q, k, v, do, what='causal', causal=True, prefix=prefix, softcap=8.0)
    spoiled = k.clone()
    spoiled[:, lk - 37:] = float('nan')
    _check(dev, q, spoiled, v, do, what='lengths', causal=True, lengths=lengths, slopes=2.0 ** -torch.arange(1.0, hq + 1))
    qd, kd = _docs(b, lq, 4, 5, pad=9), _docs(b, lk, 4, 6, pad=11)
    for t, ids in ((k, kd), (v, kd), (q, qd), (do, qd)):
        t[ids < 0] = float('nan')
    _check(dev, q, k, v, do, what='documents', documents=qd, key_documents=kd)
    _check(dev, q, k, v, do, what='causal documents', documents=qd, key_documents=kd, causal=True)


def test_attention_documents_out_of_order(dev):
    """Documents need not be sorted, and queries and keys may carry different ones."""
    g = torch.Generator().manual_seed(1)
    for lq, lk in ((150, 270), (3, 900)):
        q, k, v, do = _inputs(2, lq, lk, 2, 1, 64, F16, 21)
        qd = torch.randint(-1, 6, (2, lq), generator=g).to(torch.int32)
        kd = torch.randint(-1, 7, (2, lk), generator=g).to(torch.int32)
        _check(dev, q, k, v, do, documents=qd, key_documents=kd)
        _check(dev, q, k, v, do, documents=torch.full_like(qd, -1), key_documents=kd)


@pytest.mark.parametrize('causal', [False, True])
def test_attention_many_blocks_of_uneven_documents(dev, causal):
    """More workgroups than the chip holds at once: the blocks are taken in another order, each one once — documents in order, shuffled, one, and padding."""
    b, n, heads, d = 3, 1300, 32, 8
    q, k, v, do = _inputs(b, n, n, heads, heads, d, BF16, 25)
    docs = _docs(b, n, 9, 7, pad=300)
    docs[1] = docs[1, torch.randperm(n, generator=torch.Generator().manual_seed(3))]
    docs[2] = 0
    _check(dev, q, k, v, do, documents=docs, causal=causal)
    _check(dev, q, k, v, do, documents=docs, causal=causal, lengths=torch.tensor([1300, 1000, 0], dtype=torch.int32))


@pytest.mark.parametrize('lengths', [(64, 64, 128), (128, 128), (300, 20), (1, 255), (130, 0, 62)], ids=str)
def test_attention_padding_beside_a_single_document(dev, lengths):
    """Tiles and blocks that hold one document and padding in every arrangement: whole tiles of either, and tiles shared by both."""
    n, d = sum(lengths), 64
    for pattern in range(2 ** len(lengths)):
        ids = torch.cat([torch.full((l,), 3 if pattern >> i & 1 else -5, dtype=torch.int32) for i, l in enumerate(lengths)])[None]
        q, k, v, do = _inputs(1, n, n, 2, 1, d, BF16, 26)
        for t in (q, k, v, do):
            t[ids < 0] = float('nan')
        _check(dev, q, k, v, do, what=f'{pattern}', documents=ids)
        _check(dev, q, k, v, do, what=f'{pattern} causal', documents=ids, causal=True)


def test_attention_small_and_large_gradients_float16(dev):
    """float16 gradients of any size keep their relative accuracy (the dscores get a power of two of their own)."""
    for size in (1e-6, 1e-3, 300.0):
        q, k, v, do = _inputs(1, 200, 200, 2, 1, 64, F16, 31)
        _check(dev, q, k, v, (do.float() * size).to(F16), causal=True, what=f'{size}')
    q, k, v, do = _inputs(1, 150, 150, 1, 1, 32, F16, 32)
    _check(dev, q, k, (v.float() * 100).to(F16), (do.float() * 100).to(F16))


def test_attention_extreme_scores(dev):
    """Scores far apart: one key takes all; the running maximum rises tile after tile, or falls."""
    b, n, d = 1, 400, 64
    q, k, v, do = _inputs(b, n, n, 1, 1, d, BF16, 41)
    ramp = torch.linspace(-1, 1, n)[None, :, None, None]
    for sign in (1, -1):
        for size in (1.0, 8.0):
            qq = (q.float().abs() * size).to(BF16)
            kk = (k.float().abs() * ramp * sign * size).to(BF16)
            _check(dev, qq, kk, v, do, what=f'{sign} {size}')


def test_attention_strides(dev):
    """Heads-first tensors, slices of one projection, broadcast keys, odd offsets; gradients that are expanded."""
    from next3d_amd.torch_utils.ops import attention
    fused = _randn((2, 90, 12, 64), 51, F16).to(dev)
    heads_first = fused.transpose(1, 2).contiguous().transpose(1, 2)
    odd = _randn((2, 90, 12, 67), 52, F16).to(dev)[..., 3:]
    flat = torch.empty(2 * 90 * 12 * 64 + 4, dtype=F16, device=dev)[4:].view(2, 90, 12, 64).copy_(fused)
    wide = _randn((2, 90, 12, 128), 53, F16).to(dev)
    for src in (fused, heads_first, odd, flat, wide[..., ::2], wide[..., 32:96], fused[:1].expand(2, 90, 12, 64), fused[:, :1].expand(2, 90, 12, 64)):
        parts = [src[:, :, :6], src[:, :, 6:9], src[:, :, 9:]]
        results = []
        for ts in (parts, [t.clone(memory_format=torch.contiguous_format) for t in parts]):
            leaves = [t.detach().requires_grad_() for t in ts]
            out = attention.attention(*leaves, causal=True)
            one = torch.full((), 0.5, dtype=F16, device=dev).expand(out.shape)
            results.append([out, *torch.autograd.grad(out, leaves, one)])
        assert all(torch.equal(a, c) for a, c in zip(*results))


def test_attention_offsets_beyond_32_bits(dev):
    """One head of a cache whose tokens lie 16 KB apart: its last keys are 4.9 GB behind the first; single tokens, many queries, and the gradients."""
    lk, d = 300000, 8
    cache = torch.empty((2, lk, 64, 2 * 64), dtype=BF16, device=dev)
    k, v = _randn((2, lk, 1, d), 65, BF16), _randn((2, lk, 1, d), 66, BF16)
    cache[:, :, 63:, :d], cache[:, :, 63:, 64:64 + d] = k.to(dev), v.to(dev)
    lengths = torch.tensor([lk, lk - 999], dtype=torch.int32)
    for lq, train in ((1, False), (65, False), (3, True)):
        q, do = _randn((2, lq, 1, d), 67, BF16), _randn((2, lq, 1, d), 68, BF16)
        from next3d_amd.torch_utils.ops import attention
        leaves = [q.to(dev).requires_grad_(train), cache[:, :, 63:, :d].detach().requires_grad_(train), cache[:, :, 63:, 64:64 + d].detach().requires_grad_(train)]
        out = attention.attention(*leaves, causal=True, lengths=lengths.to(dev))
        vals, tols = R.attention(q, k, v, do if train else None, causal=True, lengths=lengths)
        got = dict(out=out)
        if train:
            got.update(zip(('dq', 'dk', 'dv'), torch.autograd.grad(out, leaves, do.to(dev))))
        for name, t in got.items():
            R.assert_within(t, vals[name], tols[name], f'{lq} {name}')
    del cache, leaves, out, got
    torch.cuda.empty_cache()


def test_attention_caps_from_tiny_to_large(dev):
    q, k, v, do = _inputs(1, 100, 100, 2, 1, 64, F16, 69)
    q[0, 7], k[0, 9] = 0, 0                                                 # scores of exactly zero
    for kw in (dict(softcap=2.0 ** -90), dict(softcap=2.0 ** -90, scale=1000.0), dict(softcap=4096.0), dict(softcap=0.01, causal=True, slopes=torch.tensor([0.5, 0.0]))):
        _check(dev, q, k, v, do, what=str(sorted(kw)), **kw)


def test_attention_one_tensor_as_query_key_and_value(dev):
    from next3d_amd.torch_utils.ops import attention
    x, _, _, do = _inputs(2, 77, 77, 2, 2, 64, BF16, 73)
    leaf = x.to(dev).requires_grad_()
    got, = torch.autograd.grad(attention.attention(leaf, leaf, leaf, causal=True), leaf, do.to(dev))
    each = _run(dev, x, x, x, do, causal=True)
    want = each['dq'].double() + each['dk'].double() + each['dv'].double()
    size = each['dq'].double().abs() + each['dk'].double().abs() + each['dv'].double().abs()
    assert bool(((got.double() - want).abs() <= 2 * 2.0 ** -8 * size).all())               # (two additions in bfloat16)


def test_attention_lazily_negated_gradients(dev):
    q, k, v, do = _inputs(1, 40, 40, 1, 1, 16, F16, 74)
    plain, negated = _run(dev, q, k, v, -do), _run_neg(dev, q, k, v, do)
    assert all(torch.equal(plain[n], negated[n]) for n in ('dq', 'dk', 'dv'))


def _run_neg(dev, q, k, v, do):
    from next3d_amd.torch_utils.ops import attention
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    return dict(zip(('dq', 'dk', 'dv'), torch.autograd.grad(attention.attention(*leaves), leaves, torch._neg_view(do.to(dev)))))


def test_attention_calls_side_by_side(dev):
    """Calls of several forms in flight on four streams at once give what they give alone."""
    from next3d_amd.torch_utils.ops import attention
    work = [(_inputs(1, 900, 900, 4, 2, 64, F16, 75), dict(causal=True)), (_inputs(2, 1, 4000, 8, 2, 128, BF16, 76), dict()), (_inputs(1, 1700, 1700, 1, 1, 64, BF16, 77), dict()),
            (_inputs(2, 500, 500, 2, 2, 72, F16, 78), dict(documents=_docs(2, 500, 4)))]
    work = [([t.to(dev) for t in ts], _to(dev, kw)) for ts, kw in work]

    def step(ts, kw):
        leaves = [t.detach().requires_grad_() for t in ts[:3]]
        out = attention.attention(*leaves, **kw)
        return [out.detach(), *torch.autograd.grad(out, leaves, ts[3])]

    alone = [step(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(5):
        together = []
        for s, w in zip(streams, work):
            with torch.cuda.stream(s):
                together.append(step(*w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for x, y in zip(alone, together) for a, c in zip(x, y))


def test_attention_empty(dev):
    from next3d_amd.torch_utils.ops import attention
    for b, lq, lk in ((0, 4, 4), (2, 0, 5), (2, 5, 0)):
        q, k, v, do = (t.to(dev) for t in _inputs(b, lq, lk, 2, 1, 16, F16))
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out, lse = attention.attention(*leaves, return_lse=True)
        grads = torch.autograd.grad(out, leaves, do)
        assert out.shape == q.shape and not bool(out.abs().sum()) and bool((lse == float('-inf')).all())
        assert [g.shape for g in grads] == [t.shape for t in leaves] and not any(bool(g.abs().sum()) for g in grads)


def test_attention_partial_gradients_and_differences(dev):
    from next3d_amd.torch_utils.ops import attention
    q, k, v, do = _inputs(1, 70, 70, 2, 1, 64, F16, 61)
    kw = dict(causal=True, softcap=5.0, slopes=torch.tensor([0.1, 0.02]))
    full = _run(dev, q, k, v, do, **kw)
    for which, name in enumerate(('dq', 'dk', 'dv')):
        leaves = [t.to(dev).requires_grad_(i == which) for i, t in enumerate((q, k, v))]
        got, = torch.autograd.grad(attention.attention(*leaves, **_to(dev, kw)), leaves[which], do.to(dev))
        assert torch.equal(got, full[name])
    h = 1e-4
    _, tols = R.attention(q, k, v, do, **kw)
    for i, name in enumerate(('dq', 'dk', 'dv')):
        step = _randn((q, k, v)[i].shape, 62 + i, torch.float64)
        vary = lambda s: [t.double() + s * h * step if x == i else t.double() for x, t in enumerate((q, k, v))]
        f = [float((_out64(*vary(s), **kw) * do.double()).sum()) for s in (1, -1)]
        analytic = float((full[name].cpu().double() * step).sum())
        # the float64 differences are exact to h^2 ~ 1e-8 of their terms; the kernel's gradient is within its bound, element by element
        assert abs((f[0] - f[1]) / (2 * h) - analytic) <= float((tols[name] * step.abs()).sum()) + 1e-5 * float((full[name].cpu().double() * step).abs().sum())


def _out64(q, k, v, causal, softcap, slopes):
    group = q.shape[2] // k.shape[2]
    q, k, v = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(group, 1), v.transpose(1, 2).repeat_interleave(group, 1)
    t = softcap * torch.tanh(q @ k.transpose(2, 3) * q.shape[3] ** -0.5 / softcap)
    n = q.shape[2]
    dist = (torch.arange(n)[:, None] - torch.arange(n)[None]).double()
    t = (t - slopes.double()[None, :, None, None] * dist.abs()).masked_fill(dist < 0, float('-inf'))
    return (torch.softmax(t, 3) @ v).transpose(1, 2)


def test_attention_reproducible_on_another_stream_and_in_graphs(dev):
    from next3d_amd.torch_utils.ops import attention
    cases = [(_inputs(2, 200, 200, 4, 2, 64, F16, 71), dict(documents=_docs(2, 200, 4), causal=True)), (_inputs(3, 1, 2000, 8, 2, 128, F16, 72), dict(causal=True, lengths=torch.tensor([1, 700, 2000], dtype=torch.int32)))]
    for tensors, kw in cases:
        q, k, v, do = (t.to(dev) for t in tensors)
        kw = _to(dev, kw)

        def step():
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            out = attention.attention(*leaves, **kw)
            return [out.detach(), *torch.autograd.grad(out, leaves, do)]

        want = [t.clone() for t in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, c) for a, c in zip(want, again))
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = step()
            graphs.append((g, out))
        for seed in range(3):
            q.copy_(_randn(tuple(q.shape), 80 + seed, F16))
            want = [t.clone() for t in step()]
            side.wait_stream(torch.cuda.current_stream())
            graphs[0][0].replay()
            with torch.cuda.stream(side):
                graphs[1][0].replay()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(a, c) for a, c in zip(want, out))


def test_attention_many_short_sequences(dev):
    """More sequences than a launch's second dimension holds, with documents."""
    b, n = 70000, 6
    q, k, v, do = _inputs(b, n, n, 1, 1, 8, BF16, 82)
    docs = torch.tensor([0, 0, 1, 1, 1, -1], dtype=torch.int32).repeat(b, 1)
    _check(dev, q, k, v, do, documents=docs, causal=True)


def test_attention_split_and_ordered_calls_in_graphs(dev):
    """Calls whose work is split over the long axis, or taken in the order of the documents' lengths, replayed beside eager ones."""
    from next3d_amd.torch_utils.ops import attention
    for size, kw in (((1, 1700, 1700, 2, 1, 64), dict(causal=True)), ((2, 1100, 1100, 64, 64, 8), dict(documents=_docs(2, 1100, 7, 4, pad=100)))):
        q, k, v, do = (t.to(dev) for t in _inputs(*size, F16, 83))
        kw = _to(dev, kw)

        def step():
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            out = attention.attention(*leaves, **kw)
            return [out.detach(), *torch.autograd.grad(out, leaves, do)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for seed in range(3):
            q.copy_(_randn(tuple(q.shape), 84 + seed, F16))
            want = [t.clone() for t in step()]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(want, out))


def test_token_block(dev):
    """The three operators as a block uses them — normalise, project, turn, attend, add — forward and gradients, against the same block in float64."""
    from next3d_amd.torch_utils.ops import attention, layer_norm, rotary
    b, t, h, w, heads, kv, d = 1, 2, 5, 7, 4, 2, 32
    n, c = t * h * w, heads * d
    pos = torch.stack(torch.meshgrid(torch.arange(t), torch.arange(h), torch.arange(w), indexing='ij'), -1).reshape(n, 3).to(torch.int32)
    x, weight, bias, g = _randn((b, n, c), 91, F16), 1 + 0.1 * torch.randn(c, generator=torch.Generator().manual_seed(92)), _randn((c,), 93, torch.float32, 0.1), _randn((b, n, c), 94, F16)
    proj = _randn((c, (heads + 2 * kv) * d), 95, F16, c ** -0.5)

    def block(x, weight, bias, proj, norm, turn, attend):
        y = norm(x, weight, bias) @ proj
        q, k, v = y.reshape(b, n, heads + 2 * kv, d).split([heads, kv, kv], dim=2)
        q, k = turn(q, k)
        return x + attend(q, k, v).reshape(b, n, c)

    leaves = [p.to(dev).requires_grad_() for p in (x, weight, bias, proj)]
    out = block(*leaves, layer_norm.layer_norm, lambda q, k: rotary.rotary(q, pos.to(dev), (8, 12, 12), k=k, pairing='half'),
                lambda q, k, v: attention.attention(q, k, v, softcap=20.0))
    got = [out, *torch.autograd.grad(out, leaves, g.to(dev))]

    def norm64(x, weight, bias):
        z = x - x.mean(-1, keepdim=True)
        return z / (z.square().mean(-1, keepdim=True) + 1e-5).sqrt() * weight + bias

    def turn64(q, k):
        ang = torch.cat([pos[:, a, None].double() * 10000.0 ** (-torch.arange(0, s, 2).double() / s) for a, s in enumerate((8, 12, 12))], 1)
        lo = torch.cat([torch.arange(o, o + s // 2) for o, s in ((0, 8), (8, 12), (20, 12))])
        hi = torch.cat([torch.arange(o + s // 2, o + s) for o, s in ((0, 8), (8, 12), (20, 12))])
        order = torch.argsort(torch.cat([lo, hi]))
        cos, sin = ang.cos()[None, :, None], ang.sin()[None, :, None]
        return [torch.cat([z[..., lo] * cos - z[..., hi] * sin, z[..., lo] * sin + z[..., hi] * cos], -1)[..., order] for z in (q, k)]

    def attend64(q, k, v):
        q, k, v = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(heads // kv, 1), v.transpose(1, 2).repeat_interleave(heads // kv, 1)
        return (torch.softmax(20 * torch.tanh(q @ k.transpose(2, 3) * d ** -0.5 / 20), 3) @ v).transpose(1, 2)

    leaves64 = [p.double().requires_grad_() for p in (x, weight, bias, proj)]
    out64 = block(*leaves64, norm64, turn64, attend64)
    want = [out64, *torch.autograd.grad(out64, leaves64, g.double())]
    # six roundings to float16 one behind the other (norm, projection, rotation, weights, output, sum), each 2^-11 of the largest value it meets; gradients
    # pass the same chain and back: twelve, and are sums over the tokens of terms that may cancel, so 2^-11 of the largest magnitude bounds each
    for name, a, ref, roundings in zip(('out', 'x', 'weight', 'bias', 'proj'), got, want, (6, 12, 12, 12, 12)):
        err = float((a.detach().cpu().double() - ref.detach()).abs().max())
        assert err <= roundings * 2.0 ** -11 * float(ref.detach().abs().max()) * 2, (name, err, float(ref.detach().abs().max()))


@pytest.mark.parametrize('dtype', [F16, BF16])
def test_attention_same_bits_with_and_without_gradients(dev, dtype):
    """Short calls, single tokens, documents and long rows: inference gives the bits that a recorded call (and a checkpoint's second pass) gives."""
    from next3d_amd.torch_utils.ops import attention
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    for size, kw in (((2, 7, 77, 8, 8, 64), dict(causal=True, slopes=2.0 ** -torch.arange(1.0, 9))), ((3, 1, 190, 8, 2, 128), dict(lengths=i32(1, 64, 190))),
                     ((2, 1, 3000, 8, 2, 128), dict(causal=True)), ((2, 150, 150, 2, 2, 72), dict(causal=True)), ((1, 200, 256, 4, 1, 128), dict(softcap=5.0)),
                     ((2, 700, 700, 2, 1, 64), dict(documents=_docs(2, 700, 6, 3, pad=50), causal=True)), ((1, 600, 600, 2, 2, 32), dict())):
        q, k, v, _ = (t.to(dev) for t in _inputs(*size, dtype, 101))
        kw = _to(dev, kw)
        plain = attention.attention(q, k, v, return_lse=True, **kw)
        with torch.no_grad():
            quiet = attention.attention(*(t.detach().requires_grad_() for t in (q, k, v)), return_lse=True, **kw)
        recorded = attention.attention(*(t.detach().requires_grad_() for t in (q, k, v)), return_lse=True, **kw)
        assert recorded[0].requires_grad and not quiet[0].requires_grad
        for a, c, e in zip(plain, quiet, recorded):
            assert torch.equal(a, c) and torch.equal(a, e), size


def test_attention_document_that_begins_at_the_end_of_64_tiles(dev):
    """A long document whose first tiles are the last of the 64 ranges that are looked at together, and one that ends right behind them."""
    n = 5200
    ids = torch.zeros(1, n, dtype=torch.int32)
    ids[0, 4000:] = 1
    ids[0, 4200:4220] = 2
    q, k, v, do = _inputs(1, n, n, 1, 1, 16, F16, 102)
    _check(dev, q, k, v, do, documents=ids)
    ids[0, 4150:] = -1
    _check(dev, q, k, v, do, documents=ids, causal=True)


@pytest.mark.parametrize('dtype', [F16, BF16])
def test_attention_of_few_queries_is_rounded_once(dev, dtype):
    """Few queries over a cache: the weights keep what their rounding left over, so results are off by their own rounding and second-order terms only."""
    from next3d_amd.torch_utils.ops import attention
    for size, kw in (((2, 1, 3000, 8, 2, 128), dict()), ((1, 5, 900, 4, 1, 64), dict(causal=True)), ((2, 1, 70, 2, 2, 80), dict())):
        q, k, v, _ = _inputs(*size, dtype, 103)
        out = attention.attention(q.to(dev), k.to(dev), v.to(dev), **kw).cpu().double()
        vals, tols = R.attention(q, k, v, **kw)
        mean = R.attention(q, k, v.abs(), **kw)[0]['out']                       # sum of weight |v|
        exact, u = vals['out'], R.HALF[dtype]
        first = u * (mean + exact.abs())                                        # the two roundings that the bound counts for every call ...
        inner = tols['out'] - first + 2 * u * u * mean                          # ... here the rounding of a left-over, and what is float32
        own = (exact.to(dtype).double() - exact).abs()                          # the exact result's own rounding; the nearest of exact + e is within own + 2 e
        assert bool(((out - exact).abs() <= own + 2 * inner).all()), size


def _gradients64(q, k, v, do, see):
    """dq, dk [L, D] of one head in float64, and the expected squared error of each row from rounding every dscore to float16 (half a step, 2^-11 of it at
    most, is uniform: a third of the square) and the result once."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    scale = q.shape[1] ** -0.5
    p = torch.softmax((q @ k.t() * scale).masked_fill(~see, float('-inf')), 1)
    dp = do @ v.t()
    ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
    dq, dk = ds @ k, ds.t() @ q
    third = 2.0 ** -22 / 3
    row = lambda ds, x, g: third * (ds.square() @ x.square().sum(1) + g.square().sum(1)) + g.shape[1] * 2.0 ** -50          # (2^-25: half a step near zero)
    return dq, dk, row(ds, k, dq), row(ds.t(), q, dk)


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('causal', [False, True])
def test_attention_float16_gradients_of_different_sizes(dev, causal, d):
    """Rows whose gradients are 2^-6 .. 2^-12 of the largest, beside it and in another document, keep their digits: the errors' norms are within twice what the
    roundings of the dscores and of the results make (they are thousands of independent ones)."""
    n = 4096
    q, k, v, do = _inputs(1, n, n, 1, 1, d, F16, 111)
    sizes = torch.tensor([8.0, 2.0, -2.0, -4.0]).exp2()
    which = torch.arange(n) % 4
    ids = (torch.arange(n) >= 1800).to(torch.int32)[None]
    see = torch.ones(n, n, dtype=torch.bool)
    see = see.tril() if causal else see
    for what, size, docs in (('rows', sizes[which], None), ('documents', sizes[3 * ids[0].long()], ids)):
        g = (do.float() * size[None, :, None, None]).to(F16)
        got = _run(dev, q, k, v, g, causal=causal, documents=docs)
        seen = see if docs is None else see & (ids[0][:, None] == ids[0][None])
        dq, dk, e_dq, e_dk = _gradients64(q[0, :, 0], k[0, :, 0], v[0, :, 0], g[0, :, 0], seen)
        for s in sizes.unique():
            rows = size == s
            if not bool(rows.any()):
                continue
            pairs = [('dq', dq, e_dq)] + ([('dk', dk, e_dk)] if docs is not None else [])
            for name, want, var in pairs:
                err = float((got[name][0, :, 0].cpu().double() - want)[rows].norm())
                assert err <= 2 * float(var[rows].sum()) ** 0.5 + 1e-5 * float(want[rows].norm()), (what, name, float(s), err, float(want[rows].norm()))


def test_attention_float16_gradients_do_not_depend_on_what_is_not_seen(dev):
    """Large gradients and values of another sequence, of another document or behind the diagonal change no bit of a row's gradients."""
    n = 1500
    for d in (64, 128):
        q, k, v, do = _inputs(2, n, n, 2, 1, d, F16, 112)
        ids = (torch.arange(n) >= 700).to(torch.int32).repeat(2, 1)
        lo, hi = slice(0, 700), slice(700, n)
        for kw, spoil, keep in ((dict(), (0, slice(0, n)), (1, slice(0, n))), (dict(documents=ids), (slice(0, 2), hi), (slice(0, 2), lo)),
                                (dict(documents=ids, causal=True), (slice(0, 2), lo), (slice(0, 2), hi))):
            plain = _run(dev, q, k, v, do, **kw)
            big_v, big_do = v.clone(), do.clone()
            big_v[spoil][..., 3] = 60000.0
            big_do[spoil][..., 5] = 30000.0
            got = _run(dev, q, k, big_v, big_do, **kw)
            for name in ('out', 'dq', 'dk', 'dv'):
                assert torch.equal(got[name][keep], plain[name][keep]), (d, sorted(kw), name)
        big_v = v.clone()
        big_v[:, hi] *= 10000.0
        plain, got = _run(dev, q, k, v, do, causal=True), _run(dev, q, k, big_v, do, causal=True)
        assert all(torch.equal(got[name][:, lo], plain[name][:, lo]) for name in ('out', 'dq'))


def _classes64(q, k, v, do, see):
    """out, dq, dk, dv [L, D] of one head in float64 with every sum over the visible pairs only, so that infinities and NaN are those of the formula."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    scale = q.shape[1] ** -0.5
    pick = lambda keep, t: torch.where(keep, t, torch.zeros_like(t))
    t = (q[:, None] * k[None]).sum(2) * scale
    p = torch.softmax(t.masked_fill(~see, float('-inf')), 1)
    p = pick(see & see.any(1, keepdim=True), p)
    out = pick(see[..., None], p[..., None] * v[None]).sum(1)
    dp = (do[:, None] * v[None]).sum(2)
    ds = pick(see, p * (dp - (do * out).sum(1, keepdim=True)) * scale)
    return dict(out=out, dq=pick(see[..., None], ds[..., None] * k[None]).sum(1), dk=pick(see[..., None], ds[..., None] * q[:, None]).sum(0),
                dv=pick(see[..., None], p[..., None] * do[:, None]).sum(0))


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('d', [16, 40, 72, 128])
def test_attention_visible_and_masked_nonfinite(dev, d, dtype):
    """Infinities and NaN in one tensor, some visible and some not: out and dv are the infinity or NaN of the formula where it has one, gradients are finite
    exactly where the formula's are, and everything finite is within the bounds of the call without them."""
    n = 150
    inf, nan = float('inf'), float('nan')
    docs = torch.zeros(1, n, dtype=torch.int32)
    docs[:, 60:], docs[:, 130:] = 1, -1
    i = torch.arange(n)
    for causal in (True, False):
        see = (docs[0][:, None] == docs[0][None]) & (docs[0] >= 0)[:, None]
        if causal:
            see = see & (i[:, None] >= i[None])
        for name in ('v', 'do', 'k', 'q'):
            ts = dict(zip(('q', 'k', 'v', 'do'), _inputs(1, n, n, 1, 1, d, dtype, 121)))
            clean = {key: t.clone() for key, t in ts.items()}
            for row, channel, x in ((20, 3, inf), (33, 5, -inf), (40, 3, inf), (41, 7, inf), (45, 7, -inf), (70, 9, nan), (100, 2, inf), (135, 4, nan), (140, 3, -inf)):
                if name in ('q', 'k') and row not in (41, 100, 135, 140):
                    continue
                ts[name][0, row, 0, channel] = x
                clean[name][0, row, 0, channel] = 0
            got = _run(dev, ts['q'], ts['k'], ts['v'], ts['do'], documents=docs, causal=causal)
            want = _classes64(*(ts[key][0, :, 0] for key in ('q', 'k', 'v', 'do')), see)
            vals, tols = R.attention(clean['q'], clean['k'], clean['v'], clean['do'], documents=docs, causal=causal)
            for key, w in want.items():
                g, what = got[key][0, :, 0].cpu(), (causal, name, key)
                finite = torch.isfinite(w)
                assert torch.equal(torch.isfinite(g), finite), what
                if (name, key) in (('v', 'out'), ('do', 'dv')):
                    assert torch.equal(g.isnan(), w.isnan()) and torch.equal(g[g.isinf()].double(), w[w.isinf()]), what
                keep = finite
                if name == 'k':                                             # (a score of -inf takes its key out of a row, which the call without it keeps)
                    rows = see[:, [41, 100]].any(1)
                    keep = finite & ~(rows if key in ('out', 'dq') else see[rows].any(0))[:, None]
                R.assert_within(g[keep], vals[key][0, :, 0][keep], tols[key][0, :, 0][keep], str(what))


@pytest.mark.parametrize('lq', [1, 6])
def test_attention_visible_nonfinite_in_a_cache(dev, lq):
    """Few queries over a cache: the infinities of the keys in use, beside NaN in keys of another document."""
    n, d = 700, 64
    q, k, v, _ = _inputs(1, lq, n, 1, 1, d, F16, 122)
    kd, qd = (torch.arange(n) % 3 == 0).to(torch.int32)[None], torch.ones(1, lq, dtype=torch.int32)
    clean = v.clone()
    for row, channel, x in ((3, 1, float('inf')), (300, 2, -float('inf')), (6, 5, float('inf')), (333, 5, -float('inf')), (699, 9, float('nan')), (4, 1, float('nan')), (5, 30, float('inf'))):
        v[0, row, 0, channel], clean[0, row, 0, channel] = x, 0
    from next3d_amd.torch_utils.ops import attention
    out = attention.attention(q.to(dev), k.to(dev), v.to(dev), documents=qd.to(dev), key_documents=kd.to(dev)).cpu()[0, :, 0]
    vals, tols = R.attention(q, k, clean, documents=qd, key_documents=kd)
    for channel, x in ((1, float('inf')), (2, -float('inf'))):
        assert bool((out[:, channel] == x).all())
    assert bool(out[:, [5, 9]].isnan().all())
    rest = [c for c in range(d) if c not in (1, 2, 5, 9)]
    R.assert_within(out[:, rest], vals['out'][0, :, 0][:, rest], tols['out'][0, :, 0][:, rest])


@pytest.mark.parametrize('d', [64, 128])
def test_attention_overflowed_step_takes_a_few_times_as_long(dev, d):
    """One infinity in the gradient, as a loss scale too large makes it, or a row of NaN: the call repeats its sums; it does not walk them key by key."""
    q, k, v, do = (t.to(dev) for t in _inputs(1, 4096, 4096, 4, 2, d, F16, 123))

    def time(q, k, v, do):
        best = float('inf')
        for _ in range(4):
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            torch.autograd.grad(attention.attention(*leaves, causal=True), leaves, do)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end))
        return best

    from next3d_amd.torch_utils.ops import attention
    usual = time(q, k, v, do)
    spoiled = do.clone()
    spoiled[0, 4000, 1, 3] = float('inf')
    late = v.clone()
    late[0, 10] = float('nan')
    for which, t in (('do', time(q, k, v, spoiled)), ('v', time(q, k, late, do))):
        assert t < 40 * usual, (which, usual, t)


def test_attention_prefix_below_zero(dev):
    """A prefix of less than nothing is none, down to the lowest number."""
    q, k, v, do = _inputs(4, 90, 90, 2, 1, 64, BF16, 131)
    prefix = torch.tensor([-2 ** 31, -2 ** 31 + 1, -1, 2 ** 31 - 1], dtype=torch.int32)
    _check(dev, q, k, v, do, causal=True, prefix=prefix)
    _check(dev, q[:, :1], k, v, causal=True, prefix=prefix, lengths=torch.tensor([90, 3, 60, 90], dtype=torch.int32))


def test_attention_repeated_sums_in_graphs_and_side_by_side(dev):
    """Calls that take their sums again — NaN in padding, an infinity in the gradient, a NaN key — captured, replayed, and in flight on several streams at once."""
    from next3d_amd.torch_utils.ops import attention
    work = []
    for size, dtype, kw in (((2, 300, 300, 4, 2, 128), F16, dict(causal=True)), ((1, 500, 500, 2, 2, 64), BF16, dict(documents=_docs(1, 500, 3, 5, pad=90))),
                            ((1, 1700, 1700, 1, 1, 64), F16, dict(causal=True)), ((3, 2, 900, 8, 2, 128), F16, dict(lengths=torch.tensor([900, 0, 444], dtype=torch.int32)))):
        q, k, v, do = _inputs(*size, dtype, 141)
        do[0, size[1] // 2, 0, 3] = float('inf')
        v[0, 40, 0] = float('nan')
        if 'documents' in kw:
            for t in (q, k, v, do):
                t[kw['documents'] < 0] = float('nan')
        work.append(([t.to(dev) for t in (q, k, v, do)], _to(dev, kw)))

    def step(ts, kw):
        leaves = [t.detach().requires_grad_() for t in ts[:3]]
        out = attention.attention(*leaves, **kw)
        return [out.detach(), *torch.autograd.grad(out, leaves, ts[3])]

    same = lambda x, y: all(torch.equal(a.nan_to_num(7.0, 8.0, 9.0), c.nan_to_num(7.0, 8.0, 9.0)) and torch.equal(a.isnan(), c.isnan()) for a, c in zip(x, y))
    alone = [step(*w) for w in work]
    assert all(bool(x[0].isnan().any()) and bool(torch.isfinite(x[0]).any()) for x in alone)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(3):
        together = []
        for s, w in zip(streams, work):
            with torch.cuda.stream(s):
                together.append(step(*w))
        torch.cuda.synchronize()
        assert all(same(x, y) for x, y in zip(alone, together))
    graphs = []
    for w in work:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*w)
        graphs.append((g, out))
    for _ in range(3):
        for s, (g, _) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        again = [step(*w) for w in work]
        torch.cuda.synchronize()
        assert all(same(x, y) for x, y in zip(alone, again))
        assert all(same(x, out) for x, (_, out) in zip(alone, graphs))


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('d', [32, 64, 72, 96, 128])
def test_attention_short_walks_are_rounded_once(dev, d, dtype):
    """Up to four tiles: weights and dscores keep what their rounding left over, forward and backward, with documents and without, so the errors' norms are those
    of rounding the exact results once; what is left (float32 sums, roundings of left-overs) is below a tenth of that."""
    slopes = torch.tensor([0.1, 0.02])
    for n, kw in ((60, dict(causal=True)), (190, dict(documents=_docs(1, 190, 3, 151, pad=11))), (255, dict(causal=True, slopes=slopes)),
                  (240, dict(documents=_docs(1, 240, 2, 152), causal=True, softcap=8.0)), (19, dict(softcap=5.0))):
        q, k, v, do = _inputs(1, n, n, 2, 1, d, dtype, 153)
        got = _run(dev, q, k, v, do, **kw)
        vals, _ = R.attention(q, k, v, do, **kw)
        for name in ('out', 'dq', 'dk', 'dv'):
            exact = vals[name]
            err, once = float((got[name].cpu().double() - exact).norm()), float((exact.to(dtype).double() - exact).norm())
            assert err <= 1.1 * once, (n, sorted(kw), name, err / once)
