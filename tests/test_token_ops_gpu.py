"""-m gpu tests of the token operators layer_norm and rotary against their definitions in float64 (tests/_token_ref.py, bounds derived there)."""
import pytest
import torch

import _token_ref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _randn(shape, seed, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype)


# ---------------------------------------------------------------------------------------------------------------------------- layer norm
LN_SIZES = [(1, 1), (3, 2), (7, 31), (300, 32), (64, 33), (9, 64), (65, 100), (4, 255), (28, 512), (130, 1001), (33, 2048), (5, 4096), (3, 5000), (2, 8191),
            (2, 16384), (3, 20001), (70, 16392)]


def _ln_case(dev, rows, c, dtype, affine, wdtype, seed=0, shift=0.3):
    from next3d_amd.torch_utils.ops import layer_norm
    x, dy = _randn((rows, c), seed, dtype, 1.7, shift), _randn((rows, c), seed + 1, dtype)
    w = _randn((c,), seed + 2, wdtype, 0.2, 1.0) if 'w' in affine else None
    b = _randn((c,), seed + 3, wdtype, 0.2) if 'b' in affine else None
    leaves = [None if t is None else t.to(dev).requires_grad_() for t in (x, w, b)]
    y = layer_norm.layer_norm(*leaves, eps=1e-5)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(dev))
    vals, tols = R.layer_norm(x, w, b, 1e-5, dy)
    got = dict(zip([n for n, t in zip(('dx', 'dw', 'db'), leaves) if t is not None], grads), y=y)
    assert got['dx'].dtype == dtype and y.dtype == dtype
    for name, t in got.items():
        R.assert_within(t, vals[name], tols[name], f'{name} {rows}x{c} {dtype} {affine}')
    with torch.no_grad():                                                   # the path without statistics gives the same bits
        assert torch.equal(layer_norm.layer_norm(*leaves, eps=1e-5), y)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,c', LN_SIZES)
def test_layer_norm(dev, rows, c, dtype):
    _ln_case(dev, rows, c, dtype, 'wb', F32)


@pytest.mark.parametrize('affine', ['', 'w', 'b', 'wb'])
@pytest.mark.parametrize('dtype,wdtype', [(F16, F16), (BF16, BF16), (BF16, F32), (F32, F32)])
def test_layer_norm_affine_forms(dev, dtype, wdtype, affine):
    for rows, c in ((50, 70), (3, 700), (5, 17000)):
        _ln_case(dev, rows, c, dtype, affine, wdtype)


def test_layer_norm_many_rows(dev):
    """More rows than workgroups: every thread visits several."""
    for rows, c, dtype in ((50000, 32, F16), (40001, 24, F32), (3000, 1030, BF16)):
        _ln_case(dev, rows, c, dtype, 'wb', F32)


def test_layer_norm_large_offset(dev):
    """Rows far from zero: the variance is taken from centred values."""
    _ln_case(dev, 40, 900, F32, 'wb', F32, shift=1000.0)


def test_layer_norm_constant_rows_and_eps(dev):
    from next3d_amd.torch_utils.ops import layer_norm
    x = torch.full((4, 96), 2.5, device=dev)
    assert torch.equal(layer_norm.layer_norm(x), torch.zeros_like(x))
    b = torch.arange(96.0, device=dev)
    assert torch.equal(layer_norm.layer_norm(x, None, b), b.expand(4, 96))


def test_layer_norm_nonfinite_rows_stay_alone(dev):
    from next3d_amd.torch_utils.ops import layer_norm
    for c in (32, 512, 3000):
        x = _randn((9, c), 5)
        clean = layer_norm.layer_norm(x.to(dev)).cpu()
        x[2, 1], x[5, 0] = float('nan'), float('inf')
        y = layer_norm.layer_norm(x.to(dev)).cpu()
        assert torch.isnan(y[2]).all() and torch.isnan(y[5]).all()
        keep = [0, 1, 3, 4, 6, 7, 8]
        assert torch.equal(y[keep], clean[keep])


def test_layer_norm_strides_and_shapes(dev):
    from next3d_amd.torch_utils.ops import layer_norm
    big = _randn((6, 10, 80), 3).to(dev)
    for view in (big[:, :, 5:69], big[::2], big[:, 3], big.transpose(0, 1), big.transpose(1, 2), big[0, 0], big[:, :, 1:2], big[:0], big[0:1, 0:1].expand(4, 5, 80)):
        x = view.detach().requires_grad_()
        y = layer_norm.layer_norm(x)
        dense = view.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
        want = layer_norm.layer_norm(dense)
        assert y.shape == view.shape and torch.equal(y, want)
        g = torch.ones((), device=dev).expand(y.shape)                      # what sum().backward() hands on: stride 0
        assert torch.equal(torch.autograd.grad(y, x, g)[0], torch.autograd.grad(want, dense, g.contiguous())[0])
    w = torch.ones(80, device=dev, requires_grad=True)
    dw, = torch.autograd.grad(layer_norm.layer_norm(big[:0], w), w, big[:0])
    assert torch.equal(dw, torch.zeros(80, device=dev))


def test_layer_norm_partial_gradients_and_differences(dev):
    """Only what is asked for is computed, with the same bits; and the gradients against differences of the float64 definition."""
    from next3d_amd.torch_utils.ops import layer_norm
    x, dy, w, b = _randn((21, 130), 1), _randn((21, 130), 2), _randn((130,), 3, F32, 0.3, 1.0), _randn((130,), 4)
    dx, dw, db = [t.cpu() for t in _grads(layer_norm.layer_norm, (x, w, b), dy, dev, (0, 1, 2))]
    for which, want in ((0, dx), (1, dw), (2, db)):
        assert torch.equal(_grads(layer_norm.layer_norm, (x, w, b), dy, dev, (which,))[0].cpu(), want)
    h = 1e-5
    for i, grad in enumerate((dx, dw, db)):
        step = _randn((x, w, b)[i].shape, 9).double()
        args = [t.double() for t in (x, w, b)]

        def f(sign):
            moved = [a + sign * h * step if j == i else a for j, a in enumerate(args)]
            return float((R.layer_norm(*moved, 1e-5)[0]['y'] * dy.double()).sum())

        numeric, analytic = (f(1) - f(-1)) / (2 * h), float((grad.double() * step).sum())
        # truncation h^2 f'''/6 ~ 1e-9, float64 cancellation 1e-11, float32 gradients: 2^-24 * 100 a term at most
        assert abs(numeric - analytic) <= 2.0 ** -17 * float((grad.double() * step).abs().sum()) + 1e-6


def _grads(fn, tensors, dy, dev, which):
    leaves = [t.to(dev).requires_grad_(i in which) for i, t in enumerate(tensors)]
    return torch.autograd.grad(fn(*leaves), [leaves[i] for i in which], dy.to(dev))


def test_layer_norm_reproducible_on_another_stream_and_in_graphs(dev):
    from next3d_amd.torch_utils.ops import layer_norm
    x, w, b, dy = (t.to(dev) for t in (_randn((5000, 96), 1, F16), _randn((96,), 2), _randn((96,), 3), _randn((5000, 96), 4, F16)))

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = layer_norm.layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, again))
    graphs = []
    for _ in range(2):                                                      # two graphs that replay side by side share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for round_ in range(3):
        x.copy_(_randn((5000, 96), 10 + round_, F16))
        want = [t.clone() for t in step()]
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(want, out))


# -------------------------------------------------------------------------------------------------------------------------------- rotary
ROT = [  # B, L, Hq, Hk, D, sections
    (1, 1, 1, 1, 2, (2,)), (2, 3, 4, 1, 8, (2, 6)), (1, 7, 3, 3, 64, (16, 24, 24)), (2, 33, 2, 0, 96, (16, 24, 24)), (1, 5, 2, 2, 70, (6, 14, 22)),
    (3, 50, 4, 2, 128, (32, 48, 48)), (1, 9, 1, 1, 40, (4, 8, 4, 12)), (8, 1, 32, 8, 128, (32, 48, 48)), (1, 3000, 1, 1, 32, (16, 16)), (1, 2, 2, 1, 512, (200, 0, 312)),
    (1, 4, 1, 1, 1000, (600, 400))]


@pytest.mark.parametrize('pairing', ['interleaved', 'half'])
@pytest.mark.parametrize('ladder', ['axis', 'shared'])
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_rotary(dev, dtype, pairing, ladder):
    from next3d_amd.torch_utils.ops import rotary
    for n, (b, l, hq, hk, d, sections) in enumerate(ROT):
        q, dq = _randn((b, l, hq, d), n, dtype), _randn((b, l, hq, d), n + 50, dtype)
        k, dk = (_randn((b, l, hk, d), n + 100, dtype), _randn((b, l, hk, d), n + 150, dtype)) if hk else (None, None)
        pos = torch.randint(-50, 5000, (b, l, len(sections)) if n % 2 else (l, len(sections)), generator=torch.Generator().manual_seed(n))
        pos = pos.to((torch.int32, torch.int64, torch.float32)[n % 3])
        lq = q.to(dev).requires_grad_()
        lk = k.to(dev).requires_grad_() if hk else None
        kw = dict(base=10000.0 if n % 2 else 150.0, pairing=pairing, ladder=ladder)
        out = rotary.rotary(lq, pos.to(dev), sections, k=lk, **kw)
        pairs = [('q', q, out[0] if hk else out, dq, lq)] + ([('k', k, out[1], dk, lk)] if hk else [])
        grads = torch.autograd.grad([p[2] for p in pairs], [p[4] for p in pairs], [p[3].to(dev) for p in pairs])
        for (name, x, y, dy, _), dx in zip(pairs, grads):
            R.assert_within(y, *R.rotary(x, pos, sections, inverse=False, **kw), f'{name} case {n}')
            R.assert_within(dx, *R.rotary(dy, pos, sections, inverse=True, **kw), f'd{name} case {n}')


def test_rotary_far_positions(dev):
    """Angles of far positions are taken in 64 bits."""
    from next3d_amd.torch_utils.ops import rotary
    q = _randn((1, 4, 2, 64), 1)
    for pos in (torch.tensor([[2 ** 31 - 1], [10 ** 9], [2 ** 24 + 1], [-(2 ** 31)]]), torch.tensor([[1e6 + 0.5], [3.7e7], [0.125], [-1e-3]], dtype=F32)):
        y = rotary.rotary(q.to(dev), pos.to(dev), (64,))
        R.assert_within(y, *R.rotary(q, pos, (64,), 10000.0, 'interleaved', 'axis'))


def test_rotary_strides(dev):
    """Views of one projection (q and k interleaved with others), transposed heads, expanded batches and gradients with stride 0."""
    from next3d_amd.torch_utils.ops import rotary
    fused = _randn((2, 11, 3 * 4, 50), 2, F16).to(dev)
    pos = torch.arange(22, dtype=torch.int32, device=dev).reshape(11, 2)
    odd = torch.randint(0, 99, (2, 11, 4), device=dev)[:, :, 1:3]
    heads_first = fused.transpose(1, 2).contiguous().transpose(1, 2)
    for q, k in ((fused[:, :, :4], fused[:, :, 4:8]), (heads_first[:, :, :4], heads_first[:, :, 4:8]), (fused[:, :, :4, 2:34], fused[:, :, 4:8, 3:35]),
                 (fused[:1].expand(3, 11, 12, 50), fused[:1, :, ::3].expand(3, 11, 4, 50)), (fused[..., ::2][:, :, :4], fused[..., 1::2][:, :, :4])):
        for p in (pos, odd if q.shape[0] == 2 else pos):
            got = rotary.rotary(q, p, (16, 8), k=k)
            want = rotary.rotary(q.contiguous(), p.contiguous(), (16, 8), k=k.contiguous())
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = fused[:, :, :4].detach().requires_grad_()
    y, _ = rotary.rotary(q, pos, (16, 8), k=fused[:, :, 4:8])
    one = torch.ones((), device=dev, dtype=F16)
    assert torch.equal(torch.autograd.grad(y, q, one.expand(y.shape), retain_graph=True)[0], torch.autograd.grad(y, q, one.expand(y.shape).contiguous())[0])
    assert rotary.rotary(fused[:0], pos, (16, 8)).shape == (0, 11, 12, 50)
    assert rotary.rotary(fused[:, :0], pos[:0], (16, 8)).shape == (2, 0, 12, 50)


def test_rotary_only_one_gradient_and_differences(dev):
    from next3d_amd.torch_utils.ops import rotary
    q, k, pos = _randn((1, 6, 2, 24), 1), _randn((1, 6, 1, 24), 2), torch.arange(12).reshape(6, 2)
    lq, lk = q.to(dev).requires_grad_(), k.to(dev).requires_grad_()
    yq, yk = rotary.rotary(lq, pos.to(dev), (8, 12), k=lk, pairing='half')
    dy = _randn(k.shape, 3)
    gk, = torch.autograd.grad(yk, lk, dy.to(dev))                            # nothing flows into q
    step, h = _randn(k.shape, 4).double(), 1e-3
    f = [float((R.rotary(k.double() + s * h * step, pos, (8, 12), 10000.0, 'half', 'axis')[0] * dy.double()).sum()) for s in (1, -1)]
    analytic = (gk.cpu().double() * step)
    assert abs((f[0] - f[1]) / (2 * h) - float(analytic.sum())) <= 2.0 ** -20 * float(analytic.abs().sum()) + 1e-9      # linear: no truncation



def test_token_ops_beyond_32_bits(dev):
    """Tensors of more than 2^31 elements: the first, a middle and the last rows."""
    from next3d_amd.torch_utils.ops import layer_norm, rotary
    rows, c = 2 ** 21 + 5, 1030
    x, dy = (torch.empty((rows, c), dtype=BF16, device=dev).normal_(0.0, 1.0) for _ in range(2))
    w = _randn((c,), 5)
    leaf = x.requires_grad_()
    y = layer_norm.layer_norm(leaf, w.to(dev))
    dx, = torch.autograd.grad(y, leaf, dy)
    some = [0, 1, rows // 2 + 1, rows - 2, rows - 1]
    vals, tols = R.layer_norm(x.detach()[some].cpu(), w, None, 1e-5, dy[some].cpu())
    R.assert_within(y[some], vals['y'], tols['y'], 'y')
    R.assert_within(dx[some], vals['dx'], tols['dx'], 'dx')
    del x, dy, leaf, y, dx
    n = 2 ** 18 + 3
    q = torch.empty((1, n, 64, 128), dtype=F16, device=dev).normal_(0.0, 1.0)
    pos = torch.randint(0, 4096, (n, 3), generator=torch.Generator().manual_seed(1))
    y = rotary.rotary(q, pos.to(dev), (32, 48, 48))
    some = [0, n // 2, n - 1]
    R.assert_within(y[:, some], *R.rotary(q[:, some].cpu(), pos[some], (32, 48, 48), 10000.0, 'interleaved', 'axis'), 'rotary')
    del q, y
    torch.cuda.empty_cache()


def test_token_ops_lazily_negated_gradients(dev):
    from next3d_amd.torch_utils.ops import layer_norm, rotary
    x, pos = _randn((1, 5, 2, 16), 6).to(dev).requires_grad_(), torch.arange(5, device=dev)[:, None]
    dy = _randn((1, 5, 2, 16), 7).to(dev)
    for fn in (layer_norm.layer_norm, lambda t: rotary.rotary(t, pos, (16,))):
        a, = torch.autograd.grad(fn(x), x, -dy)
        b, = torch.autograd.grad(fn(x), x, torch._neg_view(dy))
        assert torch.equal(a, b)


def test_token_ops_refuse_second_derivatives(dev):
    """Under create_graph the gradients come out as ever, and differentiating them again raises."""
    from next3d_amd.torch_utils.ops import attention, layer_norm, rotary
    x = _randn((3, 64), 1).to(dev).requires_grad_()
    q, k, v = (_randn((1, 5, 2, 16), s, F16).to(dev).requires_grad_() for s in (2, 3, 4))
    pos = torch.arange(5, device=dev).reshape(5, 1)
    for leaves, f in (((x,), lambda: layer_norm.layer_norm(x)), ((q,), lambda: rotary.rotary(q, pos, (16,))), ((q, k, v), lambda: attention.attention(q, k, v))):
        plain = torch.autograd.grad(f().sum(), leaves)
        graph = torch.autograd.grad(f().sum(), leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, graph))
        with pytest.raises(RuntimeError, match='differentiable once'):
            graph[0].float().square().sum().backward()


def test_token_ops_refuse_what_cannot_see_into_them(dev):
    """Forward-mode derivatives, tracers and functional transforms raise through the public functions; none returns a result without a derivative."""
    import torch.autograd.forward_ad as fwd
    from next3d_amd.torch_utils.ops import attention, layer_norm, rotary
    q = torch.ones(1, 3, 2, 8, dtype=torch.float16, device=dev)
    pos = torch.zeros(3, 1, device=dev)
    for call, x in ((layer_norm.layer_norm, torch.ones(3, 8, device=dev)), (lambda t: rotary.rotary(t, pos, (8,)), q), (lambda t: attention.attention(t, q, q), q)):
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match='forward-mode'):
                call(fwd.make_dual(x, x))
            with torch.no_grad(), pytest.raises(RuntimeError, match='forward-mode'):
                call(fwd.make_dual(x, x))
        with pytest.raises(RuntimeError, match='traced'):
            torch.jit.trace(call, (x,))
        for transform in (lambda: torch.vmap(call)(x[None]), lambda: torch.func.jvp(call, (x,), (x,)), lambda: torch.func.grad(lambda t: call(t).sum())(x)):
            with pytest.raises(RuntimeError):
                transform()
        assert call(x).shape == x.shape


def test_layer_norm_gradients_of_very_long_rows(dev):
    """More channels than a launch of the column sums has threads for."""
    from next3d_amd.torch_utils.ops import layer_norm
    c = (1 << 26) + 5
    g = torch.Generator(device=dev).manual_seed(7)
    x, dy = (torch.randn((2, c), generator=g, device=dev).half() for _ in range(2))
    w, b = torch.ones(c, device=dev).requires_grad_(), torch.zeros(c, device=dev).requires_grad_()
    dw, db = torch.autograd.grad(layer_norm.layer_norm(x, w, b), (w, b), dy)
    xd, dyd = x.double(), dy.double()
    xc = xd - xd.mean(1, keepdim=True)
    xh = xc / (xc.square().mean(1, keepdim=True) + 1e-5).sqrt()
    chain = (c / 1024 + 80) * R.U32                                        # a thread adds c / 1024 terms one after the other; the mean's terms are |x| ~ 1 on average
    assert bool(((db.double() - dyd.sum(0)).abs() <= 4 * R.U32 * dyd.abs().sum(0)).all())
    assert bool(((dw.double() - (dyd * xh).sum(0)).abs() <= (dyd.abs() * (1 + xh.abs()) * 2 * chain).sum(0)).all())
    del x, dy, xd, dyd, xc, xh, dw, db, w, b
    torch.cuda.empty_cache()
