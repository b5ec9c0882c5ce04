"""The token operators (layer_norm, rotary, attention) from their definitions in float64 on the CPU, and the error bounds of the kernels' arithmetic.

U32 is half a step of float32 (the rounding of one operation); HALF[t] half a step of the stored type.  A bound is the sum over the roundings that the
kernels make, each weighed by what it multiplies."""
import torch

U32 = 2.0 ** -24
HALF = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float64: 0.0, torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}          # absolute: half a step of the smallest numbers


def assert_within(got, want, tol, what=''):
    got, want, tol = got.detach().cpu().double(), want.double(), tol.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (f'{what}: {int(bad.sum())} of {bad.numel()} beyond the bound; worst error '
                                 f'{float((got - want).abs().nan_to_num(float("inf")).max()):.3e}, largest ratio '
                                 f'{float(((got - want).abs() / tol.clamp_min(1e-300)).nan_to_num(float("inf")).max()):.2f}')


# ---------------------------------------------------------------------------------------------------------------------------- layer norm
def layer_norm(x, weight, bias, eps, dy=None):
    """(values, bounds) of y [, dx, dw, db] for x [rows, C]; weight / bias may be None.  Bounds for a sum of n terms: the kernels add at most 16 terms a
    lane one after the other (64 in rows beyond 16384 channels), then by halves — at most 64 roundings of partial sums for any tested row — and
    rows per workgroup + 64 for the column sums."""
    dt = x.dtype
    x, w = x.double(), torch.ones(x.shape[1], dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if bias is None else bias.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    y = xh * w + b
    e_xh = U32 * (64 * x.abs().amax(1, keepdim=True) * rstd + 72 * xh.abs())                    # mean's sum; variance's sum, root, products
    # (the mean's error shifts every centred value alike: it reaches the variance in second order only)
    vals = dict(y=y)
    tols = dict(y=HALF[dt] * y.abs() + w.abs() * e_xh + 4 * U32 * (y.abs() + (xh * w).abs() + b.abs()) + TINY[dt])
    if dy is not None:
        dy = dy.double()
        g = dy * w
        s1, s2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        dx = rstd * (g - s1 - xh * s2)
        e_s1 = 65 * U32 * g.abs().mean(1, keepdim=True)
        e_s2 = (g.abs() * e_xh).mean(1, keepdim=True) + 66 * U32 * (g * xh).abs().mean(1, keepdim=True)
        size = g.abs() + s1.abs() + (xh * s2).abs()
        e_dx = rstd * (e_s1 + xh.abs() * e_s2 + e_xh * s2.abs() + 4 * U32 * size) + 40 * U32 * rstd * size
        rows = x.shape[0] / min(x.shape[0], 64) + 80                                            # longest chain of column additions
        dw, db = (dy * xh).sum(0), dy.sum(0)
        wdt = next((t.dtype for t in (weight, bias) if t is not None), torch.float32)
        vals.update(dx=dx, dw=dw, db=db)
        tols.update(dx=HALF[dt] * dx.abs() + e_dx + TINY[dt],
                    dw=HALF[wdt] * dw.abs() + rows * U32 * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0) + TINY[wdt],
                    db=HALF[wdt] * db.abs() + rows * U32 * dy.abs().sum(0) + TINY[wdt])
    return vals, tols


# -------------------------------------------------------------------------------------------------------------------------------- rotary
def rotary(x, positions, sections, base, pairing, ladder, inverse=False):
    """(values, bounds) of the turned x [B, L, H, D]; positions [L, A] or [B, L, A]."""
    dt, x = x.dtype, x.double()
    y, tol = x.clone(), torch.zeros_like(x)
    pos = positions.double() if positions.ndim == 3 else positions.double()[None]
    total, offset, p = sum(sections) // 2, 0, 0
    for a, s in enumerate(sections):
        for i in range(s // 2):
            freq = float(base) ** -(2 * i / s if ladder == 'axis' else p / total)
            angle = pos[:, :, None, a] * freq
            cos, sin = torch.cos(angle), torch.sin(angle) * (-1 if inverse else 1)
            lo, hi = (2 * p, 2 * p + 1) if pairing == 'interleaved' else (offset + i, offset + i + s // 2) if ladder == 'axis' else (p, p + total)
            y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
            y[..., hi] = x[..., lo] * sin + x[..., hi] * cos
            size = x[..., lo].abs() + x[..., hi].abs()
            # float32 cosine and sine (argument rounding, function, storage: 4 half steps of 1), two products and a sum; 64-bit angle of the position
            tol[..., lo] = tol[..., hi] = size * (8 * U32 + 2.0 ** -50 * angle.abs())
            p += 1
        offset += s
    rest = torch.zeros(x.shape[-1], dtype=torch.bool)
    rest[2 * total:] = True
    tol = tol + HALF[dt] * y.abs() + TINY[dt]
    tol[..., rest] = 0                                                                          # channels that pass through: the same bits
    return y, tol


# ----------------------------------------------------------------------------------------------------------------------------- attention
def attention(q, k, v, do=None, scale=None, causal=False, prefix=None, documents=None, key_documents=None, lengths=None, softcap=0.0, slopes=None):
    """(values, bounds) of out, lse [, dq, dk, dv].  Masked places are left out of every sum (a NaN there reaches nothing).

    Bounds.  A score is a float32 sum of D exact products (D + 2 roundings), a multiplication into base 2 and, with a cap, 1 - 2 / (1 + e^2x), which is off
    by 2^-22 of the cap; the weight of a score off by e is off by e relatively, plus 2^-21 for the exponential.  Weights, dscores and results are each
    rounded once to the inputs' type: HALF of themselves, or half of its smallest step.  What falls below 2^-126, the smallest normal number of float32
    and bfloat16, may become zero: a weight (exp2's result; then its 16-bit form) is off by 2 * 2^-126 more, a dscore by as much times |dP| + |delta|."""
    flush = 2.0 ** -125
    dt = q.dtype
    u, n_q, n_k, d = HALF[dt], q.shape[1], k.shape[1], q.shape[3]
    group, scale = q.shape[2] // k.shape[2], d ** -0.5 if scale is None else scale
    step = 2.0 ** -25 if dt == torch.float16 else 0.0                                       # half the smallest step of float16 (bfloat16: 2^-134)
    if documents is not None and key_documents is None:
        key_documents = documents
    heads = lambda t: t.double().transpose(1, 2)                                            # [B, H, L, D]
    spread = lambda t: heads(t).repeat_interleave(group, dim=1)
    q_, k_, v_ = heads(q), spread(k), spread(v)
    b = q.shape[0]
    n = torch.full((b,), n_k) if lengths is None else lengths.long().clamp(0, n_k)
    pos = torch.arange(n_q)[None, :, None] + n[:, None, None] - n_q
    j = torch.arange(n_k)[None, None, :]
    see = (j < n[:, None, None]).expand(b, n_q, n_k).clone()
    if causal:
        see &= (j <= pos) | (j < (prefix.long() if prefix is not None else torch.zeros(b).long())[:, None, None])
    if documents is not None:
        see &= (documents[:, :, None] == key_documents[:, None, :]) & (documents[:, :, None] >= 0)
    see = see[:, None].expand(b, q.shape[2], n_q, n_k)
    clean = lambda t, keep: torch.where(keep, t, torch.zeros_like(t))
    any_q, any_k = see.any(3)[..., None], see.any(2)[..., None]
    q_, k_, v_ = clean(q_, any_q), clean(k_, any_k), clean(v_, any_k)

    raw = q_ @ k_.transpose(2, 3)
    e_s = abs(scale) * (d + 4) * U32 * (q_.abs() @ k_.abs().transpose(2, 3))
    t = raw * scale
    th = torch.tanh(t / softcap) if softcap else torch.zeros_like(t)
    if softcap:
        t = softcap * th
        e_s = e_s + 2.0 ** -21 * softcap
    if slopes is not None:
        bias = slopes.double()[None, :, None, None] * (pos - j).abs()[:, None]
        t = t - bias
        e_s = e_s + 4 * U32 * bias.abs()
    e_s = e_s + 8 * U32 * t.abs() + 2.0 ** -21
    low = torch.full_like(t, float('-inf'))
    t = torch.where(see, t, low)
    top = t.amax(3, keepdim=True)
    top = torch.where(top == float('-inf'), torch.zeros_like(top), top)
    w = torch.exp(t - top)
    total = w.sum(3, keepdim=True)
    p = w / torch.where(total == 0, torch.ones_like(total), total)
    lse = torch.log(total.squeeze(3)) + top.squeeze(3)
    e_p = torch.where(see, e_s, torch.zeros_like(e_s)).amax(3, keepdim=True)                # relative error of a row's weights, and of their sum
    chain = (n_k + 64) * U32
    pv = p @ v_.abs()
    o = p @ v_
    e_o = (u + 2 * e_p + chain) * pv + (step + flush) * clean(v_.abs(), any_k).sum(2, keepdim=True) * any_q + u * o.abs() + TINY[dt]
    vals = dict(out=o.transpose(1, 2), lse=lse)
    tols = dict(out=e_o.transpose(1, 2), lse=(e_p.squeeze(3) + chain + 4 * U32 * (lse.abs().nan_to_num(0.0, 0.0, 0.0) + 1)))
    if do is None:
        return vals, tols
    do_ = clean(heads(do), any_q)
    e_w = 2 * e_p + e_s + chain + 8 * U32 * lse.abs().nan_to_num(0.0, 0.0, 0.0)[..., None]  # weights again, from the stored lse
    fold = lambda t: t.reshape(b, k.shape[2], group, *t.shape[2:]).sum(2)
    dv = p.transpose(2, 3) @ do_
    e_dv = ((p * (u + e_w + (group * n_q + 64) * U32)).transpose(2, 3) @ do_.abs()) + (step * 2.0 ** -12 + flush) * do_.abs().sum(2, keepdim=True)
    delta = (do_ * o).sum(3, keepdim=True)
    dp = do_ @ v_.transpose(2, 3)
    e_oo = e_o - u * (1 - 2 * u) * o.abs()                                                  # (what out's rounding left over is kept, and rounded itself)
    e_d = (do_.abs() * e_oo).sum(3, keepdim=True) + (d + 4) * U32 * (do_.abs() @ v_.abs().transpose(2, 3) + (do_ * o).abs().sum(3, keepdim=True))
    cap = 1 - th * th
    dt_ = p * (dp - delta)
    ds = torch.where(see, dt_ * cap * scale, torch.zeros_like(dt_))
    e_ds = torch.where(see, abs(scale) * (p * (e_d + (dp - delta).abs() * (e_w + 2.0 ** -20))) + u * ds.abs() + abs(scale) * flush * (dp.abs() + delta.abs() + 1), torch.zeros_like(ds))
    if dt == torch.float16:                                                                 # ds 2^e in float16: e as the kernels choose it
        a, c = float(do_.abs().max()), float(v_.abs().max())
        if a and c:
            import math
            e = 7 - math.frexp(a)[1] - math.frexp(c)[1]
            e_ds = e_ds + torch.where(see, torch.full_like(ds, step * 2.0 ** -e * abs(scale)), torch.zeros_like(ds))
    dq, dk = ds @ k_, ds.transpose(2, 3) @ q_
    e_dq = e_ds @ k_.abs() + chain * (ds.abs() @ k_.abs())
    e_dk = e_ds.transpose(2, 3) @ q_.abs() + (group * n_q + 64) * U32 * (ds.abs().transpose(2, 3) @ q_.abs())
    out = lambda val, err: (val.transpose(1, 2), (err + u * val.abs() + TINY[dt]).transpose(1, 2))
    vals['dq'], tols['dq'] = out(dq, e_dq)
    vals['dk'], tols['dk'] = out(fold(dk), fold(e_dk))
    vals['dv'], tols['dv'] = out(fold(dv), fold(e_dv))
    return vals, tols
