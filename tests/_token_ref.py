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
