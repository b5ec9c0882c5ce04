"""Measured cases of the token operators: `layer_norm`, `rotary` and `attention` of next3d_amd.torch_utils.ops.

They are the operators of a transformer block over the tokens that this repository's generator handles — w vectors, tri-plane texels, frames of a
video — and each case runs one of them in one direction: the forward pass, or (train) the forward pass and the gradients of every input.  `run` with
`own` false is the plain form in float32 torch operations, with `own` true the call of the library.  `exact` restates each definition in float64.
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}
EPS = 1e-5
BASE = 10000.0


# ---------------------------------------------------------------------------------------------------------------------------------- cases
def _ln(name, rows, cols, dtype, train):
    return dict(name=name, op='layer_norm', rows=rows, cols=cols, dtype=dtype, train=train)


def _rope(name, batch, t, h, w, heads, kv_heads, dim, sections, dtype, pairing, ladder, train):
    """`sections` is a text such as '16+24+24': channels of the time, height and width axes."""
    return dict(name=name, op='rotary', batch=batch, t=t, h=h, w=w, heads=heads, kv_heads=kv_heads, dim=dim, sections=sections, dtype=dtype,
                pairing=pairing, ladder=ladder, train=train)


def _attn(name, batch, lq, lk, heads, kv_heads, dim, dtype, train=False, causal=False, prefix=0, docs=0, ragged=False, softcap=0.0, slopes=False):
    """prefix: keys every query sees; docs: documents packed in a row, the last 1/16 of it padding; ragged: keys per sequence differ."""
    return dict(name=name, op='attention', batch=batch, lq=lq, lk=lk, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, train=train,
                causal=causal, prefix=prefix, docs=docs, ragged=ragged, softcap=softcap, slopes=slopes)


def listed():
    return [
        # the 28 w vectors of 4 seeds, normalised between two layers of a mapping network: latency
        _ln('norm_w_vectors', 4 * 28, 512, 'f32', False),
        # every texel of the tri-planes of 4 samples (3 x 256 x 256, 32 channels): very short rows, float16
        _ln('norm_plane_texels_train', 4 * 3 * 256 * 256, 32, 'f16', True),
        # a training batch of tokens of a wide block
        _ln('norm_tokens_train', 16384, 4096, 'bf16', True),
        # odd counts of rows and channels in float32
        _ln('norm_odd_train', 5003, 1001, 'f32', True),
        # one new token of each of 8 sequences: latency
        _rope('rotary_token', 8, 1, 1, 1, 32, 8, 128, '32+48+48', 'bf16', 'half', 'shared', False),
        # two clips of 16 frames of 32 x 32 patches
        _rope('rotary_clip', 2, 16, 32, 32, 16, 16, 128, '32+48+48', 'bf16', 'half', 'axis', False),
        # odd frame sizes, channels that pass through, with the gradients
        _rope('rotary_odd_train', 3, 9, 17, 31, 12, 12, 96, '16+24+24', 'f16', 'interleaved', 'axis', True),
        # one new token of each of 16 sequences over a cache of up to 16384 tokens, ragged
        _attn('attend_token', 16, 1, 16384, 32, 8, 128, 'bf16', causal=True, ragged=True),
        # a short question to few keys: latency
        _attn('attend_few', 2, 7, 77, 8, 8, 64, 'f16', causal=True, slopes=True),
        # frames of several clips packed into one row, every clip its own document
        _attn('attend_packed', 1, 16384, 16384, 16, 16, 64, 'f16', docs=12),
        # a training step: a prefix seen by all, then causal, scores capped, shared key heads
        _attn('attend_prefix_train', 2, 4096, 4096, 16, 4, 128, 'bf16', train=True, causal=True, prefix=1000, softcap=30.0),
        # a training step at odd sizes: packed documents, causal, bias by distance
        _attn('attend_odd_train', 3, 1021, 1021, 6, 6, 72, 'f16', train=True, causal=True, docs=5, slopes=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['layer_norm', 'rotary', 'attention', 'attention'])
    if op == 'layer_norm':
        cols = _log_uniform(rng, 16, 8192)
        rows = _log_uniform(rng, 16, 2 ** 25 // cols)
        c = _ln('', rows, cols, rng.choice(['f32', 'f16', 'bf16']), rng.random() < 0.7)
    elif op == 'rotary':
        pairing, ladder = rng.choice(['interleaved', 'half']), rng.choice(['axis', 'shared'])
        parts = [2 * rng.randint(2, 24) for _ in range(3)] if rng.random() < 0.5 else rng.choice([[32, 48, 48], [16, 24, 24], [16, 56, 56]])
        rest = rng.choice([0, 0, 8, 32])
        dim = (sum(parts) + rest + 7) // 8 * 8
        heads = rng.choice([1, 4, 12, 16, 24])
        kv = heads if heads % 4 else rng.choice([heads, heads // 4])
        h, w = _log_uniform(rng, 1, 32), _log_uniform(rng, 1, 32)
        most = max(1, 2 ** 26 // (h * w * (heads + kv) * dim))                   # frames of the whole batch: 2^26 elements at most
        batch = min(most, rng.randint(1, 4))
        c = _rope('', batch, min(most // batch, _log_uniform(rng, 1, 16)), h, w, heads, kv, dim, '+'.join(str(p) for p in parts),
                  rng.choice(['f32', 'f16', 'bf16']), pairing, ladder, rng.random() < 0.5)
    elif rng.random() < 0.3:                                                     # single tokens, or a few, over a cache
        group = rng.choice([1, 2, 4, 8])
        kv = rng.choice([1, 2, 4, 8])
        c = _attn('', rng.randint(1, 16), rng.choice([1, 1, 1, 2, 5]), _log_uniform(rng, 64, 16384), group * kv, kv, rng.choice([64, 80, 128]),
                  rng.choice(['f16', 'bf16']), causal=True, ragged=rng.random() < 0.7, softcap=rng.choice([0.0, 0.0, 50.0]), slopes=rng.random() < 0.3)
    else:
        train = rng.random() < 0.6
        length = _log_uniform(rng, 17, 4096)
        group = rng.choice([1, 1, 2, 4])
        kv = rng.choice([1, 2, 4])
        causal = rng.random() < 0.6
        c = _attn('', rng.randint(1, 2), length, length, group * kv, kv, rng.choice([32, 64, 72, 96, 128]), rng.choice(['f16', 'bf16']), train=train,
                  causal=causal, prefix=rng.randint(1, length) if causal and rng.random() < 0.4 else 0,
                  docs=rng.randint(1, max(1, length // 16)) if rng.random() < 0.4 else 0, softcap=rng.choice([0.0, 0.0, 20.0]),
                  slopes=rng.random() < 0.3)
    del c['name']
    return c


# ------------------------------------------------------------------------------------------------------------------- layouts the case fixes
def _doc_ids(case, length):
    """Documents of uneven lengths, ids rising; the last 1/16 of the row belongs to none (-1)."""
    used, n = length - length // 16, case['docs']
    weights = [1 + (5 * d) % 7 for d in range(n)]
    total, ids, at = sum(weights), [], 0
    for d in range(n):
        end = used if d == n - 1 else min(used, at + used * weights[d] // total)
        ids += [d] * (end - at)
        at = end
    return ids + [-1] * (length - used)


def _lengths(case):
    """Keys in use per sequence, from about half of the cache to all of it."""
    lk = case['lk']
    return [max(case['lq'], lk - (b * 977 + b * b * 131) % (lk // 2 + 1)) for b in range(case['batch'])] if case['ragged'] else [lk] * case['batch']


def _visible_pairs(case):
    """Visible (query, key) pairs of one head, summed over the batch."""
    total = 0
    for n in _lengths(case):
        if case['docs']:
            ids = _doc_ids(case, case['lk'])
            start = {}
            for j, d in enumerate(ids):
                start.setdefault(d, j)
            count = {d: ids.count(d) for d in start}
            for i, d in enumerate(ids):
                if d >= 0:
                    total += count[d] if not case['causal'] else max(i + 1, min(case['prefix'], start[d] + count[d])) - start[d] \
                        if case['prefix'] > start[d] else i + 1 - start[d]
        elif case['causal']:
            total += sum(min(n, max(i + n - case['lq'] + 1, case['prefix'], 0)) for i in range(case['lq']))
        else:
            total += case['lq'] * n
    return total


def work(case):
    e = BYTES[case['dtype']]
    if case['op'] == 'layer_norm':
        n = case['rows'] * case['cols']
        if not case['train']:
            return {'bytes': 2 * n * e + 2 * case['cols'] * 4, 'flops': 8 * n}
        return {'bytes': 5 * n * e + 4 * case['cols'] * 4 + 8 * case['rows'] * 2, 'flops': 22 * n}
    if case['op'] == 'rotary':
        tokens = case['batch'] * case['t'] * case['h'] * case['w']
        n = tokens * (case['heads'] + case['kv_heads']) * case['dim']
        passes = 2 if case['train'] else 1
        return {'bytes': passes * (2 * n * e + tokens // case['batch'] * 12), 'flops': passes * 3 * n}
    pairs = _visible_pairs(case) * case['heads'] * case['dim']
    q = case['batch'] * case['lq'] * case['heads'] * case['dim'] * e
    kv = 2 * sum(_lengths(case)) * case['kv_heads'] * case['dim'] * e
    if not case['train']:
        return {'bytes': 2 * q + kv, 'flops': 4 * pairs}
    return {'bytes': 2 * q + kv + 4 * q + 2 * kv, 'flops': 14 * pairs}


# --------------------------------------------------------------------------------------------------------------------------------- inputs
def _normal(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device='cuda') * scale).to(dtype)


def _sections(case):
    return tuple(int(s) for s in case['sections'].split('+'))


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dt = DTYPES[case['dtype']]
    st = dict(case=case)
    if case['op'] == 'layer_norm':
        st['x'] = _normal((case['rows'], case['cols']), gen, dt, 1.7)
        st['x'] += 0.3
        st['weight'] = 1 + 0.1 * torch.randn(case['cols'], generator=gen, device='cuda')
        st['bias'] = 0.1 * torch.randn(case['cols'], generator=gen, device='cuda')
        if case['train']:
            st['dy'] = _normal((case['rows'], case['cols']), gen, dt)
        return st
    if case['op'] == 'rotary':
        t, h, w = case['t'], case['h'], case['w']
        start = torch.randint(0, 4096, (1,), generator=gen, device='cuda', dtype=torch.int32)              # the clip begins somewhere in a long video
        axes = torch.meshgrid(*[torch.arange(n, device='cuda', dtype=torch.int32) for n in (t, h, w)], indexing='ij')
        st['positions'] = torch.stack([(axes[0] + start).reshape(-1), axes[1].reshape(-1), axes[2].reshape(-1)], dim=1).contiguous()
        for name, heads in (('q', case['heads']), ('k', case['kv_heads'])):
            st[name] = _normal((case['batch'], t * h * w, heads, case['dim']), gen, dt)
            if case['train']:
                st['d' + name] = _normal((case['batch'], t * h * w, heads, case['dim']), gen, dt)
        return st
    b, lq, lk, d = case['batch'], case['lq'], case['lk'], case['dim']
    st['q'] = _normal((b, lq, case['heads'], d), gen, dt)
    st['k'] = _normal((b, lk, case['kv_heads'], d), gen, dt)
    st['v'] = _normal((b, lk, case['kv_heads'], d), gen, dt)
    st['lengths'] = torch.tensor(_lengths(case), dtype=torch.int32, device='cuda') if case['ragged'] else None
    st['prefix'] = torch.full((b,), case['prefix'], dtype=torch.int32, device='cuda') if case['prefix'] else None
    st['documents'] = torch.tensor(_doc_ids(case, lk), dtype=torch.int32, device='cuda').repeat(b, 1) if case['docs'] else None
    st['slopes'] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case['heads']) for h in range(case['heads'])], device='cuda') if case['slopes'] else None
    if case['train']:
        st['do'] = _normal((b, lq, case['heads'], d), gen, dt)
    return st


# ------------------------------------------------------------------------------------------------------------- the framework's operators
def _leaf(t):
    return t.detach().requires_grad_()


def _run_own(st):
    from next3d_amd.torch_utils.ops import attention, layer_norm, rotary
    case = st['case']
    if case['op'] == 'layer_norm':
        if not case['train']:
            return layer_norm.layer_norm(st['x'], st['weight'], st['bias'], eps=EPS)
        x, w, b = _leaf(st['x']), _leaf(st['weight']), _leaf(st['bias'])
        y = layer_norm.layer_norm(x, w, b, eps=EPS)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), st['dy'])
        return dict(y=y.detach(), dx=dx, dw=dw, db=db)
    if case['op'] == 'rotary':
        kw = dict(base=BASE, pairing=case['pairing'], ladder=case['ladder'])
        if not case['train']:
            q, k = rotary.rotary(st['q'], st['positions'], _sections(case), k=st['k'], **kw)
            return dict(q=q, k=k)
        q, k = _leaf(st['q']), _leaf(st['k'])
        yq, yk = rotary.rotary(q, st['positions'], _sections(case), k=k, **kw)
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (st['dq'], st['dk']))
        return dict(q=yq.detach(), k=yk.detach(), dq=dq, dk=dk)
    kw = dict(causal=case['causal'], prefix=st['prefix'], documents=st['documents'], lengths=st['lengths'], softcap=case['softcap'], slopes=st['slopes'])
    if not case['train']:
        return attention.attention(st['q'], st['k'], st['v'], **kw)
    q, k, v = _leaf(st['q']), _leaf(st['k']), _leaf(st['v'])
    o = attention.attention(q, k, v, **kw)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), st['do'])
    return dict(o=o.detach(), dq=dq, dk=dk, dv=dv)


# ------------------------------------------------------------------------------------------------------------------------- the plain form
def _plain_layer_norm(st):
    case = st['case']
    x = st['x'].float()
    mean = x.mean(dim=1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(dim=1, keepdim=True) + EPS)
    xhat = xc * rstd
    y = (xhat * st['weight'] + st['bias']).to(st['x'].dtype)
    if not case['train']:
        return y
    dy = st['dy'].float()
    g = dy * st['weight']
    dx = rstd * (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True))
    return dict(y=y, dx=dx.to(st['x'].dtype), dw=(dy * xhat).sum(dim=0), db=dy.sum(dim=0))


def _pairs(case):
    """(axis, frequency exponent, first channel, second channel) of every rotated pair."""
    sections = _sections(case)
    total = sum(sections) // 2
    out, p, offset = [], 0, 0
    for a, s in enumerate(sections):
        for i in range(s // 2):
            exponent = 2 * i / s if case['ladder'] == 'axis' else p / total
            if case['pairing'] == 'interleaved':
                lo, hi = 2 * p, 2 * p + 1
            elif case['ladder'] == 'axis':
                lo, hi = offset + i, offset + i + s // 2
            else:
                lo, hi = p, p + total
            out.append((a, exponent, lo, hi))
            p += 1
        offset += s
    return out


def _plain_rotary(st):
    case = st['case']
    pairs = _pairs(case)
    dev = st['q'].device
    axis = torch.tensor([p[0] for p in pairs], device=dev)
    freq = torch.tensor([BASE ** -p[1] for p in pairs], dtype=torch.float64, device=dev)
    lo = torch.tensor([p[2] for p in pairs], device=dev)
    hi = torch.tensor([p[3] for p in pairs], device=dev)
    angle = st['positions'].double()[:, axis] * freq
    cos, sin = torch.cos(angle).float()[None, :, None, :], torch.sin(angle).float()[None, :, None, :]

    def turn(x, s):
        f = x.float()
        y = f.clone()
        a, b = f[..., lo], f[..., hi]
        y[..., lo] = a * cos - b * s
        y[..., hi] = a * s + b * cos
        return y.to(x.dtype)

    out = dict(q=turn(st['q'], sin), k=turn(st['k'], sin))
    if case['train']:
        out['dq'], out['dk'] = turn(st['dq'], -sin), turn(st['dk'], -sin)
    return out


def _plain_mask(st, b, i0, i1):
    """[i1 - i0, Lk] of sequence b: which keys the queries see, and how far away they are."""
    case = st['case']
    dev = st['q'].device
    n = st['lengths'][b] if st['lengths'] is not None else case['lk']
    pos = torch.arange(i0, i1, device=dev)[:, None] + (n - case['lq'])
    j = torch.arange(case['lk'], device=dev)[None, :]
    see = (j < n).expand(i1 - i0, case['lk'])
    if case['causal']:
        open_ = j <= pos
        if st['prefix'] is not None:
            open_ = open_ | (j < st['prefix'][b])
        see = see & open_
    if st['documents'] is not None:
        dq, dk = st['documents'][b, i0:i1, None], st['documents'][b, None, :]
        see = see & (dq == dk) & (dq >= 0)
    return see, (pos - j).abs().float()


def _plain_attention(st):
    case = st['case']
    hq, hk, d, lq, lk = case['heads'], case['kv_heads'], case['dim'], case['lq'], case['lk']
    group, scale, cap = hq // hk, 1.0 / math.sqrt(case['dim']), case['softcap']
    dt, train = st['q'].dtype, case['train']
    out = torch.empty_like(st['q'])
    grads = [torch.empty_like(st[n]) for n in 'qkv'] if train else None
    rows = max(1, min(lq, 2 ** 28 // (hq * lk)))
    for b in range(case['batch']):
        k = st['k'][b].float().transpose(0, 1).contiguous()                             # [hk, lk, d]
        v = st['v'][b].float().transpose(0, 1).contiguous()
        kt, vt = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
        if train:
            dk, dv = torch.zeros_like(k), torch.zeros_like(v)
        for i0 in range(0, lq, rows):
            i1 = min(lq, i0 + rows)
            m = i1 - i0
            q = st['q'][b, i0:i1].float().transpose(0, 1).reshape(hk, group * m, d)     # query heads of a key head are neighbours
            s = (q @ kt).reshape(hq, m, lk) * scale
            if cap:
                th = torch.tanh(s / cap)
                s = cap * th
            see, dist = _plain_mask(st, b, i0, i1)
            if st['slopes'] is not None:
                s = s - st['slopes'][:, None, None] * dist
            s = s.masked_fill(~see, float('-inf'))
            top = s.amax(dim=2, keepdim=True)
            p = torch.exp(s - torch.where(top == float('-inf'), torch.zeros_like(top), top))
            total = p.sum(dim=2, keepdim=True)
            p = p / torch.where(total == 0, torch.ones_like(total), total)
            o = p.reshape(hk, group * m, lk) @ v
            out[b, i0:i1] = o.reshape(hq, m, d).transpose(0, 1).to(dt)
            if train:
                do = st['do'][b, i0:i1].float().transpose(0, 1).reshape(hk, group * m, d)
                delta = (do * o).sum(dim=2).reshape(hq, m, 1)
                dv += p.reshape(hk, group * m, lk).transpose(1, 2).contiguous() @ do
                ds = p * ((do @ vt).reshape(hq, m, lk) - delta)
                if cap:
                    ds = ds * (1 - th * th)
                ds = (ds * scale).reshape(hk, group * m, lk)
                grads[0][b, i0:i1] = (ds @ k).reshape(hq, m, d).transpose(0, 1).to(dt)
                dk += ds.transpose(1, 2).contiguous() @ q
        if train:
            grads[1][b], grads[2][b] = dk.transpose(0, 1).to(dt), dv.transpose(0, 1).to(dt)
    return dict(o=out, dq=grads[0], dk=grads[1], dv=grads[2]) if train else out


def run(state):
    if own:
        return _run_own(state)
    return {'layer_norm': _plain_layer_norm, 'rotary': _plain_rotary, 'attention': _plain_attention}[state['case']['op']](state)


# --------------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_layer_norm(st):
    train = st['case']['train']
    x, w, b = (st[n].double().requires_grad_(train) for n in ('x', 'weight', 'bias'))
    centred = x - x.sum(1, keepdim=True) / x.shape[1]
    y = centred / (centred.square().sum(1, keepdim=True) / x.shape[1] + EPS).sqrt() * w + b
    if not train:
        return y
    dx, dw, db = torch.autograd.grad(y, (x, w, b), st['dy'].double())
    return dict(y=y.detach(), dx=dx, dw=dw, db=db)


def _exact_rotary(st):
    case = st['case']
    sections = _sections(case)
    pos = st['positions'].double()
    half = sum(sections) // 2
    if case['ladder'] == 'axis':
        angles = [pos[:, a, None] * torch.pow(BASE, -torch.arange(0, s, 2, device=pos.device, dtype=torch.float64) / s) for a, s in enumerate(sections)]
    else:
        ladder = torch.pow(BASE, -torch.arange(half, device=pos.device, dtype=torch.float64) / half).split([s // 2 for s in sections])
        angles = [pos[:, a, None] * f for a, f in enumerate(ladder)]

    def as_pairs(x):                                                              # -> one (first, second) block per axis
        if case['pairing'] == 'interleaved':
            return [(c[..., 0::2], c[..., 1::2]) for c in x[..., :2 * half].split(sections, dim=-1)]
        if case['ladder'] == 'axis':
            return [c.chunk(2, dim=-1) for c in x[..., :2 * half].split(sections, dim=-1)]
        cut = [s // 2 for s in sections]
        return list(zip(x[..., :half].split(cut, dim=-1), x[..., half:2 * half].split(cut, dim=-1)))

    def turn(x, sign):
        x = x.double()
        firsts, seconds = [], []
        for (a, b), t in zip(as_pairs(x), angles):
            z = torch.complex(a.contiguous(), b.contiguous()) * torch.polar(torch.ones_like(t), sign * t)[:, None, :]
            firsts.append(z.real)
            seconds.append(z.imag)
        if case['pairing'] == 'interleaved':
            body = [torch.stack(p, dim=-1).flatten(-2) for p in zip(firsts, seconds)]
        elif case['ladder'] == 'axis':
            body = [torch.cat(p, dim=-1) for p in zip(firsts, seconds)]
        else:
            body = firsts + seconds
        return torch.cat(body + [x[..., 2 * half:]], dim=-1)

    out = {n: turn(st[n], 1.0) for n in ('q', 'k')}
    if case['train']:
        out.update({n: turn(st[n], -1.0) for n in ('dq', 'dk')})
    return out


def _exact_attention(st):
    case = st['case']
    train, group, lq, lk = case['train'], case['heads'] // case['kv_heads'], case['lq'], case['lk']
    dev = st['q'].device
    shape = {n: st[n].shape for n in 'qkv'}
    res = {n: torch.zeros(s, dtype=torch.float64, device=dev) for n, s in (('o', shape['q']), ('dq', shape['q']), ('dk', shape['k']), ('dv', shape['v']))}
    for b, n in enumerate(_lengths(case)):
        i, j = torch.arange(lq, device=dev)[:, None] + n - lq, torch.arange(lk, device=dev)[None, :]
        hidden = j >= n
        if case['causal']:
            hidden = hidden | ((j > i) & (j >= case['prefix']))
        if case['docs']:
            ids = torch.tensor(_doc_ids(case, lk), device=dev)
            hidden = hidden | (ids[:, None] != ids[None, :]) | (ids[:, None] < 0)
        empty = hidden.expand(lq, lk).all(dim=1, keepdim=True)
        for h in range(case['heads']):
            q, k, v = (st[m][b, :, g].double().requires_grad_(train) for m, g in (('q', h), ('k', h // group), ('v', h // group)))
            score = torch.mm(q, k.t().contiguous()) / math.sqrt(case['dim'])
            if case['softcap']:
                score = torch.tanh(score / case['softcap']) * case['softcap']
            if case['slopes']:
                score = score - float(st['slopes'][h]) * (i - j).abs()
            score = score.masked_fill(hidden, -1e300)
            prob = torch.softmax(score, dim=1).masked_fill(empty, 0.0)
            o = torch.mm(prob, v)
            res['o'][b, :, h] = o.detach()
            if train:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), st['do'][b, :, h].double())
                res['dq'][b, :, h] = dq
                res['dk'][b, :, h // group] += dk
                res['dv'][b, :, h // group] += dv
    return res if train else res['o']


def exact(case, seed):
    return {'layer_norm': _exact_layer_norm, 'rotary': _exact_rotary, 'attention': _exact_attention}[case['op']](prepare(case, seed))
