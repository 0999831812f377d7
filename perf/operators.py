"""What is measured of three operators of a decoder layer and its training step: differential attention, the gated
projection of a feed-forward block, and clipping of gradients by their global norm.

``run`` computes them in plain torch (fp32, rounded once at the end) where ``own`` is false, and calls
``focalformer3d_amd.autograd.differential_attention`` / ``gated_linear``, ``focalformer3d_amd.ops.diff_attention`` and
``focalformer3d_amd.training.clip_grads`` where it is true.  ``exact`` gives the same results in fp64.

  attention   out = softmax(s q1 k1^T) v - lam softmax(s q2 k2^T) v per head; a head of q / k is [q1 | q2] of d each, of v 2 d;
              blocked keys count as absent, a row with no key left gives zeros
  gated       h = act(x Wg^T + bg) * (x Wu^T + bu), the weight being [Wg ; Wu] of (2 F, C)
  clip        n = || all gradients ||,  out_i = g_i * min(1, max_norm / (n + 1e-6))
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
# a drawn case costs at most what the largest listed one of its operator does
ATTN_FLOPS, GATED_FLOPS, CLIP_ELEMENTS = 150e9, 500e9, 160e6


def _attn(name, dtype, B, Nq, Nk, heads, kv_heads, d, mask, train):
    return dict(name=name, op='attn', dtype=dtype, B=B, Nq=Nq, Nk=Nk, heads=heads, kv_heads=kv_heads, d=d, mask=mask, train=train)


def _gated(name, dtype, M, C, F, act, bias, train):
    return dict(name=name, op='gated', dtype=dtype, M=M, C=C, F=F, act=act, bias=bias, train=train)


def _clip(name, dtype, layers, C, F, max_norm):
    return dict(name=name, op='clip', dtype=dtype, layers=layers, C=C, F=F, max_norm=max_norm)


def listed():
    return [
        # one frame's 600 queries at width 256, 8 heads, evaluation: a latency-bound launch of the detector
        _attn('attn_queries_eval_f32', 'f32', 1, 600, 600, 8, 8, 16, 'none', False),
        # a training step of four frames: 600 queries + 3 ground-truth groups of 40 that do not see each other
        _attn('attn_queries_train_f32', 'f32', 4, 720, 720, 8, 8, 16, 'groups', True),
        # a long causal sequence with shared key heads in bf16, forward and backward: the matrix-core bound case
        _attn('attn_causal_train_bf16', 'bf16', 1, 4096, 4096, 16, 4, 64, 'causal', True),
        # queries over another, padded sequence, odd lengths, some rows with no key left
        _attn('attn_cross_train_f16', 'f16', 3, 333, 1777, 4, 4, 32, 'holes', True),
        # one new token per sequence over a long padded cache: bound by reading keys and values
        _attn('attn_token_bf16', 'bf16', 8, 1, 16384, 16, 4, 64, 'lens', False),
        # feed-forward width 1024 over one frame's queries: latency
        _gated('gated_frame_f32', 'f32', 600, 256, 1024, 'relu', True, False),
        # the same block in the four-frame training step
        _gated('gated_train_f32', 'f32', 2880, 256, 1024, 'gelu', True, True),
        # a wide block over many rows in bf16, forward and backward: the matrix-core bound case
        _gated('gated_train_bf16', 'bf16', 16384, 1024, 2736, 'silu', False, True),
        # few rows through a wide block: bound by reading the weight
        _gated('gated_token_bf16', 'bf16', 4, 1024, 2736, 'silu', False, False),
        # the gradients of a decoder of width 128: many small tensors, latency
        _clip('clip_decoder_f32', 'f32', 3, 128, 1024, 0.1),
        # a wide model's gradients, clipped
        _clip('clip_wide_f32', 'f32', 5, 1024, 4100, 35.0),
        # bf16 gradients, odd sizes
        _clip('clip_wide_bf16', 'bf16', 5, 1023, 7001, 1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['attn', 'attn', 'gated', 'gated', 'clip'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    while True:
        if op == 'attn':
            heads = rng.choice([1, 2, 4, 6, 8, 12, 16])
            kv = rng.choice([g for g in range(1, heads + 1) if heads % g == 0])
            mask = rng.choice(['none', 'groups', 'causal', 'holes', 'lens'])
            nk = _log(rng, 1, 16384)
            nq = nk if mask == 'groups' else rng.choice([1, nk, _log(rng, 1, 4096)])
            c = _attn('', dtype, rng.randint(1, 8), nq, nk, heads, kv, rng.choice([8, 16, 32, 64]), mask, rng.random() < 0.6)
            fits = (work(c)['flops'] <= ATTN_FLOPS * (0.2 if dtype == 'f32' else 1)
                    and c['B'] * heads * nq * nk <= 16 * 4096 * 4096)
        elif op == 'gated':
            c = _gated('', dtype, _log(rng, 1, 16384), _log(rng, 16, 1536), _log(rng, 16, 4096), rng.choice(['silu', 'gelu', 'relu', 'sigmoid']),
                       rng.random() < 0.5, rng.random() < 0.6)
            if rng.random() < 0.6:                       # most widths are multiples of 8, some are odd
                c['C'], c['F'] = -(-c['C'] // 8) * 8, -(-c['F'] // 8) * 8
            fits = work(c)['flops'] <= GATED_FLOPS * (0.2 if dtype == 'f32' else 1)
        else:
            c = _clip('', dtype, rng.randint(1, 5), _log(rng, 16, 1200), _log(rng, 16, 6000), rng.choice([0.1, 1.0, 35.0, 1e9]))
            fits = sum(math.prod(s) for s in _clip_shapes(c)) <= CLIP_ELEMENTS
        if fits:
            c.pop('name')
            return c


def _clip_shapes(c):
    """Parameter shapes of `layers` decoder layers: attention, a gated block, norms, biases (11 each), and a head."""
    C, F = c['C'], c['F']
    layer = [(3 * C, C), (3 * C,), (C, C), (C,), (2 * F, C), (2 * F,), (C, F), (C,), (C,), (C,), (2, C)]
    return layer * c['layers'] + [(F, C, 3, 3) if F * C * 9 < 4e6 else (F, C), (10, C)]


def prepare(case, seed):
    c, dt, dev = case, DTYPES[case['dtype']], 'cuda'
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    if c['op'] == 'attn':
        B, Nq, Nk, H, G, d = (c[k] for k in ('B', 'Nq', 'Nk', 'heads', 'kv_heads', 'd'))
        st = dict(case=c, q=randn(B, Nq, H * 2 * d), k=randn(B, Nk, G * 2 * d), v=randn(B, Nk, G * 2 * d),
                  lam=(0.2 + 0.6 * torch.rand(H, generator=g, device=dev)).to(dt), mask=None, kv_lens=None)
        if c['mask'] == 'groups':                        # 5/6 ordinary queries, three groups: a query sees its own kind only
            kind = (torch.arange(Nk, device=dev) - Nk * 5 // 6).clamp(min=-1)
            kind = torch.where(kind < 0, -1, kind * 3 // max(Nk - Nk * 5 // 6, 1))
            blocked = kind[:, None] != kind[None, :]
            blocked[:, : Nk * 5 // 6] &= (kind < 0)[:, None]
            st['mask'] = blocked[None].expand(B, -1, -1).contiguous()
        if c['mask'] == 'holes':                         # a tenth of the pairs blocked, every 16th query sees nothing
            blocked = torch.rand(B, Nq, Nk, generator=g, device=dev) < 0.1
            blocked[:, 5::16] = True
            st['mask'] = blocked
        if c['mask'] in ('holes', 'lens'):
            lens = torch.randint(Nk // 2, Nk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
            lens[0] = Nk
            st['kv_lens'] = lens
        if c['train']:
            st['dout'] = randn(B, Nq, H * 2 * d)
            for n in ('q', 'k', 'v', 'lam'):
                st[n].requires_grad_(True)
    elif c['op'] == 'gated':
        M, C, F = c['M'], c['C'], c['F']
        st = dict(case=c, x=randn(M, C), weight=randn(2 * F, C, scale=C ** -0.5), bias=randn(2 * F, scale=0.1) if c['bias'] else None)
        if c['train']:
            st['dh'] = randn(M, F, scale=1e-3)
            for n in ('x', 'weight', 'bias'):
                if st[n] is not None:
                    st[n].requires_grad_(True)
    else:
        shapes = _clip_shapes(c)
        grads = [randn(*s, scale=0.01 * (1 + i % 5)) for i, s in enumerate(shapes)]
        st = dict(case=c, grads=grads, out=[torch.empty_like(t) for t in grads])
    return st


def run(state):
    op, train = state['case']['op'], state['case'].get('train')
    if own:
        return _own(state, op, train)
    if op == 'attn':
        return _plain_attn(state, train)
    if op == 'gated':
        return _plain_gated(state, train)
    return _plain_clip(state)


def _own(st, op, train):
    from focalformer3d_amd import ops
    from focalformer3d_amd.autograd import differential_attention, gated_linear
    from focalformer3d_amd.training import clip_grads
    c = st['case']
    if op == 'attn':
        kw = dict(kv_heads=c['kv_heads'], mask=st['mask'], kv_lens=st['kv_lens'], causal=c['mask'] == 'causal')
        if not train:
            return ops.diff_attention(st['q'], st['k'], st['v'], st['lam'], c['heads'], **kw)
        out = differential_attention(st['q'], st['k'], st['v'], st['lam'], c['heads'], **kw)
        return (out, *torch.autograd.grad(out, (st['q'], st['k'], st['v'], st['lam']), st['dout']))
    if op == 'gated':
        if not train:
            return ops.gated_linear(st['x'], st['weight'], st['bias'], act=c['act'])
        h = gated_linear(st['x'], st['weight'], st['bias'], act=c['act'])
        leaves = (st['x'], st['weight']) + ((st['bias'],) if st['bias'] is not None else ())
        return (h, *torch.autograd.grad(h, leaves, st['dh']))
    norm = clip_grads(st['grads'], c['max_norm'], out=st['out'])
    return (norm, *st['out'])


def _blocked(st, dev):
    """(B or 1, 1, 1, Nq, Nk) truth values, True = key not attended; None if every key is."""
    c = st['case']
    Nq, Nk = c['Nq'], c['Nk']
    out = None if st['mask'] is None else st['mask'][:, None, None]
    j = torch.arange(Nk, device=dev)
    if st['kv_lens'] is not None:
        past = (j >= st['kv_lens'][:, None])[:, None, None, None]
        out = past.expand(-1, -1, -1, Nq, -1) if out is None else out | past
    if c['mask'] == 'causal':                            # the last query sees the last key
        later = (j > torch.arange(Nq, device=dev)[:, None] + (Nk - Nq))[None, None, None]
        out = later if out is None else out | later
    return out


@torch.no_grad()
def _plain_attn(st, train):
    c = st['case']
    B, Nq, Nk, H, G, d = (c[k] for k in ('B', 'Nq', 'Nk', 'heads', 'kv_heads', 'd'))
    dt, s, r = st['q'].dtype, d ** -0.5, H // G
    q = st['q'].float().view(B, Nq, H, 2, d).permute(0, 2, 3, 1, 4).contiguous()
    k = st['k'].float().view(B, Nk, G, 2, d).permute(0, 2, 3, 1, 4).repeat_interleave(r, 1).contiguous()
    v = st['v'].float().view(B, Nk, G, 2 * d).permute(0, 2, 1, 3).repeat_interleave(r, 1).contiguous()
    lam = st['lam'].float()[:, None, None]
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(s)
    blocked = _blocked(st, q.device)
    if blocked is not None:
        score.masked_fill_(blocked, -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    p1, p2 = p[:, :, 0], p[:, :, 1]
    w = p1 - lam * p2
    rows = lambda t: t.transpose(1, 2).reshape(B, Nq, H * 2 * d).to(dt)  # noqa: E731
    out = rows(torch.matmul(w, v))
    if not train:
        return out
    do = st['dout'].float().view(B, Nq, H, 2 * d).transpose(1, 2).contiguous()
    dv = torch.matmul(w.transpose(-1, -2).contiguous(), do)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    D = (p * dp[:, :, None]).sum(-1, keepdim=True)
    dlam = -D[:, :, 1].sum((0, 2, 3))
    ds = p.mul_(dp[:, :, None] - D).mul_(s)
    ds[:, :, 1] *= -lam
    dq = torch.matmul(ds, k).permute(0, 3, 1, 2, 4).reshape(B, Nq, H * 2 * d)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q).view(B, G, r, 2, Nk, d).sum(2).permute(0, 3, 1, 2, 4).reshape(B, Nk, G * 2 * d)
    dv = dv.view(B, G, r, Nk, 2 * d).sum(2).transpose(1, 2).reshape(B, Nk, G * 2 * d)
    return out, dq.to(dt), dk.to(dt), dv.to(dt), dlam.to(dt)


def _act(g, act):
    """act(g) and its derivative."""
    if act == 'relu':
        return g.clamp(min=0), (g > 0).to(g.dtype)
    if act == 'gelu':
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    sig = torch.sigmoid(g)
    if act == 'sigmoid':
        return sig, sig * (1 - sig)
    return g * sig, sig * (1 + g * (1 - sig))


@torch.no_grad()
def _plain_gated(st, train):
    c, dt = st['case'], st['x'].dtype
    F = c['F']
    x, w = st['x'].float(), st['weight'].float()
    gu = torch.matmul(x, w.t())
    if st['bias'] is not None:
        gu += st['bias'].float()
    g, u = gu[:, :F], gu[:, F:]
    a, da = _act(g, c['act'])
    h = (a * u).to(dt)
    if not train:
        return h
    dh = st['dh'].float()
    dgu = torch.cat([dh * u * da, dh * a], 1)
    out = (h, torch.matmul(dgu, w).to(dt), torch.matmul(dgu.t(), x).to(dt))
    return out if st['bias'] is None else out + (dgu.sum(0).to(dt),)


@torch.no_grad()
def _plain_clip(st):
    norm = torch.stack([t.float().square().sum() for t in st['grads']]).sum().sqrt()
    coef = (st['case']['max_norm'] / (norm + 1e-6)).clamp(max=1.0)
    return (norm, *[(t.float() * coef).to(t.dtype) for t in st['grads']])


def exact(case, seed):
    """The same results from the definitions in fp64: gradients by automatic differentiation of the forward formulas."""
    st, c = prepare(case, seed), case
    f64 = lambda t: None if t is None else t.detach().double()  # noqa: E731
    if c['op'] == 'clip':
        grads = [f64(t) for t in st['grads']]
        norm = torch.linalg.vector_norm(torch.cat([t.reshape(-1) for t in grads]))
        coef = min(1.0, c['max_norm'] / (float(norm) + 1e-6))
        return (norm, *[t * coef for t in grads])
    if c['op'] == 'gated':
        x, w, b = f64(st['x']).requires_grad_(c['train']), f64(st['weight']).requires_grad_(c['train']), f64(st['bias'])
        if b is not None:
            b.requires_grad_(c['train'])
        gate = torch.nn.functional.linear(x, w[: c['F']], None if b is None else b[: c['F']])
        up = torch.nn.functional.linear(x, w[c['F']:], None if b is None else b[c['F']:])
        h = {'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu, 'relu': torch.relu, 'sigmoid': torch.sigmoid}[c['act']](gate) * up
        if not c['train']:
            return h
        leaves = (x, w) if b is None else (x, w, b)
        return (h.detach(), *torch.autograd.grad(h, leaves, f64(st['dh'])))
    B, Nq, Nk, H, G, d = (c[k] for k in ('B', 'Nq', 'Nk', 'heads', 'kv_heads', 'd'))
    q, k, v, lam = (f64(st[n]) for n in ('q', 'k', 'v', 'lam'))
    out = torch.zeros_like(q)
    dq, dk, dv, dlam = (torch.zeros_like(t) for t in (q, k, v, lam))
    blocked = _blocked(st, q.device)
    for b in range(B):
        bl = None if blocked is None else blocked[b if blocked.shape[0] > 1 else 0, 0, 0]
        for h in range(H):
            cq, ck = slice(h * 2 * d, (h + 1) * 2 * d), slice(h // (H // G) * 2 * d, (h // (H // G) + 1) * 2 * d)
            qh, kh, vh, lh = (t.clone().requires_grad_(c['train']) for t in (q[b, :, cq], k[b, :, ck], v[b, :, ck], lam[h]))
            maps = []
            for m in range(2):
                e = (qh[:, m * d:(m + 1) * d] @ kh[:, m * d:(m + 1) * d].t()) / math.sqrt(d)
                if bl is not None:
                    e = e.masked_fill(bl, -1e300)
                pr = torch.softmax(e, -1)
                maps.append(pr if bl is None else pr.masked_fill(bl, 0.0))
            o = (maps[0] - lh * maps[1]) @ vh
            out[b, :, cq] = o.detach()
            if c['train']:
                gq, gk, gv, gl = torch.autograd.grad(o, (qh, kh, vh, lh), f64(st['dout'])[b, :, cq])
                dq[b, :, cq] += gq
                dk[b, :, ck] += gk
                dv[b, :, ck] += gv
                dlam[h] += gl
    return (out, dq, dk, dv, dlam) if c['train'] else out


def work(case):
    c = case
    size = 4 if c['dtype'] == 'f32' else 2
    if c['op'] == 'clip':
        n = sum(math.prod(s) for s in _clip_shapes(c))
        return {'bytes': 2 * n * size, 'flops': 3 * n}
    if c['op'] == 'gated':
        M, C, F = c['M'], c['C'], c['F']
        fwd = 4.0 * M * C * F
        moved = M * C + 2 * F * C + M * F
        return {'bytes': size * (moved + (M * F + M * C + 2 * F * C if c['train'] else 0)), 'flops': fwd * (3 if c['train'] else 1)}
    B, Nq, Nk, H, G, d = (c[k] for k in ('B', 'Nq', 'Nk', 'heads', 'kv_heads', 'd'))
    pairs = float(B) * H * Nq * Nk
    if c['mask'] == 'causal':
        pairs = float(B) * H * sum(max(0, Nk - Nq + i + 1) for i in range(Nq))
    elif c['mask'] in ('lens', 'holes'):                 # lengths between half and all of the keys
        pairs *= 0.75
    fwd = pairs * (2 * 2 * d + 2 * 2 * 2 * d)            # two score products of d, two value products of 2 d
    moved = B * (2 * Nq * H + 2 * Nk * G * (1 if c['mask'] not in ('lens', 'holes') else 0.75)) * 2 * d * size
    if c['mask'] in ('groups', 'holes'):
        moved += B * Nq * Nk
    if not c['train']:
        return {'bytes': moved, 'flops': fwd}
    # backward: both scores, dP, dV, both dQ and dK: 2 d products each
    return {'bytes': 2 * moved, 'flops': fwd + pairs * 2 * (5 * 2 * d)}
