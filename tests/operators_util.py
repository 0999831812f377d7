"""Definitions in fp64 of the operators in three types, and how far a right kernel may be from them.

Bounds count roundings: a rounding to a type is off by at most U[type] relative to the value; a sum of n products in fp32 by at most
(n + 16) * 2^-24 of the sum of their absolute values (16: splitting an fp32 operand and combining partial sums)."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# the smallest positive number of the type: what a rounding near zero is off by at most (half of it is enough)
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
E32 = 2.0 ** -24


def act64(g, act):
    """(act, act', bound on |act'|, bound on |act''| away from kinks)."""
    if act == 'relu':
        return g.clamp(min=0), (g > 0).double(), 1.0, 0.0
    if act == 'gelu':
        cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi), 1.13, 0.8
    s = torch.sigmoid(g)
    if act == 'sigmoid':
        return s, s * (1 - s), 0.25, 0.1
    return g * s, s * (1 + g * (1 - s)), 1.1, 0.5


def gated64(x, w, b, act, dh=None):
    """Results of the gated projection in fp64 with a bound for each: [(h, bound)] or with (dx, dw, db) too."""
    dt = x.dtype
    u, tiny = U[dt], TINY[dt]
    F, C = w.shape[0] // 2, w.shape[1]
    x, w = x.double().reshape(-1, C), w.double()
    pre = x @ w.t() + (0 if b is None else b.double())
    mag = x.abs() @ w.abs().t() + (0 if b is None else b.double().abs())
    e = (C + 16) * E32 * mag                                           # of g and u
    g, up, eg, eu = pre[:, :F], pre[:, F:], e[:, :F], e[:, F:]
    a, da, d1, d2 = act64(g, act)
    ea = d1 * eg + 16 * E32 * (a.abs() + 1e-3) + g.abs() * 2.0 ** -22 * a.abs()      # exp of a rounded argument
    h = a * up
    out = [(h, u * h.abs() + 1.01 * (ea * up.abs() + a.abs() * eu) + tiny)]
    if dh is None:
        return out
    dh = dh.double().reshape(-1, F)
    eda = d2 * eg + 16 * E32 * (1 + g.abs()) + g.abs() * 2.0 ** -22
    if act == 'relu':
        eda = eda + (g.abs() <= eg).double()                           # the sign of g is not known there
    dg, du = dh * up * da, dh * a
    d = torch.cat([dg, du], 1)
    ed = torch.cat([dh.abs() * (eu * da.abs() + (up.abs() + eu) * eda), dh.abs() * ea], 1) * 1.01 + 4 * E32 * d.abs()
    rd = ed + u * d.abs() + tiny                                       # d is rounded to the type for the two products
    M = x.shape[0]
    for value, bound in ((d @ w, rd @ w.abs() + (2 * F + 16) * E32 * (d.abs() @ w.abs())),
                         (d.t() @ x, rd.t() @ x.abs() + (M + 16) * E32 * (d.abs().t() @ x.abs()))):
        out.append((value, 1.01 * (u * value.abs() + bound) + tiny))
    if b is not None:
        out.append((d.sum(0), 1.01 * (u * d.sum(0).abs() + ed.sum(0) + (M + 16) * E32 * d.abs().sum(0)) + tiny))
    return out


def assert_within(got, want, what=''):
    """|got - value| <= bound, element by element."""
    value, bound = want
    assert got.numel() == value.numel(), (what, tuple(got.shape), tuple(value.shape))
    off = (got.detach().double().reshape(value.shape) - value).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float((off / bound)[bad].max()), float(off[bad].max()))


def blocked_pairs(B, Nq, Nk, mask, lens, causal, device):
    """(B, Nq, Nk) truth values: the pairs that the mask, the lengths or the causal order leave out."""
    j = torch.arange(Nk, device=device)
    out = torch.zeros(B, Nq, Nk, dtype=torch.bool, device=device)
    if mask is not None:
        out |= (mask != 0)
    if lens is not None:
        out |= (j >= lens.clamp(0, Nk)[:, None])[:, None]
    if causal:
        out |= j > torch.arange(Nq, device=device)[:, None] + Nk - Nq
    return out


def diff_attention64(q, k, v, lam, heads, kv_heads, blocked, scale=None, dout=None):
    """[(out, bound)] or with (dq, dk, dv, dlam) too, in fp64, (B, N, C) as the operator lays them out."""
    dt = q.dtype
    u, tiny = U[dt], TINY[dt]
    up = 0.0 if dt == torch.float32 else u                              # rounding of the probabilities, and of dS, to the type
    low = 2.0 ** -25 if dt == torch.float16 else 0.0                    # what fp16 loses of a probability next to one of 1
    # the exponential gives zero where its result lies below the smallest normal number of fp32: a probability, which is at most such a
    # result, is then off by up to 2^-126, and dS and dv by that times their other factors
    under = 2.0 ** -126
    B, Nq, Nk, r = q.shape[0], q.shape[1], k.shape[1], heads // kv_heads
    d = q.shape[2] // (2 * heads)
    scale = d ** -0.5 if scale is None else scale
    q_ = q.double().view(B, Nq, heads, 2, d).permute(0, 2, 3, 1, 4)
    k_ = k.double().view(B, Nk, kv_heads, 2, d).permute(0, 2, 3, 1, 4).repeat_interleave(r, 1)
    v_ = v.double().view(B, Nk, kv_heads, 2 * d).transpose(1, 2).repeat_interleave(r, 1)
    lam_ = lam.double().view(1, heads, 1, 1)
    bl = blocked[:, None, None]
    k_ = torch.where(k_.isfinite(), k_, 0.0)                            # keys that nobody attends may hold anything
    v_ = torch.where(v_.isfinite(), v_, 0.0)
    s = (q_ @ k_.transpose(-1, -2)) * scale
    es = (d + 16) * E32 * scale * (q_.abs() @ k_.abs().transpose(-1, -2))
    s = s.masked_fill(bl, -1e300)
    es, mag = es.masked_fill(bl, 0.0), s.masked_fill(bl, 0.0).abs()
    p = torch.softmax(s, -1).masked_fill(bl, 0.0)
    # the exponent, scaled by log2(e) and less the maximum, is off by a few roundings of the scores; so is every term of the sum
    delta = 2.1 * (es.amax(-1, keepdim=True) * 2 + (mag.amax(-1, keepdim=True) + 8) * 2.0 ** -22) + (Nk + 16) * E32
    p1, p2, va = p[:, :, 0], p[:, :, 1], v_.abs()
    d1, d2 = delta[:, :, 0], delta[:, :, 1]
    some = (~blocked).any(-1)[:, None, :, None].double()
    lost = (low + under) * some * torch.where(bl[:, :, 0], 0.0, 1.0) @ va
    o2 = p2 @ v_
    e1, e2 = (up + d1) * (p1 @ va) + lost, (up + d2) * (p2 @ va) + lost
    o = p1 @ v_ - lam_ * o2
    eo = u * o.abs() + 1.02 * (e1 + lam_.abs() * e2) + 4 * E32 * (lam_ * o2).abs() + tiny
    rows = lambda t: t.transpose(1, 2).reshape(B, Nq, heads * 2 * d)  # noqa: E731
    out = [(rows(o), rows(eo))]
    if dout is None:
        return out
    do = dout.double().view(B, Nq, heads, 2 * d).transpose(1, 2)
    da = do.abs()
    dp, edp = do @ v_.transpose(-1, -2), (2 * d + 16) * E32 * (da @ va.transpose(-1, -2))
    D2 = (do * o2).sum(-1, keepdim=True)
    eD2 = (da * (e2 + 2 * d * E32 * o2.abs())).sum(-1, keepdim=True) * 1.02
    D1 = (do * (o + lam_ * o2)).sum(-1, keepdim=True)
    eD1 = (da * (eo + 2 * d * E32 * o.abs())).sum(-1, keepdim=True) * 1.02 + lam_.abs() * eD2 + 2 * E32 * (D1.abs() + (lam_ * D2).abs())
    w = p1 - lam_ * p2
    ew = (up * w.abs() + 1.02 * (d1 * p1 + d2 * p2 * lam_.abs())) + 2 * E32 * (p1 + p2 * lam_.abs())
    ew = ew + (under + (2.0 ** -33 if low else 0.0)) * (1 + lam_.abs())
    ds, eds = [], []
    for pm, dm, D, eD, f in ((p1, d1, D1, eD1, torch.ones_like(lam_)), (p2, d2, D2, eD2, -lam_)):
        x = f * pm * (dp - D)
        e = f.abs() * under * (dp - D).abs() + f.abs() * pm * (1.02 * dm * (dp - D).abs() + edp + eD + 2 * E32 * (dp.abs() + D.abs())) * 1.02 + (up + 4 * E32) * x.abs()
        if low:                                                         # a column shares one scale: its largest value sets the step
            e = e + 2.0 ** -32 * torch.maximum(x.abs().amax(-1, keepdim=True), x.abs().amax(-2, keepdim=True))
        ds.append(x)
        eds.append(e)
    group = lambda t: t.view(B, kv_heads, r, Nk, -1).sum(2).transpose(1, 2).reshape(B, Nk, -1)  # noqa: E731

    def product(x, e, y, n, fold, f=1.0):
        val, bound = fold(x @ y) * f, fold(e @ y.abs() + (n + 16) * E32 * (x.abs() @ y.abs())) * f
        return val, 1.02 * (u * val.abs() + bound) + tiny
    dq = [product(ds[m], eds[m], k_[:, :, m], Nk, lambda t: t.transpose(1, 2), scale) for m in range(2)]
    out.append(tuple(torch.stack([a, b], 3).reshape(B, Nq, -1) for a, b in zip(*dq)))
    dk = [product(ds[m].transpose(-1, -2), eds[m].transpose(-1, -2), q_[:, :, m], Nq * r, group, scale) for m in range(2)]
    out.append(tuple(torch.stack([a.view(B, Nk, kv_heads, d), b.view(B, Nk, kv_heads, d)], 3).reshape(B, Nk, -1) for a, b in zip(*dk)))
    out.append(product(w.transpose(-1, -2), ew.transpose(-1, -2), do, Nq * r, group))
    dl = -D2.sum((0, 2, 3))
    out.append((dl, 1.02 * (u * dl.abs() + eD2.sum((0, 2, 3))) + 4 * E32 * D2.abs().sum((0, 2, 3)) + tiny))
    return out
