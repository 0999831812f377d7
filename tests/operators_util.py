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
