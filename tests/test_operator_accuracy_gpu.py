"""Kernel variants that only some sizes select, against the fp64 definitions, and the accuracy that the 16-bit forms claim.

``ratio`` is the norm of a result's error over the norm of the error that one rounding of the exact result makes.  What it may be:
  a single rounding (h, db, and gradients whose terms are kept to twice the type's digits)  1; measured up to 1.2, and norms of a few thousand
      random errors scatter by 1 / sqrt(2 n) of themselves, some percent: 1.3
  a sum whose terms are rounded once before (dx and dW of the gated projection): the terms' errors are as large as the result's and
      independent of them, sqrt(2) = 1.41; 1.5 with the scatter
  the same for dq, dk and dv at 64 columns per map and long sums: measured 1.4 to 1.5; 1.6
  out: the weights of both maps are rounded.  For scores of variance 1, sum p^2 = e / n and sum p1 p2 = 1 / n, so the terms' error is
      (1 + lam^2) / (1 + lam^2 - 2 lam / e) of the result's, at most 1.58 (lam = 1): sqrt(2.58) = 1.61; 1.7"""
import pytest
import torch

from tests.operators_util import assert_within, blocked_pairs, diff_attention64, gated64

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _inputs(B, Nq, Nk, H, G, d, dt, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    return (r(B, Nq, H * 2 * d).to(dt), r(B, Nk, G * 2 * d).to(dt), r(B, Nk, G * 2 * d).to(dt), r(H).clamp(-1, 1).to(dt), r(B, Nq, H * 2 * d).to(dt))


def _results(q, k, v, lam, dout, H, **kw):
    from focalformer3d_amd import ops
    saved = ops.diff_attention_train_fwd(q, k, v, lam, H, **kw)
    return (saved[0], *ops.diff_attention_bwd(q, k, v, lam, H, *saved, dout, **kw))


def _exact(q, k, v, lam, dout, H, G, mask=None, kv_lens=None, causal=False):
    blocked = blocked_pairs(q.shape[0], q.shape[1], k.shape[1], mask, kv_lens, causal, q.device)
    return diff_attention64(q, k, v, lam, H, G, blocked, None, dout)


NAMES = ('out', 'dq', 'dk', 'dv', 'dlam')


def ratio(got, exact, dtype):
    exact = exact.reshape(got.shape)
    return float((got.double() - exact).norm() / (exact.to(dtype).double() - exact).norm())


# blocks of 128 rows that share keys and values need 256 of them
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('B,Nq,Nk,H,G,d', [(8, 300, 150, 16, 16, 8), (4, 301, 97, 32, 32, 16), (2, 1500, 203, 24, 12, 32), (6, 260, 131, 15, 15, 64)])
def test_many_rows(dtype, B, Nq, Nk, H, G, d):
    dt = DT[dtype]
    assert B * G * -(-Nq * (H // G) // 128) >= 256
    q, k, v, lam, dout = _inputs(B, Nq, Nk, H, G, d, dt, 1)
    g = torch.Generator(device='cuda').manual_seed(2)
    mask = torch.rand(B, Nq, Nk, generator=g, device='cuda') < 0.3
    mask[:, 3::7] = True
    lens = torch.randint(0, Nk + 1, (B,), generator=g, device='cuda', dtype=torch.int32)
    lens[0] = 0
    for kw in ({}, dict(mask=mask), dict(mask=mask[0], causal=True), dict(mask=mask, kv_lens=lens), dict(kv_lens=lens)):
        for name, t, want in zip(NAMES, _results(q, k, v, lam, dout, H, kv_heads=G, **kw), _exact(q, k, v, lam, dout, H, G, **kw)):
            assert_within(t, want, (name, list(kw)))


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('masked', [False, True])
def test_long_sequences_of_64_columns(dtype, masked):
    """More than 2^24 (row, key) pairs to a key head, shared heads, the causal order, with a mask too."""
    dt, H, G, d, N = DT[dtype], 4, 1, 64, 2200
    q, k, v, lam, dout = _inputs(1, N, N, H, G, d, dt, 3)
    kw = dict(causal=True)
    if masked:
        kw['mask'] = torch.rand(1, N, N, generator=torch.Generator(device='cuda').manual_seed(4), device='cuda') < 0.2
    exact = _exact(q, k, v, lam, dout, H, G, **kw)
    for name, t, want in zip(NAMES, _results(q, k, v, lam, dout, H, kv_heads=G, **kw), exact):
        assert_within(t, want, name)
        if dt != torch.float32 and name != 'dlam':
            assert ratio(t, want[0], dt) <= (1.7 if name == 'out' else 1.6), name


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('B,Nq,Nk,H,G,d', [(2, 300, 300, 8, 4, 16), (2, 200, 500, 4, 4, 8), (2, 400, 333, 4, 2, 32), (2, 256, 256, 8, 2, 64),
                                           (4, 260, 4, 4, 4, 32), (4, 260, 3, 4, 2, 16)])
def test_accuracy_of_differential_attention(dtype, B, Nq, Nk, H, G, d):
    dt = DT[dtype]
    args = _inputs(B, Nq, Nk, H, G, d, dt, 5)
    for name, t, want in zip(NAMES, _results(*args, H, kv_heads=G), _exact(*args, H, G)):
        assert ratio(t, want[0], dt) <= (1.7 if name == 'out' else 1.3), name


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('act', ['silu', 'gelu'])
def test_accuracy_of_the_gated_projection(dtype, act):
    from focalformer3d_amd import ops
    dt, M, C, F = DT[dtype], 700, 200, 304
    g = torch.Generator(device='cuda').manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    x, w, b, dh = r(M, C).to(dt), (r(2 * F, C) * C ** -0.5).to(dt), (r(2 * F) * 0.3).to(dt), (r(M, F) * 0.1).to(dt)
    got = (ops.gated_linear(x, w, b, act), *ops.gated_linear_bwd(x, w, b, act, dh))
    for name, t, want, most in zip(('h', 'dx', 'dw', 'db'), got, gated64(x, w, b, act, dh), (1.3, 1.5, 1.5, 1.3)):
        assert ratio(t, want[0], dt) <= most, name


# the few-row kernel with eight waves (rows of 2048 bytes and more), up to its last number of rows and past it
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('M', [1, 4, 8, 9, 31, 32, 33, 70, 96, 97])
@pytest.mark.parametrize('C,F,bias', [(1024, 333, True), (1032, 64, False), (1347, 40, True)])
def test_few_rows_of_wide_blocks(dtype, M, C, F, bias):
    from focalformer3d_amd import ops
    dt = DT[dtype]
    g = torch.Generator(device='cuda').manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    x, w, b = r(M, C).to(dt), (r(2 * F, C) * C ** -0.5).to(dt), (r(2 * F) * 0.3).to(dt) if bias else None
    for act in ('silu', 'relu'):
        assert_within(ops.gated_linear(x, w, b, act), gated64(x, w, b, act)[0], act)
