"""Calls of the operators in three types that their documentation allows: rows of unusual strides, forward-mode differentiation, second derivatives, modules with 16-bit
activations, gradients near the ends of fp16's range, sequences in large batches, long caches."""
import math

import pytest
import torch

from tests.operators_util import assert_within, blocked_pairs, diff_attention64, gated64

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _randn(seed, dt=torch.float32):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device='cuda').to(dt)


# ------------------------------------------------------------------------------------------------ one row
def _one_row(kind, C, dt):
    """A (1, C) view whose row stride says nothing, since there is one row."""
    r = _randn(21, dt)
    if kind == 'last token':
        t = torch.zeros(1, 4096, C, device='cuda', dtype=dt)
        t[:, -1] = r(1, C)
        return t[:, -1]
    if kind == 'column':
        return r(C, 1).t()
    flat = torch.zeros((1 << 20) + 1 + C, device='cuda', dtype=dt)
    t = flat.as_strided((1, C), ((1 << 20) + 1 if kind == 'odd' else 0, 1))
    t.copy_(r(1, C))
    return t


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('kind', ['last token', 'column', 'odd', 'zero'])
@pytest.mark.parametrize('C', [1024, 100])
def test_gated_linear_of_one_strided_row(dtype, kind, C):
    from focalformer3d_amd import ops
    from focalformer3d_amd.autograd import gated_linear
    dt, F = DT[dtype], 48
    x = _one_row(kind, C, dt)
    assert x.is_contiguous() and (x.stride(0) != C or kind == 'last token')
    r = _randn(22, dt)
    w, b, dh = r(2 * F, C) * C ** -0.5, r(2 * F), r(1, F)
    dense = x.clone(memory_format=torch.contiguous_format)
    want = (ops.gated_linear(dense, w, b), *ops.gated_linear_bwd(dense, w, b, 'silu', dh))
    got = (ops.gated_linear(x, w, b), *ops.gated_linear_bwd(x, w, b, 'silu', dh))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    leaf = x.detach().requires_grad_(True)
    h = gated_linear(leaf, w, b)
    dh_row = torch.zeros(F + 1, device='cuda', dtype=dt).as_strided((1, F), (1, 1)).copy_(dh)      # a gradient of such a row
    assert torch.equal(torch.autograd.grad(h, leaf, dh_row)[0], want[1])
    with torch.autograd.graph.save_on_cpu():
        h = gated_linear(leaf, w, b)
    assert torch.equal(torch.autograd.grad(h, leaf, dh)[0], want[1])
    assert torch.equal(ops.gated_linear(x[0], w, b), want[0][0])


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_gated_linear_of_one_value(dtype):
    """M = F = 1 and a gradient that is a broadcast scalar: every stride is 0."""
    from focalformer3d_amd.autograd import gated_linear
    dt = DT[dtype]
    r = _randn(23, dt)
    x, w = r(1, 16).requires_grad_(True), r(2, 16).requires_grad_(True)
    h = gated_linear(x, w)
    h.sum().backward()
    want = gated64(x.detach(), w.detach(), None, 'silu', torch.ones(1, 1, device='cuda', dtype=dt))
    for t, e in zip((h, x.grad, w.grad), want):
        assert_within(t, e)


# ------------------------------------------------------------------------------------------------ forward mode
def test_forward_mode_is_refused():
    """Neither operator has a forward-mode derivative: a dual operand is an error, not a result without a tangent."""
    import torch.autograd.forward_ad as fw
    from focalformer3d_amd.autograd import differential_attention, gated_linear
    from focalformer3d_amd.transformer import DifferentialAttention, GatedFFN
    r = _randn(24)
    q, k, v, lam = r(1, 6, 32), r(1, 7, 32), r(1, 7, 32), r(1)
    x, w = r(5, 16), r(8, 16)
    ffn, attention = GatedFFN(16, 32).cuda().eval(), DifferentialAttention(32, 2, batch_first=True).cuda().eval()
    want, h, y = differential_attention(q, k, v, lam, 1), gated_linear(x, w), ffn(x)
    with fw.dual_level():
        for i in range(4):
            args = [q, k, v, lam]
            args[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError), match='forward'):
                    differential_attention(*args, 1)
        dual = fw.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError), match='forward'):
                gated_linear(dual, w)
            with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError), match='forward'):
                ffn(dual)
            with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError), match='forward'):
                attention(fw.make_dual(q, torch.ones_like(q)))
        assert torch.equal(differential_attention(q, k, v, lam, 1), want) and torch.equal(gated_linear(x, w), h) and torch.equal(ffn(x), y)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: differential_attention(t, k, v, lam, 1), (q,), (torch.ones_like(q),))


# ------------------------------------------------------------------------------------------------ second derivatives
def test_second_derivatives_are_refused():
    """A graph of the gradients can be asked for; differentiating it again is an error, also where the incoming gradient is a constant."""
    from focalformer3d_amd.autograd import differential_attention, gated_linear
    r = _randn(33)
    q, lam, w = r(1, 6, 64).requires_grad_(True), r(2).requires_grad_(True), r(8, 64).requires_grad_(True)
    for y, leaf in ((differential_attention(q, q, q, lam, 2), q), (differential_attention(q.detach(), q.detach(), q.detach(), lam, 2), lam),
                    (gated_linear(q, w), w)):
        want, = torch.autograd.grad(y.sum(), leaf, retain_graph=True)
        got, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
        assert torch.equal(got, want) and got.requires_grad
        with pytest.raises(RuntimeError, match='twice'):
            (y.sum() + got.square().sum()).backward()


# ------------------------------------------------------------------------------------------------ modules in 16 bits
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_gated_ffn_evaluates_what_it_trains_on(dtype):
    """16-bit activations beside fp32 parameters under autocast: the inference route takes what the training route takes.  Four roundings of
    the type (input, hidden row, weights, result)."""
    from focalformer3d_amd.transformer import GatedFFN
    torch.manual_seed(25)
    m = GatedFFN(64, 96).cuda()
    x = torch.randn(2, 20, 64, device='cuda')
    P = {n: p.detach().double() for n, p in m.named_parameters()}

    def plain(x):
        g, u = torch.nn.functional.linear(x, P['in_proj.weight'], P['in_proj.bias']).chunk(2, -1)
        return x + torch.nn.functional.linear(torch.nn.functional.silu(g) * u, P['out_proj.weight'], P['out_proj.bias'])
    for inp in (x.to(dtype), x):
        want = plain(inp.double())
        with torch.autocast('cuda', dtype):
            y = m.train()(inp)
            with torch.no_grad():
                for z in (m.train()(inp), m.eval()(inp)):
                    assert float((z.double() - want).norm() / want.norm()) <= 4 * torch.finfo(dtype).eps / 2
        assert float((y.double() - want).norm() / want.norm()) <= 4 * torch.finfo(dtype).eps / 2


def test_gated_ffn_under_autocast_runs_in_the_autocast_type():
    """fp32 activations, as a LayerNorm under autocast hands them on, are cast as the Linear layers beside the operator cast theirs."""
    from focalformer3d_amd.transformer import GatedFFN
    torch.manual_seed(26)
    m = GatedFFN(64, 96).cuda().train()
    x = torch.randn(30, 64, device='cuda', requires_grad=True)
    h32 = m.hidden(x)[0]
    for dtype in (torch.bfloat16, torch.float16):
        with torch.autocast('cuda', dtype):
            h = m.hidden(x)[0]
            y = m(x)
        assert h.dtype == dtype and h32.dtype == torch.float32
        assert float((h.double() - h32.double()).norm() / h32.double().norm()) <= 4 * torch.finfo(dtype).eps / 2
        grads = torch.autograd.grad(y.float().square().sum(), [x, *m.parameters()])
        assert all(g.dtype == torch.float32 and bool(g.isfinite().all()) for g in grads)
        with torch.autocast('cuda', dtype), torch.autocast('cuda', enabled=False):
            assert m.hidden(x)[0].dtype == torch.float32
        with torch.autocast('cuda', dtype), pytest.raises(RuntimeError, match='float64'):      # which autocast leaves as it is
            m.hidden(x.double())


# ------------------------------------------------------------------------------------------------ fp16's range
def _gated_gradients(x, w, b, act, dh):
    from focalformer3d_amd import ops
    return ops.gated_linear_bwd(x, w, b, act, dh)


@pytest.mark.parametrize('act', ['silu', 'gelu', 'relu', 'sigmoid'])
@pytest.mark.parametrize('M,C,F,bias', [(2000, 64, 96, True), (300, 40, 33, False)])
def test_small_fp16_gradients_keep_their_digits(act, M, C, F, bias):
    """dh of 2^-19: dg and du lie below fp16's normal numbers, dx and dW do not.  A power of two scales the operands of both products exactly,
    so the results are those for 2^12 dh, up to one rounding of each, whose step does not fall below 2^-24."""
    r = _randn(27)
    x, w, b = (r(M, C) * 8).half(), (r(2 * F, C) * 0.3).half(), (r(2 * F) * 0.3).half() if bias else None
    small = (r(M, F) * 2.0 ** -19).half()
    big = (small.double() * 4096).half()
    assert torch.equal(big.double(), small.double() * 4096) and float(small.abs().max()) < 2.0 ** -14
    for name, s, t in zip(('dx', 'dw', 'db'), _gated_gradients(x, w, b, act, small), _gated_gradients(x, w, b, act, big)):
        if s is None:
            continue
        s, t = s.double() * 4096, t.double()
        assert bool(((s - t).abs() <= 2 * 2.0 ** -11 * t.abs() * 1.01 + 4096 * 2.0 ** -25).all()), name
    # and dW, which sums many rows, is as near the exact result as one rounding of its terms and one of itself leave it
    exact = gated64(x, w, b, act, small)[2][0]
    err = (_gated_gradients(x, w, b, act, small)[1].double() - exact).norm()
    assert float(err) <= 1.5 * float((exact.half().double() - exact).norm())


def test_large_fp16_gradients_stay_finite():
    """dh u act' beyond 65504 at one place, dx and dW within the range: the sums are what the formula says.  The rounding of that one term, at
    most 2^-11 of it, is common to a whole row of dx and of dW, whose own roundings are 0.42 of that in the mean (a relative error uniform in
    +- 2^-11 m^-1, m uniform in the binade): sqrt(1 + 0.42^-2) = 2.6; 2.75 with the scatter."""
    from focalformer3d_amd import ops
    M, C, F = 70, 48, 64
    r = _randn(28)
    x, w, dh = (r(M, C) * 0.05).half(), (r(2 * F, C) * 0.03).half(), (r(M, F) * 0.1).half()
    b = torch.full((2 * F,), 6.0, device='cuda', dtype=torch.half)
    dh[5, 7] = 30000.0                                   # times u = 6: 1.8e5
    want = gated64(x, w, b, 'silu', dh)
    got = (ops.gated_linear(x, w, b), *ops.gated_linear_bwd(x, w, b, 'silu', dh))
    assert float(want[1][0].abs().max()) < 65504 and float(want[2][0].abs().max()) < 65504
    for name, t, (value, _) in list(zip(('h', 'dx', 'dw'), got, want)):
        assert bool(t.isfinite().all()), name
        assert float((t.double() - value).norm()) <= 2.75 * float((value.half().double() - value).norm()), name
    rows = torch.arange(M, device='cuda') != 5           # and the other rows keep their digits
    e = want[1][0][rows]
    assert float((got[1][rows].double() - e).norm()) <= 1.5 * float((e.half().double() - e).norm())


def test_infinite_fp16_gradient_stays_in_its_row():
    from focalformer3d_amd import ops
    r = _randn(29)
    x, w, dh = r(70, 40).half(), (r(64, 40) * 0.1).half(), (r(70, 32) * 0.1).half()
    want = ops.gated_linear_bwd(x, w, None, 'silu', dh)[0]
    for bad in (float('inf'), float('nan')):
        d2 = dh.clone()
        d2[9, 3] = bad
        got = ops.gated_linear_bwd(x, w, None, 'silu', d2)[0]
        keep = torch.arange(70, device='cuda') != 9
        assert not bool(got[9].isfinite().any())
        # (the scale of the operands may be another power of two)
        assert bool(((got[keep].double() - want[keep].double()).abs() <= 2.0 ** -10 * want[keep].double().abs() + 2.0 ** -24).all())


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
def test_gated_gradients_without_signal(dtype):
    """A gradient of zeros, and one that underflows in every product."""
    from focalformer3d_amd import ops
    r = _randn(30)
    x, w, b = r(40, 24).to(DT[dtype]), r(32, 24).to(DT[dtype]), r(32).to(DT[dtype])
    for t in ops.gated_linear_bwd(x, w, b, 'silu', torch.zeros(40, 16, device='cuda', dtype=DT[dtype])):
        assert not t.any()
    for t in ops.gated_linear_bwd(torch.zeros_like(x), w, b * 0, 'silu', torch.ones(40, 16, device='cuda', dtype=DT[dtype])):
        assert not t.any()


def test_fp16_gradients_in_a_graph():
    """Replays over gradients of very different sizes, each against the eager call."""
    from focalformer3d_amd import ops
    r = _randn(31)
    x, w, b, dh = r(500, 64).half(), (r(96, 64) * 0.1).half(), r(96).half(), r(500, 48).half()
    ops.gated_linear_bwd(x, w, b, 'gelu', dh)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.gated_linear_bwd(x, w, b, 'gelu', dh)
    for f in (1.0, 2.0 ** -14, 1000.0, 0.0, 2.0 ** -6):
        dh.copy_((r(500, 48) * f).half())
        g.replay()
        want = ops.gated_linear_bwd(x, w, b, 'gelu', dh)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


# ------------------------------------------------------------------------------------------------ batches
@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
def test_accuracy_does_not_depend_on_the_batch(dtype):
    """64 tokens of 16 heads of 64 columns, alone and as one of 512 sequences: the error of its gradients stays that of one rounding (1.3: with
    the scatter of a norm of some thousand errors)."""
    from focalformer3d_amd import ops
    dt, B, N, H, d = DT[dtype], 512, 64, 16, 64
    r = _randn(32, dt)
    q, k, v, lam, dout = r(B, N, H * 2 * d), r(B, N, H * 2 * d), r(B, N, H * 2 * d), r(H).clamp(-1, 1), r(B, N, H * 2 * d)
    n = 2
    want = diff_attention64(q[:n], k[:n], v[:n], lam, H, H, blocked_pairs(n, N, N, None, None, False, 'cuda'), None, dout[:n])
    for part in (n, B):
        a = [t[:part] for t in (q, k, v)]
        saved = ops.diff_attention_train_fwd(*a, lam, H)
        got = ops.diff_attention_bwd(*a, lam, H, *saved, dout[:part])
        for name, t, (exact, _) in zip(('dq', 'dk', 'dv'), got, want[1:]):
            one = (exact.to(dt).double() - exact).norm()
            assert float((t[:n].double() - exact).norm() / one) <= 1.3, (part, name)


# ------------------------------------------------------------------------------------------------ long caches
@pytest.mark.parametrize('Nq,H,Nk', [(1, 2, 120000), (600, 8, 40000), (4500, 8, 20000)])
def test_fp16_weights_of_many_faint_keys(Nq, H, Nk):
    """Tens of thousands of keys have 10.45 * 2^-24 of the largest weight each, between two of fp16's smallest numbers, and values that make their
    sum count.  The three sizes are slices of the keys, blocks of 32 and blocks of 128 rows.  With weights kept to 2^-11 the output is off
    by a rounding of the weights and its own, and all terms are of one sign: 3 * 2^-11 of it with the fp32 sums."""
    from focalformer3d_amd import ops
    d, top = 8, 1829 / 128                               # exp(-top) = 10.448 * 2^-24; top and all else is exact in fp16
    q = torch.zeros(1, Nq, H * 2 * d, device='cuda', dtype=torch.half)
    k, v = torch.zeros(1, Nk, 2 * d, device='cuda', dtype=torch.half), torch.full((1, Nk, 2 * d), 2.0, device='cuda', dtype=torch.half)
    q[..., ::d], k[0, 0, ::d], v[0, 0] = 1.0, top, 0.25
    lam = torch.zeros(H, device='cuda', dtype=torch.half)
    faint = (Nk - 1) * math.exp(-top)
    want = (0.25 + 2.0 * faint) / (1.0 + faint)
    out = ops.diff_attention(q, k, v, lam, H, kv_heads=1, scale=1.0)
    assert float((out.double() - want).abs().max()) <= 3 * 2.0 ** -11 * want
    saved = ops.diff_attention_train_fwd(q, k, v, lam, H, kv_heads=1, scale=1.0)
    assert torch.equal(saved[0], out)
    assert float((saved[1].double() - want).abs().max()) <= 3 * 2.0 ** -11 * want
