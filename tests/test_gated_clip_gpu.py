"""Gated projection and gradient clipping on the GPU against fp64 definitions, with bounds that count the roundings."""
import pytest
import torch

from tests.operators_util import E32, U, assert_within, gated64

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _inputs(M, C, F, dt, bias, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    return (r(M, C).to(dt), (r(2 * F, C) * C ** -0.5).to(dt), (r(2 * F) * 0.3).to(dt) if bias else None, (r(M, F) * 0.1).to(dt))


def _check(x, w, b, act, dh):
    from focalformer3d_amd.autograd import gated_linear
    leaves = [t.detach().requires_grad_(True) for t in (x, w) + ((b,) if b is not None else ())]
    h = gated_linear(leaves[0], leaves[1], leaves[2] if b is not None else None, act)
    got = (h, *torch.autograd.grad(h, leaves, dh))
    for name, t, want in zip(('h', 'dx', 'dw', 'db'), got, gated64(x, w, b, act, dh)):
        assert t.dtype == x.dtype
        assert_within(t, want, name)
    return got


# one row, sizes below, at and just past the tiles, widths that are no multiple of a granule
@pytest.mark.parametrize('M,C,F', [(1, 1, 1), (1, 256, 1024), (5, 8, 3), (33, 40, 17), (64, 64, 64), (65, 72, 65), (129, 130, 129),
                                   (600, 256, 1024), (257, 200, 530), (1100, 64, 31), (2100, 24, 40)])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('act,bias', [('silu', False), ('gelu', True)])
def test_gated_linear(M, C, F, dtype, act, bias):
    x, w, b, dh = _inputs(M, C, F, DT[dtype], bias)
    _check(x, w, b, act, dh)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('act', ['relu', 'sigmoid'])
def test_gated_linear_other_activations(dtype, act):
    _check(*_args(_inputs(70, 48, 50, DT[dtype], True, 3), act))


def _args(t, act):
    return t[0], t[1], t[2], act, t[3]


# large tiles of every operand order: enough of them for the widest tile
@pytest.mark.parametrize('M,C,F', [(4096, 512, 1808), (3001, 1032, 1300)])
@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32'])
def test_gated_linear_large(M, C, F, dtype):
    x, w, b, dh = _inputs(M, C, F, DT[dtype], True, 5)
    _check(x, w, b, 'silu', dh)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_gated_linear_layouts(dtype):
    """Leading dimensions, a column block of a wider matrix, a base that is not 16-byte aligned, a broadcast gradient."""
    from focalformer3d_amd import ops
    from focalformer3d_amd.autograd import gated_linear
    dt = DT[dtype]
    x, w, b, dh = _inputs(60, 96, 40, dt, True, 7)
    wide = torch.zeros(60, 200, dtype=dt, device='cuda')
    for at in (0, 8, 51):
        wide[:, at:at + 96] = x
        _check(wide[:, at:at + 96], w, b, 'silu', dh)
    want = ops.gated_linear(x, w, b)
    assert torch.equal(ops.gated_linear(x.view(3, 4, 5, 96), w, b).view(60, 40), want)
    off = torch.empty(w.numel() + 1, dtype=dt, device='cuda')[1:].view(w.shape).copy_(w)
    assert torch.equal(ops.gated_linear(x, off, b), want)
    assert torch.equal(ops.gated_linear(x, w.t().contiguous().t(), b), want)
    leaf = x.clone().requires_grad_(True)
    gated_linear(leaf, w, b).sum().backward()                          # an expanded gradient: every stride is 0
    assert_within(leaf.grad, gated64(x, w, b, 'silu', torch.ones_like(dh))[1], 'dx')


def test_gated_linear_empty_and_wanted_gradients_only():
    from focalformer3d_amd import ops
    from focalformer3d_amd.autograd import gated_linear
    x, w, b, dh = _inputs(40, 32, 24, torch.float32, True)
    assert ops.gated_linear(x[:0], w, b).shape == (0, 24)
    dx, dw, db = ops.gated_linear_bwd(x[:0], w, b, 'silu', dh[:0])
    assert dx.shape == (0, 32) and not dw.any() and not db.any()
    full = ops.gated_linear_bwd(x, w, b, 'silu', dh)
    for i in range(3):
        got = ops.gated_linear_bwd(x, w, b, 'silu', dh, tuple(j == i for j in range(3)))
        assert all((t is None) == (j != i) for j, t in enumerate(got)) and torch.equal(got[i], full[i])
    leaf = w.clone().requires_grad_(True)
    gated_linear(x, leaf, b).backward(dh)
    assert torch.equal(leaf.grad, full[1])


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_gated_linear_against_differences(dtype):
    """Directional derivatives of sum(h * c) in fp64 inputs' neighbourhood: f(x + e v) - f(x - e v) of the fp64 definition."""
    from focalformer3d_amd import ops
    x, w, b, dh = _inputs(17, 24, 10, DT[dtype], True, 11)
    grads = ops.gated_linear_bwd(x, w, b, 'silu', dh)
    bounds = gated64(x, w, b, 'silu', dh)[1:]
    f = lambda x, w, b: float((gated64(x, w, b, 'silu')[0][0] * dh.double()).sum())  # noqa: E731
    args = [t.double() for t in (x, w, b)]

    def at(i, e, v):
        a = list(args)
        a[i] = a[i] + e * v
        F, pre = w.shape[0] // 2, a[0] @ a[1].t() + a[2]
        return float((torch.nn.functional.silu(pre[:, :F]) * pre[:, F:] * dh.double()).sum())
    for i in range(3):
        v = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
        e = 1e-5
        slope = (at(i, e, v) - at(i, -e, v)) / (2 * e)
        got = float((grads[i].double() * v).sum())
        assert abs(got - slope) <= float((bounds[i][1] * v.abs()).sum()) + 1e-7 * (1 + abs(slope))


def test_gated_linear_is_deterministic_streams_and_graph():
    """The same bits on every run, on another stream, and from a captured forward + backward replayed on new inputs."""
    from focalformer3d_amd import ops
    x, w, b, dh = _inputs(1500, 128, 96, torch.bfloat16, True, 13)
    want = (ops.gated_linear(x, w, b), *ops.gated_linear_bwd(x, w, b, 'silu', dh))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = (ops.gated_linear(x, w, b), *ops.gated_linear_bwd(x, w, b, 'silu', dh))
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    sx, sdh = x.clone(), dh.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = (ops.gated_linear(sx, w, b), *ops.gated_linear_bwd(sx, w, b, 'silu', sdh))
    for seed in (20, 21, 22):
        x2, _, _, dh2 = _inputs(1500, 128, 96, torch.bfloat16, True, seed)
        sx.copy_(x2), sdh.copy_(dh2)
        g.replay()
        ref = (ops.gated_linear(x2, w, b), *ops.gated_linear_bwd(x2, w, b, 'silu', dh2))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ref))


def test_gated_linear_nan_stays_in_its_rows():
    from focalformer3d_amd import ops
    x, w, b, _ = _inputs(70, 40, 20, torch.float32, True)
    want = ops.gated_linear(x, w, b, 'relu')
    x[9, 3] = float('nan')
    got = ops.gated_linear(x, w, b, 'relu')
    assert bool(got[9].isnan().all())
    keep = torch.arange(70, device='cuda') != 9
    assert torch.equal(got[keep], want[keep])


# ------------------------------------------------------------------------------------------------ clipping
def _grads(sizes, dtypes, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return [torch.randn(*s, generator=g, device='cuda').mul_(1 + i % 3).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


SIZES = [(1,), (3, 5), (0, 7), (2048,), (2049, 3), (511, 129), (64, 64, 3, 3), (100001,)]


def _norm64(grads, kind):
    flat = torch.cat([t.double().reshape(-1) for t in grads])
    return float(torch.linalg.vector_norm(flat, kind))


@pytest.mark.parametrize('dtypes', [['f32'], ['bf16'], ['f16'], ['f32', 'bf16', 'f16']])
@pytest.mark.parametrize('kind', [2.0, 1.0, float('inf')])
@pytest.mark.parametrize('max_norm', [0.0, 0.5, 1e9])
def test_clip_grads(dtypes, kind, max_norm):
    """Norm to a rounding of fp32 (sums are fp64), every element to the roundings of the factor and its own; both in place and out."""
    from focalformer3d_amd import ops
    grads = _grads(SIZES, [DT[d] for d in dtypes])
    norm64 = _norm64(grads, kind)
    assert abs(float(ops.grad_norm(grads, kind)) - norm64) <= 2 * E32 * norm64
    coef = min(1.0, max_norm / (norm64 + 1e-6))
    out = [torch.full_like(t, float('nan')) for t in grads]
    mine = [t.clone() for t in grads]
    for norm in (ops.clip_grads(grads, max_norm, kind, out=out), ops.clip_grads(mine, max_norm, kind)):
        assert norm.dtype == torch.float32 and abs(float(norm) - norm64) <= 2 * E32 * norm64
    for t, o, m in zip(grads, out, mine):
        want = t.double() * coef
        # the factor: max_norm, the norm, the sum and the quotient are rounded to fp32; then the product to fp32 and to the type
        bound = want.abs() * (6 * E32 + U[t.dtype] * 1.01) + (2.0 ** -24 if t.dtype == torch.float16 else 2.0 ** -126)
        assert_within(o, (want, bound))
        assert torch.equal(o, m)
        if coef == 1.0:
            assert torch.equal(o, t)


def test_clip_grads_many_tensors_and_types():
    """More tensors than one launch takes, gradients converted on the way, tensors that are dense in another order of dimensions."""
    from focalformer3d_amd import ops
    grads = _grads([(7 + 13 * i,) for i in range(250)] + [(16, 8, 3, 3)], [torch.bfloat16])
    grads[-1] = grads[-1].contiguous(memory_format=torch.channels_last)
    out = [torch.empty_like(t, dtype=torch.float32) for t in grads]
    norm = ops.clip_grads(grads, 1.0, out=out)
    n64 = _norm64(grads, 2.0)
    assert abs(float(norm) - n64) <= 2 * E32 * n64
    for t, o in zip(grads, out):
        assert_within(o, (t.double() / (n64 + 1e-6), t.double().abs() / n64 * 6 * E32 + 2.0 ** -126))


def test_clip_grads_extremes():
    """Squares that overflow fp32, values that vanish when squared, infinities and NaN, misaligned bases."""
    from focalformer3d_amd import ops
    big = [torch.full((1000,), 1e30, device='cuda'), torch.full((10,), -1e30, device='cuda')]
    assert abs(float(ops.grad_norm(big)) / (1e30 * 1010 ** 0.5) - 1) < 4 * E32
    small = [torch.full((1000,), 1e-30, device='cuda')]
    assert abs(float(ops.grad_norm(small)) / (1e-30 * 1000 ** 0.5) - 1) < 4 * E32
    g = [torch.ones(300, device='cuda'), torch.ones(5, device='cuda')]
    g[1][2] = float('inf')
    for kind in (2.0, 1.0, float('inf')):
        assert float(ops.grad_norm(g, kind)) == float('inf')
    c = [t.clone() for t in g]
    ops.clip_grads(c, 1.0)
    assert not c[0].any() and bool(c[1][2].isnan()) and not c[1][:2].any()        # 1 / inf = 0, inf * 0 = NaN
    g[0][299] = float('nan')
    for kind in (2.0, 1.0, float('inf')):
        assert bool(ops.grad_norm(g, kind).isnan())
    ops.clip_grads(g, 1.0)
    assert all(bool(t.isnan().all()) for t in g)
    base = torch.randn(5000, device='cuda')
    odd = base[1:4998]
    want = odd.double() / float(odd.double().norm())
    ops.clip_grads([odd], 1.0)
    assert float((odd.double() - want).abs().max()) <= 8 * E32 * float(want.abs().max())


def test_clip_grads_graph_and_stream():
    from focalformer3d_amd import ops
    grads = _grads(SIZES, [torch.float32], 5)
    out = [torch.empty_like(t) for t in grads]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = ops.clip_grads(grads, 1.0, out=out)
    for seed in (6, 7, 8):
        for t, n in zip(grads, _grads(SIZES, [torch.float32], seed)):
            t.copy_(n)
        g.replay()
        ref = [torch.empty_like(t) for t in grads]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            n2 = ops.clip_grads(grads, 1.0, out=ref)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(out, ref))


def test_clip_grad_norm_of_parameters():
    """As torch.nn.utils.clip_grad_norm_: parameters without a gradient are skipped, one given twice counts once."""
    from focalformer3d_amd.training import clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(4, 5, device='cuda')) for _ in range(3)]
    ps[0].grad, ps[2].grad = torch.ones(4, 5, device='cuda'), torch.full((4, 5), 2.0, device='cuda')
    version = ps[0].grad._version
    n = clip_grad_norm_(iter(ps + ps[:1]), 5.0)
    assert abs(float(n) - 10.0) <= 1e-5 and ps[1].grad is None
    assert float((ps[0].grad - 0.5).abs().max()) < 1e-6 and float((ps[2].grad - 1.0).abs().max()) < 1e-6
    assert ps[0].grad._version > version
    ps[0].grad[0, 0] = float('inf')
    with pytest.raises(RuntimeError, match='not finite'):
        clip_grad_norm_(ps, 5.0, error_if_nonfinite=True)
    assert float((ps[2].grad - 1.0).abs().max()) < 1e-6


def test_refusals_on_device():
    from focalformer3d_amd import ops
    g = torch.ones(64, device='cuda')
    for bad in ([g, g], [g, g[:8]], [g[:40], g[39:]]):
        with pytest.raises(RuntimeError, match='share memory'):
            ops.clip_grads(bad, 1.0)
    h = torch.zeros(64, device='cuda')
    with pytest.raises(RuntimeError, match='share memory'):
        ops.clip_grads([g[:32], g[32:]], 1.0, out=[g[32:], h[:32]])
    with pytest.raises(RuntimeError, match='share memory'):
        ops.clip_grads([g[:32]], 1.0, out=[g[16:48]])
    assert bool((g == 1).all()) and not h.any()
    with pytest.raises(RuntimeError, match='without gaps'):
        ops.clip_grads([torch.ones(4, 8, device='cuda')[:, ::2]], 1.0)
    with pytest.raises(RuntimeError, match='out'):
        ops.clip_grads([g], 1.0, out=[h[:32]])
    with pytest.raises(RuntimeError, match='dense'):
        ops.grad_norm([g, torch.ones(3)])
    for bad in (-1.0, float('nan')):
        with pytest.raises(ValueError):
            ops.clip_grads([g], bad)
    x, w, b, dh = _inputs(4, 16, 8, torch.float32, True)
    for args in ((x.double(), w, b), (x, w.bfloat16(), b), (x, w[:15], b), (x, w, b[:8]), (x[:, :8], w, b), (x, w.cpu(), b)):
        with pytest.raises(RuntimeError):
            ops.gated_linear(*args)
    with pytest.raises(ValueError):
        ops.gated_linear(x, w, b, 'tanh')
    with pytest.raises(RuntimeError):
        ops.gated_linear_bwd(x, w, b, 'silu', dh[:, :4])
