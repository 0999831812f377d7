"""Differential attention on the GPU, forward and backward, against the definition in fp64 with bounds that count the roundings."""
import pytest
import torch

from tests.operators_util import assert_within, blocked_pairs, diff_attention64

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _inputs(B, Nq, Nk, H, G, d, dt, seed=0, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    return ((r(B, Nq, H * 2 * d) * scale).to(dt), (r(B, Nk, G * 2 * d) * scale).to(dt), r(B, Nk, G * 2 * d).to(dt),
            (r(H) * 0.7).to(dt), r(B, Nq, H * 2 * d).to(dt))


def _check(q, k, v, lam, dout, H, G, mask=None, kv_lens=None, causal=False, scale=None):
    from focalformer3d_amd import ops
    from focalformer3d_amd.autograd import differential_attention
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    kw = dict(kv_heads=G, mask=mask, kv_lens=kv_lens, causal=causal, scale=scale)
    out = differential_attention(*leaves, H, **kw)
    got = (out, *torch.autograd.grad(out, leaves, dout))
    blocked = blocked_pairs(q.shape[0], q.shape[1], k.shape[1], mask, kv_lens, causal, q.device)
    for name, t, want in zip(('out', 'dq', 'dk', 'dv', 'dlam'), got, diff_attention64(q, k, v, lam, H, G, blocked, scale, dout)):
        assert t.dtype == q.dtype
        assert_within(t, want, name)
    assert torch.equal(ops.diff_attention(q, k, v, lam, H, **kw), out)
    return got


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 37, 2, 1, 16), (1, 33, 31, 2, 2, 8), (2, 64, 64, 2, 2, 16), (1, 130, 65, 4, 2, 32), (2, 129, 200, 3, 1, 64),
          (1, 5, 700, 6, 2, 32), (3, 257, 96, 2, 1, 16), (1, 300, 300, 16, 16, 8)]


@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('causal', [False, True])
def test_diff_attention(shape, dtype, causal):
    B, Nq, Nk, H, G, d = shape
    _check(*_inputs(B, Nq, Nk, H, G, d, DT[dtype]), H, G, causal=causal)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('d', [8, 16, 32, 64])
def test_diff_attention_masks_and_lengths(dtype, d):
    """Masks of each broadcast form and alignment, rows that the mask or the length leaves empty, a sequence of length zero, lengths
    outside the tensor, all of them together; keys behind a length hold NaN."""
    B, Nq, Nk, H, G = 3, 70, 93, 4, 2
    q, k, v, lam, dout = _inputs(B, Nq, Nk, H, G, d, DT[dtype], 1)
    g = torch.Generator(device='cuda').manual_seed(2)
    mask = torch.rand(B, Nq, Nk, generator=g, device='cuda') < 0.4
    mask[:, 3::7] = True
    mask[1, :, 10:50] = True
    _check(q, k, v, lam, dout, H, G, mask=mask)
    _check(q, k, v, lam, dout, H, G, mask=mask[0])
    _check(q, k, v, lam, dout, H, G, mask=mask[:1].to(torch.uint8) * 7)
    wide = torch.zeros(B, Nq, 101, dtype=torch.bool, device='cuda')
    wide[:, :, 3:96] = mask
    _check(q, k, v, lam, dout, H, G, mask=wide[:, :, 3:96])
    lens = torch.tensor([0, 41, 200], dtype=torch.int32, device='cuda')
    k[1, 41:], v[1, 41:] = float('nan'), float('inf')
    k[0], v[0] = float('nan'), float('nan')
    got = _check(q, k, v, lam, dout, H, G, kv_lens=lens)
    assert not got[0][0].any() and not got[1][0].any() and not got[2][0].any() and not got[3][1, 41:].any()
    _check(q, k, v, lam, dout, H, G, mask=mask, kv_lens=lens, causal=True)
    _check(q, k, v, lam, dout, H, G, mask=torch.ones_like(mask), kv_lens=lens)
    _check(q, k, v, lam, dout, H, G, kv_lens=torch.tensor([-5, 1, 92], dtype=torch.int32, device='cuda'))


@pytest.mark.parametrize('B,Nq,H,G,d', [(2, 100, 6, 2, 16), (1, 45, 5, 1, 64), (1, 333, 4, 4, 32), (2, 70, 8, 1, 8)])
@pytest.mark.parametrize('dtype', ['f32', 'f16'])
def test_diff_attention_mask_words(dtype, B, Nq, H, G, d):
    """Tiles of 32 packed rows that begin anywhere in a word of 32 queries: 3, 5, 1 and 8 heads per key head."""
    q, k, v, lam, dout = _inputs(B, Nq, 131, H, G, d, DT[dtype], 19)
    mask = torch.rand(B, Nq, 131, generator=torch.Generator(device='cuda').manual_seed(20), device='cuda') < 0.5
    _check(q, k, v, lam, dout, H, G, mask=mask)
    _check(q, k, v, lam, dout, H, G, mask=mask[0], causal=True)


# few rows over long keys: slices that a second kernel joins, some of them without a key
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('B,Nq,Nk,H,G,d', [(1, 1, 5000, 1, 1, 64), (2, 1, 3001, 8, 2, 32), (3, 7, 1024, 4, 4, 16), (1, 2, 2050, 16, 1, 8)])
def test_diff_attention_single_tokens(dtype, B, Nq, Nk, H, G, d):
    q, k, v, lam, dout = _inputs(B, Nq, Nk, H, G, d, DT[dtype], 3)
    _check(q, k, v, lam, dout, H, G)
    lens = torch.tensor([1, 700, 0], dtype=torch.int32, device='cuda')[:B]
    _check(q, k, v, lam, dout, H, G, kv_lens=lens)
    _check(q, k, v, lam, dout, H, G, causal=True, kv_lens=torch.full((B,), Nk - 3, dtype=torch.int32, device='cuda'))


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_diff_attention_four_wave_blocks(dtype):
    """Enough rows for the wide blocks, shared heads, tiles cut by the causal order."""
    _check(*_inputs(2, 2100, 130, 16, 16, 16, DT[dtype], 4), 16, 16)
    _check(*_inputs(1, 1090, 1090, 32, 8, 32, DT[dtype], 5), 32, 8, causal=True)
    _check(*_inputs(1, 2049, 300, 16, 16, 64, DT[dtype], 6), 16, 16)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_diff_attention_layouts(dtype):
    """Column blocks of one projection, a broadcast batch, misaligned and unusual strides, an expanded gradient."""
    from focalformer3d_amd import ops
    from focalformer3d_amd.autograd import differential_attention
    dt, H, d = DT[dtype], 2, 16
    q, k, v, lam, dout = _inputs(2, 50, 50, H, H, d, dt, 7)
    want = ops.diff_attention(q, k, v, lam, H)
    C = H * 2 * d
    for pad in (0, 8, 3):
        fused = torch.zeros(2, 50, 3 * C + pad, dtype=dt, device='cuda')
        fused[..., pad:pad + C], fused[..., pad + C:pad + 2 * C], fused[..., pad + 2 * C:] = q, k, v
        parts = fused[..., pad:pad + C], fused[..., pad + C:pad + 2 * C], fused[..., pad + 2 * C:]
        assert torch.equal(ops.diff_attention(*parts, lam, H), want)
        _check(*parts, lam, fused[..., pad:pad + C], H, H)
    t = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(ops.diff_attention(*t, lam, H), want)
    _check(q[:1].expand(2, -1, -1), k, v, lam, dout, H, H)
    _check(q, k[:1].expand(2, -1, -1), v[:1].expand(2, -1, -1), lam, dout, H, H)
    leaf = q.clone().requires_grad_(True)
    differential_attention(leaf, k, v, lam, H).sum().backward()
    ref = diff_attention64(q, k, v, lam, H, H, blocked_pairs(2, 50, 50, None, None, False, 'cuda'), None, torch.ones_like(q))
    assert_within(leaf.grad, ref[1], 'dq')


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_diff_attention_ranges(dtype):
    """Scores of a thousand, a very small and a large gradient, equal maps that cancel, lam of zero."""
    dt, H = DT[dtype], 2
    q, k, v, lam, dout = _inputs(1, 80, 90, H, H, 32, dt, 8, scale=12.0)
    _check(q, k, v, lam, dout, H, H)
    q, k, v, lam, dout = _inputs(1, 80, 90, H, H, 32, dt, 9)
    for f in (1e-3, 100.0):
        _check(q, k, v, lam, (dout.float() * f).to(dt), H, H)
    _check(q, k, v, torch.zeros_like(lam), dout, H, H)
    _check(q, k, v, lam, dout, H, H, scale=0.01)
    same = q.view(1, 80, H, 2, 32)[:, :, :, :1].expand(-1, -1, -1, 2, -1).reshape(q.shape)
    ks = k.view(1, 90, H, 2, 32)[:, :, :, :1].expand(-1, -1, -1, 2, -1).reshape(k.shape)
    _check(same, ks, v, torch.ones_like(lam), dout, H, H)


def test_diff_attention_small_fp16_gradients_keep_their_digits():
    """Gradients of 2^-16: dS lies below fp16's normal numbers, and dq, dk keep the relative accuracy of the ordinary case."""
    q, k, v, lam, dout = _inputs(1, 200, 600, 2, 2, 32, torch.float16, 10)
    from focalformer3d_amd import ops
    saved = ops.diff_attention_train_fwd(q, k, v, lam, 2)
    big = ops.diff_attention_bwd(q, k * 64, v, lam, 2, *ops.diff_attention_train_fwd(q, k * 64, v, lam, 2, scale=2.0 ** -6), dout, scale=2.0 ** -6)
    small = ops.diff_attention_bwd(q, k * 64, v, lam, 2, *ops.diff_attention_train_fwd(q, k * 64, v, lam, 2, scale=2.0 ** -6), dout * 2.0 ** -10, scale=2.0 ** -6)
    # a power of two scales every step exactly, up to the rounding of dout and of results below the normal numbers
    ref = big[0].double() * 2.0 ** -10
    assert float((small[0].double() - ref).norm() / ref.norm()) < 4e-3
    assert saved[0].isfinite().all()


def test_diff_attention_wanted_gradients_only():
    from focalformer3d_amd import ops
    q, k, v, lam, dout = _inputs(2, 40, 50, 2, 2, 16, torch.float32, 11)
    saved = ops.diff_attention_train_fwd(q, k, v, lam, 2)
    full = ops.diff_attention_bwd(q, k, v, lam, 2, *saved, dout)
    for i in range(4):
        got = ops.diff_attention_bwd(q, k, v, lam, 2, *saved, dout, want=tuple(j == i for j in range(4)))
        assert all((t is None) == (j != i) for j, t in enumerate(got)) and torch.equal(got[i], full[i])


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('Nq,H,G,d', [(1, 12, 12, 16), (5, 4, 2, 64), (40, 2, 1, 32)])
def test_diff_attention_one_key(dtype, Nq, H, G, d):
    """Its weight is 1 whatever the score: no gradient reaches q and k, and out = (1 - lam) v."""
    got = _check(*_inputs(3, Nq, 1, H, G, d, DT[dtype], 33), H, G)
    assert float(got[1].abs().max()) == 0.0 and float(got[2].abs().max()) == 0.0
    lens = torch.tensor([1, 0, 1], dtype=torch.int32, device='cuda')
    got = _check(*_inputs(3, Nq, 1, H, G, d, DT[dtype], 34), H, G, kv_lens=lens)
    assert float(got[1].abs().max()) == 0.0 and float(got[2].abs().max()) == 0.0 and float(got[0].detach()[1].abs().max()) == 0.0


def test_diff_attention_empty():
    from focalformer3d_amd import ops
    q, k, v, lam, dout = _inputs(2, 5, 6, 2, 2, 16, torch.float32, 12)
    assert ops.diff_attention(q[:0], k[:0], v[:0], lam, 2).shape == (0, 5, 64)
    assert ops.diff_attention(q[:, :0], k, v, lam, 2).shape == (2, 0, 64)
    out = ops.diff_attention_train_fwd(q, k[:, :0], v[:, :0], lam, 2)
    assert not out[0].any()
    grads = ops.diff_attention_bwd(q, k[:, :0], v[:, :0], lam, 2, *out, dout)
    assert not grads[0].any() and grads[1].shape == (2, 0, 64) and not grads[3].any()


def test_diff_attention_against_differences():
    """Directional derivatives of <out, dout> against differences of the fp64 definition."""
    from focalformer3d_amd import ops
    H, G, d = 4, 2, 8
    q, k, v, lam, dout = _inputs(1, 9, 11, H, G, d, torch.float32, 13)
    bl = blocked_pairs(1, 9, 11, None, None, True, 'cuda')
    grads = ops.diff_attention_bwd(q, k, v, lam, H, *ops.diff_attention_train_fwd(q, k, v, lam, H, G, causal=True), dout, kv_heads=G, causal=True)
    bounds = diff_attention64(q, k, v, lam, H, G, bl, None, dout)[1:]

    def f(args):
        q, k, v, lam = args
        qm = q.view(9, H, 2, d).permute(1, 2, 0, 3)
        km = k.view(11, G, 2, d).permute(1, 2, 0, 3).repeat_interleave(2, 0)
        vm = v.view(11, G, 2 * d).transpose(0, 1).repeat_interleave(2, 0)
        p = torch.softmax((qm @ km.transpose(-1, -2) / d ** 0.5).masked_fill(bl[0], -1e300), -1)
        return float((((p[:, 0] - lam[:, None, None] * p[:, 1]) @ vm).transpose(0, 1).reshape(1, 9, -1) * dout.double()).sum())
    args = [t.double() for t in (q, k, v, lam)]
    for i in range(4):
        x = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
        up, dn = list(args), list(args)
        up[i], dn[i] = args[i] + 1e-5 * x, args[i] - 1e-5 * x
        slope = (f(up) - f(dn)) / 2e-5
        assert abs(float((grads[i].double() * x).sum()) - slope) <= float((bounds[i][1] * x.abs()).sum()) + 1e-7 * (1 + abs(slope))


def test_diff_attention_deterministic_stream_graph():
    from focalformer3d_amd import ops
    H, G, d = 8, 2, 32
    a = _inputs(2, 200, 900, H, G, d, torch.bfloat16, 14)
    lens = torch.tensor([900, 333], dtype=torch.int32, device='cuda')

    def both(q, k, v, lam, dout):
        saved = ops.diff_attention_train_fwd(q, k, v, lam, H, G, kv_lens=lens)
        return (saved[0], *ops.diff_attention_bwd(q, k, v, lam, H, *saved, dout, kv_heads=G, kv_lens=lens), ops.diff_attention(q[:, :1], k, v, lam, H, G))
    want = both(*a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(*a)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    st = [t.clone() for t in a]
    graphs = []
    for _ in range(2):                                                  # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both(*st)
        graphs.append((g, out))
    for seed in (15, 16, 17):
        new = _inputs(2, 200, 900, H, G, d, torch.bfloat16, seed)
        for x, y in zip(st, new):
            x.copy_(y)
        for g, out in graphs:
            g.replay()
        ref = both(*new)
        torch.cuda.synchronize()
        for g, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, ref))


def test_refusals_on_device():
    from focalformer3d_amd import ops
    q, k, v, lam, dout = _inputs(2, 5, 6, 2, 2, 16, torch.float32, 18)
    ok = dict(q=q, k=k, v=v, lam=lam, heads=2)
    for bad in (dict(q=q.double()), dict(k=k.bfloat16()), dict(v=v[:, :5]), dict(lam=lam[:1]), dict(lam=lam.cpu()), dict(q=q[..., :60]), dict(q=q[0]),
                dict(mask=torch.zeros(5, 5, device='cuda', dtype=torch.bool)), dict(mask=torch.zeros(5, 6, device='cuda')),
                dict(mask=torch.zeros(3, 5, 6, device='cuda', dtype=torch.bool)), dict(mask=torch.zeros(5, 6, dtype=torch.bool)),
                dict(kv_lens=torch.zeros(2, device='cuda')), dict(kv_lens=torch.zeros(3, dtype=torch.int32, device='cuda')),
                dict(kv_lens=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(RuntimeError):
            ops.diff_attention(**{**ok, **bad})
    for bad in (dict(kv_heads=3), dict(heads=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf'))):
        with pytest.raises(ValueError):
            ops.diff_attention(**{**ok, **bad})
    saved = ops.diff_attention_train_fwd(q, k, v, lam, 2)
    with pytest.raises(RuntimeError):
        ops.diff_attention_bwd(q, k, v, lam, 2, *saved, dout[:, :4])
    for i, bad in ((0, saved[0][:, :4]), (0, saved[0].half()), (1, saved[1].half()), (1, saved[1].transpose(0, 1)), (2, saved[2][:, :1]), (2, saved[2].cpu())):
        with pytest.raises(RuntimeError):
            ops.diff_attention_bwd(q, k, v, lam, 2, *saved[:i], bad, *saved[i + 1:], dout)
