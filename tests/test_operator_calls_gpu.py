"""Calls of the operators in three types that their documentation allows: rows of unusual strides."""
import pytest
import torch

from tests.operators_util import assert_within, gated64

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
