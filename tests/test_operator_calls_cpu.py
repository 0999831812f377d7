"""Host-side parts of the operators in three types that need no GPU."""
import pytest
import torch

from focalformer3d_amd import ops


ROWS = [torch.randn(1, 30, 8)[:, -1], torch.randn(8, 1).t(), torch.randn(1).expand(1, 1), torch.randn(1).expand(1, 8),
        torch.randn((1 << 20) + 9).as_strided((1, 8), ((1 << 20) + 1, 1)), torch.randn(5, 8), torch.randn(5, 16)[:, 4:12], torch.randn(8, 5).t(),
        torch.randn(5, 16)[:, ::2], torch.randn(1).expand(5, 1), torch.randn(8).expand(5, 8), torch.randn(2, 1 << 20)[:, :8], torch.randn(1, 16)[:, ::2],
        torch.randn(5, 3)[:, :1]]


@pytest.mark.parametrize('i', range(len(ROWS)))
def test_rows_have_a_stride_that_holds(i):
    """Whatever the strides of the view, the tensor that goes to the kernel has dense rows of a stride that it can take; one row is not copied."""
    x = ROWS[i]
    M, n = x.shape
    args = ops._gated_args(x, torch.zeros(4, n), None, 'silu')
    again = ops._gated_again((x, torch.zeros(4, n), None), (2, n, 0, 0, 0, x.shape))
    t, row = ops._whole_rows(x)
    assert t.stride() == (row, 1) and row == n and (t.data_ptr() == x.data_ptr()) == (M == 1 and (x.stride(1) == 1 or n == 1))
    for t in (t, args[0], again[0]):
        assert torch.equal(t, x) and t.stride(1) == 1 and n <= t.stride(0) < 1 << 20
    assert args[5] == again[5] == (3 if n % 4 else (1 if args[0].stride(0) % 4 or args[0].data_ptr() % 16 else 0) | args[5] & 2)


def test_once_differentiable_backward_refuses_a_second_derivative():
    """Also where the incoming gradient is a constant; the first derivative is the same with and without a graph of the gradients."""
    from focalformer3d_amd.autograd import _once

    class Square(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, y):
            ctx.save_for_backward(x)
            return x * x, 2 * y

        @staticmethod
        @_once
        def backward(ctx, g, h):
            return 2 * ctx.saved_tensors[0] * g, None if h is None else 2 * h
    x, y = torch.randn(3, requires_grad=True), torch.randn(3, requires_grad=True)
    assert torch.equal(torch.autograd.grad(Square.apply(x, y)[0].sum(), x)[0], 2 * x)
    g, = torch.autograd.grad(Square.apply(x, y)[0].sum(), x, create_graph=True)
    assert torch.equal(g, 2 * x)
    with pytest.raises(RuntimeError, match='twice'):
        g.sum().backward()
