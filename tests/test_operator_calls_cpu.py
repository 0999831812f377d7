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
