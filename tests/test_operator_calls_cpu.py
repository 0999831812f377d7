"""Host-side parts of the operators in three types that need no GPU."""
import pytest
import torch

from focalformer3d_amd import ops


@pytest.mark.parametrize('x,copied', [
    (torch.randn(1, 30, 8)[:, -1], False), (torch.randn(8, 1).t(), False), (torch.randn(1).expand(1, 1), False), (torch.randn(1).expand(1, 8), True),
    (torch.randn(9).as_strided((1, 8), (300, 1)), False), (torch.randn(5, 8), False), (torch.randn(5, 16)[:, 4:12], False), (torch.randn(8, 5).t(), True),
    (torch.randn(5, 16)[:, ::2], True), (torch.randn(1).expand(5, 1), True), (torch.randn(8).expand(5, 8), True), (torch.randn(5, 300)[:, :8], True),
    (torch.randn(1, 16)[:, ::2], True), (torch.randn(5, 3)[:, :1], False)])
def test_rows_have_a_stride_that_holds(x, copied):
    """Whatever the strides of the view, the row stride that goes to the kernel is that of the tensor that goes with it."""
    t, row = ops._whole_rows(x, 256)
    M, n = x.shape
    assert torch.equal(t, x) and t.stride() == (row, 1) and n <= row < 256
    assert (t.data_ptr() != x.data_ptr()) == copied
    pack = ops._gated_args(x, torch.zeros(4, n), None, 'silu')
    assert pack[0].stride(0) >= n and pack[0].stride(0) < 1 << 20
