"""The rows that the calls for many sequences read and write: what is taken as it is, copied or refused (host only)."""
import pytest
import torch

from innerq_amd import ops


def readable(t):
    r = ops.readable_rows(t)
    assert torch.equal(r, t) and r.stride(-1) == 1 and r.data_ptr() % 16 == 0 and not any(s % 8 for s in r.stride()[:-1])
    return r


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_are_readable(dtype):
    x = torch.randn(5, 4100).to(dtype)[:, :4096].view(5, 32, 128)
    assert x.data_ptr() % 16 == 0
    for t in (x, x[:1], x[1:2], x[:, :2], x[1:3, 1:2]):  # odd row strides, also where a dim of size 1 has one
        assert readable(t) is not t
    flat = torch.randn(4 + 3 * 2 * 64).to(dtype)
    assert flat[4:].is_contiguous() and readable(flat[4:].view(3, 2, 64)) is not flat  # contiguous, 8 bytes off
    y = torch.randn(5, 6, 64).to(dtype)
    for t in (y, y[1:], y[:, 2:4], y.transpose(0, 1), y[:1].expand(5, 6, 64)):
        assert readable(t) is t
    for t in (y[..., ::2], y.permute(0, 2, 1)[:, :, :1].expand(5, 64, 64)):
        assert readable(t) is not t


def test_no_rows():
    assert ops.readable_rows(torch.zeros(0, 4, 64)).shape == (0, 4, 64)
