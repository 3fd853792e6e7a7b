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


def test_rows_of_their_own():
    x = torch.zeros(6, 8, 128, dtype=torch.float16)
    for t in (x, x[1:], x[:, 2:6], x[::2], x.transpose(0, 1), x[:1], x[:, :1], x[:, :1].expand(6, 1, 128), x[:0],
              x.view(2, 3, 8, 128), x.view(2, 3, 8, 128).permute(2, 0, 1, 3), x[..., :64],
              x.as_strided((2, 2, 2, 64), (256, 64, 1024, 1)), x.as_strided((1, 4, 128), (8, 128, 1))):
        assert ops.writable_rows(t), t.stride()
    for size, stride in (((4, 8, 128), (8, 128, 1)),      # rows that slide over one another by 8 elements
                         ((4, 8, 128), (1016, 128, 1)),   # a row's last head is the next row's first, but for 8
                         ((4, 8, 128), (128, 128, 1)), ((4, 8, 128), (1024, 120, 1)), ((4, 8, 128), (0, 128, 1)),
                         ((4, 8, 128), (1024, 0, 1)), ((2, 3, 4, 64), (128, 64, 256, 1)), ((4, 2, 128), (64, 512, 1))):
        assert not ops.writable_rows(x.as_strided(size, stride)), stride
    assert not ops.writable_rows(x[..., 4:68]) and not ops.writable_rows(x[..., ::2])


def test_outputs_apart():
    x = torch.zeros(6, 8, 128, dtype=torch.float16)
    y = torch.zeros(6, 2, 8, 64, dtype=torch.float16)
    for a, b in ((x, torch.zeros_like(x)), (x[:3], x[3:]), (x[:, :4], x[:, 4:]), (x[:, 4:], x[:, :4]), (x[::2], x[1::2]),
                 (x[..., :64], x[..., 64:]), (y[:, 0], y[:, 1]), (x[:0], x[:0]), (x[:, ::2], x[:, 1::2])):
        assert ops.writable_rows(a) and ops.writable_rows(b) and ops.apart(a, b) and ops.apart(b, a)
    for a, b in ((x, x), (x[:3], x[2:5]), (x[:, :4], x[:, 3:7]), (x[..., :64], x[..., 8:72]), (x[:, :4], x[:, :4]),
                 (x[:4, :4], x.view(-1)[64:].as_strided((4, 4, 128), (512, 128, 1)))):
        assert not ops.apart(a, b) and not ops.apart(b, a)


def test_autograd_follows_tensors_only():
    x = torch.zeros(3)
    assert not ops.autograd_follows(None, x, 5, [x]) and ops.autograd_follows(None, 5, x.clone().requires_grad_())
    with torch.no_grad():
        assert not ops.autograd_follows(x.clone().requires_grad_())
