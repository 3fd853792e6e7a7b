"""The C ABI of gathered weights takes what its limits allow (no GPU here: calls of no rows end behind their checks)."""
import pytest

from test_dropping_refusals import _diff_prompt, _prompt


@pytest.mark.parametrize("fn", [_prompt, _diff_prompt])
def test_head_strides(fn):
    """A head stride times Hq / H below 2^29, where Hq / H divides it (8) and where it does not (31, 3)."""
    for r in (8, 31, 3, 1, 512):
        most = (2 ** 29 - 1) // r // 8 * 8  # the largest that keeps rows on 16 bytes
        assert most * r < 2 ** 29 <= (most + 8) * r
        assert fn(N=0, Hq=8 * r, sq_h=most) == 0, r
        assert fn(N=0, Hq=8 * r, sq_h=most + 8) == -4, r
    for huge in (1 << 40, 1 << 60, (1 << 63) - 8):
        assert fn(N=0, Hq=64, sq_h=huge) == -4
