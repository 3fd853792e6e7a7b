"""The status word's entry point refuses bad pointers on the host."""
import ctypes

import pytest

from innerq_amd import _lib


@pytest.mark.parametrize("status,taken,err", [(None, 0x1000, -1), (0x1000, None, -1), (0x1002, 0x1000, -5), (0x1000, 0x1001, -5)])
def test_take_status_rejects(status, taken, err):
    assert _lib.lib().iq_paged_take_status(ctypes.c_void_p(status), ctypes.c_void_p(taken), None) == err
