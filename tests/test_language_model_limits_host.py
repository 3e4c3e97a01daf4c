"""Host side of the language model operators: what they refuse besides wrong extents and types."""
import ctypes as C

import pytest

from flashlight_b200 import _lib as L


@pytest.mark.parametrize("off", [1, 8, 16, 24])
def test_linear_cce_gradient_refuses_a_workspace_off_32_bytes(off):
    """It stores the scores' gradient 32 bytes at a time at multiples of 256 from the workspace's start."""
    d = L.LinearCceDesc(rows=4, features=8, classes=16, reduction=L.REDUCE_MEAN, ignore_index=-1, dtype=L.BF16)
    assert L.lib.flb200_linear_cce_backward(C.byref(d), 16, 16, None, 16, 16, 16, 16, 16, 16, L.BF16, None, 4096 + off,
                                            1 << 40, None) == L.WORKSPACE_TOO_SMALL
    assert b"32-byte aligned" in L.lib.flb200_last_error()
