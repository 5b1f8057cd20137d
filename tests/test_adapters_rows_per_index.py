"""The adapters' C entries divide a row by rows_per_index in 32 bits: what does not fit is refused before a launch (CPU)."""

import ctypes

import pytest

from ksdraft_amd import _lib
from tests.test_adapters_host import backward, forward


@pytest.mark.parametrize("per", [0, -1, 1 << 31, 1 << 32, (1 << 32) + 1, 1 << 40])
def test_refused(per):
    need = ctypes.c_int64()
    assert forward(per=per) == 1 and backward(per=per) == 1
    for name in ("ksd_adapter_linear_workspace", "ksd_adapter_linear_backward_workspace"):
        assert getattr(_lib.load(), name)(4, 8, 16, 4, 2, per, 0, ctypes.byref(need)) == 1


def test_largest():
    need = ctypes.c_int64()
    for name in ("ksd_adapter_linear_workspace", "ksd_adapter_linear_backward_workspace"):
        assert getattr(_lib.load(), name)(4, 8, 16, 4, 2, (1 << 31) - 1, 0, ctypes.byref(need)) == 0
