"""What the verification's C entry refuses, and its workspace (CPU)."""

import ctypes

import pytest
import torch

from ksdraft_amd import _lib
from ksdraft_amd.kernels.speculate import sample_tokens, verify_draft


def test_abi_refusals():
    lib, p = _lib.load(), ctypes.c_void_p(256)  # never dereferenced
    need = ctypes.c_int64()

    def call(B=2, L=3, V=50, dtype=0, strides=(200, 50, 150, 50), tokens=p, u=p, temps=p, temp=1.0, work=p, size=1 << 40):
        return lib.ksd_verify_draft(p, p, dtype, B, L, V, *strides, tokens, u, 0, temps, temp, None, p, p, work, size, None)
    assert call(B=0) == 0
    assert call(B=-1) == 1 and call(L=-1) == 1 and call(V=0) == 1 and call(V=1 << 31) == 1 and call(B=1 << 21) == 1
    assert call(B=1 << 18, L=1 << 10) == 1
    assert call(dtype=5) == 2
    assert call(strides=(200, -50, 150, 50)) == 1 and call(tokens=None) == 1 and call(u=None) == 1
    assert call(u=None, temps=None, temp=0.5) == 1 and call(work=None) == 1
    assert lib.ksd_verify_draft_workspace(2, 3, 50, 1, ctypes.byref(need)) == 0 and need.value > 0
    assert call(size=need.value - 1) == 1
    assert lib.ksd_verify_draft_workspace(2, 3, 0, 1, ctypes.byref(need)) == 1
    assert lib.ksd_verify_draft_workspace(2, 3, 50, 1, None) == 1


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError):
        verify_draft(torch.zeros(1, 2, 5), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 2))
    with pytest.raises(RuntimeError):
        sample_tokens(torch.zeros(1, 5), torch.zeros(1))
