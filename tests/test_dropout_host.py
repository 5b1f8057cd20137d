"""The mask's generator against its published known answers, and the calls that dropout refuses (CPU)."""

import ctypes

import numpy as np
import pytest
import torch

from ksdraft_amd import _lib
from ksdraft_amd.kernels.dropout import Dropout, dropout, mask_arguments
from tests.philox import halves, philox

CPU = torch.device("cpu")


def test_known_answers():
    """The generator's published vectors: zeros, ones and the digits of pi."""
    cases = [((0,) * 4, (0,) * 2, (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
             ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
             ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
              (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]
    for counter, key, out in cases:
        assert tuple(int(v) for v in philox(counter, key)) == out


def test_halves_are_uniform():
    """512 x 128 values: the mean of 16 bits has a standard deviation of 2^16 / sqrt(12) / 256."""
    u = halves(512, 128, 5, 0).astype(np.float64)
    assert abs(u.mean() - 32767.5) < 6 * 2 ** 16 / 12 ** 0.5 / 256
    assert len(np.unique(halves(64, 8, 5, 0) * 65536 + halves(64, 8, 5, 1))) > 500


def test_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError):
        dropout(x, 0.1, 0)
    for p, seed, stream in ((-0.1, 0, 0), (1.5, 0, 0), (float("nan"), 0, 0), (0.1, -1, 0), (0.1, 1 << 64, 0), (0.1, 0, 1 << 32),
                            (0.1, 0, -1), (0.1, torch.zeros(2, dtype=torch.int64), 0), (0.1, torch.zeros(1), 0)):
        with pytest.raises(ValueError):
            mask_arguments(p, seed, stream, CPU)
    with pytest.raises(ValueError):
        Dropout(1.1)


def test_abi_refusals():
    p = ctypes.c_void_p(256)  # never dereferenced
    f = _lib.load().ksd_dropout
    assert f(p, 0, 4, 8, 7, 100, 1, None, 0, None, 0, p, None) == 1      # rows overlap
    assert f(p, 0, 4, 8, 8, 100, 1, None, 0, p, 7, p, None) == 1
    assert f(p, 7, 4, 8, 8, 100, 1, None, 0, None, 0, p, None) == 2
    assert f(p, 0, 4, 8, 8, 65537, 1, None, 0, None, 0, p, None) == 1
    assert f(p, 0, 4, 8, 8, -1, 1, None, 0, None, 0, p, None) == 1
    assert f(p, 0, 4, 8, 8, 100, 1, None, 1 << 32, None, 0, p, None) == 1
    assert f(p, 0, 4, 8, 8, 100, 1, ctypes.c_void_p(260), 0, None, 0, p, None) == 1  # seed's address
    assert f(None, 0, 4, 8, 8, 100, 1, None, 0, None, 0, p, None) == 1
    assert f(p, 0, 1, 1 << 35, 1 << 35, 100, 1, None, 0, None, 0, p, None) == 1
    assert f(None, 0, 0, 8, 8, 100, 1, None, 0, None, 0, None, None) == 0
