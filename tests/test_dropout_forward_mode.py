"""Forward-mode derivatives of dropout: the tangent goes through the same mask (CPU: the kernel is replaced by its formula)."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from ksdraft_amd import _lib
from ksdraft_amd.kernels.adapters import adapt
from ksdraft_amd.kernels.dropout import dropout
from tests.philox import mask


@pytest.fixture
def kernel(monkeypatch):
    """ksdraft's dropout call on CPU memory."""
    def view(at, rows, d):
        return torch.frombuffer((ctypes.c_float * (rows * d)).from_address(at), dtype=torch.float32).view(rows, d)

    def call_on(dev, name, *args):
        if name == "ksd_dropout":
            ksd_dropout(*args)

    def ksd_dropout(x, dt, rows, d, pitch, drop, seed, seed_from, stream, res, res_pitch, out):
        assert pitch == d
        seed = ctypes.c_int64.from_address(seed_from).value if seed_from else seed
        y = view(x, rows, d) * mask(rows, d, drop / 65536, seed, stream)
        view(out, rows, d).copy_(y if res is None else y + view(res, rows, d))
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "capture_guard", lambda *t: None)
    monkeypatch.setattr(_lib, "call_on", call_on)


@pytest.mark.parametrize("seed", [7, torch.tensor([7])])
@pytest.mark.parametrize("leaf", [False, True])
def test_tangent(kernel, leaf, seed):
    x, t = torch.randn(5, 24), torch.randn(5, 24)
    res, rt = torch.randn(5, 24), torch.randn(5, 24)
    x.requires_grad_(leaf)
    keep = mask(5, 24, 0.5, 7, 2)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        y = forward_ad.unpack_dual(dropout(dual, 0.5, seed, 2))
        assert torch.equal(y.primal.detach(), x.detach() * keep) and torch.equal(y.tangent, t * keep)
        y = forward_ad.unpack_dual(dropout(dual, 0.5, seed, 2, residual=res))
        assert torch.equal(y.tangent, t * keep)
        y = forward_ad.unpack_dual(dropout(dual, 0.5, seed, 2, residual=forward_ad.make_dual(res, rt)))
        assert torch.equal(y.tangent, t * keep + rt)
        y = forward_ad.unpack_dual(dropout(x, 0.5, seed, 2, residual=forward_ad.make_dual(res, rt)))
        assert torch.equal(y.tangent, rt)
        with torch.no_grad():
            assert torch.equal(forward_ad.unpack_dual(dropout(dual, 0.5, seed, 2)).tangent, t * keep)
    plain = dropout(x.detach(), 0.5, seed, 2)
    assert torch.equal(plain, x.detach() * keep) and not plain.requires_grad


def test_backward_as_before(kernel):
    x = torch.randn(5, 24, requires_grad=True)
    dropout(x, 0.5, 7, 2).sum().backward()
    assert torch.equal(x.grad, mask(5, 24, 0.5, 7, 2))


def test_adapters_refuse_it(kernel):
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.randn(4, 8), torch.randn(4, 8))
        with pytest.raises((RuntimeError, NotImplementedError)):
            adapt(x, torch.randn(2, 3, 8), torch.randn(2, 5, 3), torch.tensor([0, 1, -1, 0]))
