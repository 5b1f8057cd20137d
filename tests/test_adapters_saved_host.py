"""What the backward pass of ``adapt`` is called with when its saved tensors come back elsewhere (CPU: the kernels are replaced)."""

import pytest
import torch

from ksdraft_amd import _lib
from ksdraft_amd.kernels import adapters


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "capture_guard", lambda *t: None)
    monkeypatch.setattr(_lib, "call_on", lambda dev, name, *args: seen.append((name, args)))
    return seen


def inputs():
    x = torch.randn(4, 8, requires_grad=True)
    return x, torch.randn(2, 3, 8, requires_grad=True), torch.randn(2, 5, 3, requires_grad=True), torch.tensor([0, 1, -1, 0])


FORWARD, BACKWARD = slice(-8, -4), slice(-9, -5)  # the mask's four arguments: (65536 p, seed, device seed's address, stream)


def test_device_seed_through_hooks(calls):
    """The mask's key is read where the saved seed is now, not where the forward had it."""
    back = []

    def unpack(t):
        back.append(t)
        return t
    seed = torch.tensor([77])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
        y = adapters.adapt(*inputs(), dropout=0.25, seed=seed, stream=3)
    y.sum().backward()
    (first, f), (second, b) = calls
    assert (first, second) == ("ksd_adapter_linear", "ksd_adapter_linear_backward")
    assert f[FORWARD][0] == b[BACKWARD][0] == 16384 and f[FORWARD][3] == b[BACKWARD][3] == 3
    at = [t for t in back if t.data_ptr() == b[BACKWARD][2]]
    assert len(at) == 1 and at[0].dtype == torch.int64 and at[0].tolist() == [77]


def test_number_as_seed(calls):
    y = adapters.adapt(*inputs(), dropout=0.25, seed=1 << 40, stream=5)
    y.sum().backward()
    assert calls[0][1][FORWARD] == calls[1][1][BACKWARD] == (16384, 1 << 40, None, 5)


def test_unused_seed_may_change(calls):
    """At a probability of 0 nothing reads the seed: counting it on before the backward pass is no write into a saved tensor."""
    seed = torch.tensor([77])
    y = adapters.adapt(*inputs(), dropout=0.0, seed=seed)
    seed += 1
    y.sum().backward()
    assert calls[1][1][BACKWARD][0] == 0
