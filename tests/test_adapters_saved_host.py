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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_parameters_keep_their_gradients_bits(calls, monkeypatch, dtype):
    """An adapted layer's fp32 parameters get the kernels' fp32 sums: what 16 bits would round, or not hold."""
    from ksdraft_amd.model.adapters import AdaptedLinear, AdapterSelection
    lin = AdaptedLinear(torch.nn.Linear(8, 5, dtype=dtype).requires_grad_(False), 2, 3, AdapterSelection())
    lin.selection.index = torch.tensor([0, 1, -1, 0])
    da, db = torch.randn(2, 3, 8) * 1e6, torch.randn(2, 5, 3) * 1e6 + 2.0 ** -10
    monkeypatch.setattr(adapters, "adapter_linear_backward", lambda g, s, *a: (g.new_zeros(4, 8), da, db))
    lin(torch.randn(4, 8, dtype=dtype)).sum().backward()
    assert torch.equal(lin.adapter_a.grad, da) and torch.equal(lin.adapter_b.grad, db)
    # what the kernels read is of x's type
    assert calls[0][1][1] == _lib.dtype_code(dtype)


def test_types_of_adapters(calls):
    """Banks of x's type or fp32; the gradient is of the bank's type."""
    x, a, b, index = inputs()
    h = x.detach().half()
    y = adapters.adapt(h, a.detach().half().requires_grad_(), b, index)
    assert y.dtype == torch.float16 and y.requires_grad
    y = adapters.adapt(h, a, b, index, base=torch.zeros(4, 5, dtype=torch.float16))
    y.sum().backward()
    assert a.grad.dtype == b.grad.dtype == torch.float32
    with pytest.raises(TypeError):
        adapters.adapt(h, a.bfloat16(), b, index)
    with pytest.raises(TypeError):
        adapters.adapt(x, a.half(), b, index)


def test_out_over_an_operand(calls):
    """The kernel reads the scales of every row while it writes out."""
    x, a, b, index = (t.detach() for t in inputs())
    room = torch.zeros(64)
    out, scales = room[:20].view(4, 5), room[18:20]
    with pytest.raises(ValueError, match="scales"):
        adapters.adapter_linear(x, a, b, index, scales, out=out)
    adapters.adapter_linear(x, a, b, index, room[20:22], out=out)
    assert len(calls) == 1
