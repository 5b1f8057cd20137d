"""Gradients of gradients: refused where the backward is a kernel, which autograd would otherwise take for a
constant; first gradients under create_graph are the plain ones."""

import pytest
import torch

from ksdraft_amd.kernels import TokenChannelLinear
from ksdraft_amd.kernels.embedding import scaled_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"


def linear():
    lin = TokenChannelLinear.from_float(torch.nn.Linear(64, 20).to(DEV))
    x = torch.randn(5, 64, generator=torch.Generator().manual_seed(0)).to(DEV).requires_grad_(True)
    res = torch.ones(5, 20, device=DEV, requires_grad=True)
    return lambda: lin(x, residual=res), [x, lin.weight, lin.bias, res]


def lookup():
    w = torch.randn(9, 16, generator=torch.Generator().manual_seed(0)).to(DEV).requires_grad_(True)
    ids = torch.tensor([1, 8, 1], device=DEV)
    return lambda: scaled_rows(w, ids, 2.0), [w]


@pytest.mark.parametrize("make", [linear, lookup])
def test_second_gradient_is_refused(make):
    call, inputs = make()
    plain = torch.autograd.grad(call().square().sum(), inputs)
    first = torch.autograd.grad(call().square().sum(), inputs, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, first))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first[0].square().sum().backward()
