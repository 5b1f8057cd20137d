"""The bias gradient of a layer whose weight is frozen and whose input needs none: the column sums of dY, as
nn.Linear gives them, with and without a residual.

A sum of M terms in fp32 is within M roundings of the magnitudes' sum of the exact one."""

import pytest
import torch

from ksdraft_amd.kernels import Int8Linear, TokenChannelLinear

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAYERS = [TokenChannelLinear, Int8Linear]


@pytest.mark.parametrize("layer", LAYERS)
@pytest.mark.parametrize("residual", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(1, 128, 20), (3, 128, 64), (300, 256, 77)])
def test_bias_alone_trains(M, K, N, dtype, residual, layer):
    g = torch.Generator().manual_seed(M)
    lin = layer.from_float(torch.nn.Linear(K, N).to(DEV))
    lin.weight.requires_grad_(False)
    x = torch.randn(M, K, generator=g).to(dtype).to(DEV)
    res = None if residual is None else torch.randn(M, N, generator=g).to(residual).to(DEV)
    with torch.no_grad():
        want = lin(x, residual=res)
    y = lin(x, residual=res)
    assert torch.equal(y, want) and y.requires_grad
    dy = torch.randn(M, N, generator=g).to(y.dtype).to(DEV)
    y.backward(dy)
    ref = dy.to(dtype).double()
    assert bool(((lin.bias.grad.double() - ref.sum(0)).abs() <= (M + 1) * 2.0 ** -24 * ref.abs().sum(0)).all())
    assert lin.weight.grad is None


@pytest.mark.parametrize("layer", LAYERS)
def test_nothing_trains(layer):
    lin = layer.from_float(torch.nn.Linear(128, 20).to(DEV)).requires_grad_(False)
    assert not lin(torch.ones(3, 128, device=DEV)).requires_grad
