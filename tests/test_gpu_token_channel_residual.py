"""A residual that is not shaped like the output is refused in every call, also where its elements are as many."""

import pytest
import torch

from ksdraft_amd.kernels import token_channel as tc

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("shape", [(3, 2, 8), (6, 8), (1, 6, 8), (2, 3, 4, 2), (2, 3, 1), (8,)])
def test_other_shapes(shape):
    x, w, res = torch.ones(2, 3, 64, device=DEV), torch.ones(8, 64, device=DEV), torch.ones(shape, device=DEV)
    codes, scales = tc.quantize_rows(w)
    lin = tc.TokenChannelLinear(64, 8).to(DEV)
    with pytest.raises(ValueError, match="residual"):
        tc.token_channel_linear(x, codes, scales, residual=res)
    with pytest.raises(ValueError, match="residual"):
        tc.token_channel_linear_train(x, w, residual=res)
    with pytest.raises(ValueError, match="residual"):
        lin(x, residual=res)
    with torch.no_grad(), pytest.raises(ValueError, match="residual"):
        lin(x, residual=res)


@pytest.mark.parametrize("lead", [(), (5,), (2, 3), (2, 1, 3)])
def test_any_leading_shape(lead):
    x, w, res = torch.ones(*lead, 64, device=DEV), torch.ones(8, 64, device=DEV), torch.ones(*lead, 8, device=DEV)
    y = tc.token_channel_linear(x, *tc.quantize_rows(w), residual=res)
    assert y.shape == res.shape and torch.equal(y, tc.token_channel_linear_train(x, w, residual=res)[0])
    assert bool((y == 65).all())
