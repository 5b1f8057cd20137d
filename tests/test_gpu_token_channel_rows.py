"""A layer's training call on more tokens than 65535 blocks of rows (2.1 million tokens of few channels, 4.2
million of many): every gradient against the same call on a part of the tokens that holds all that is not zero.

With zeros in all other tokens, their codes are zero and a channel's scale is the part's, so dX's rows and
dW are the part's bits; db's sum of the same terms in another order is within a rounding each."""

import pytest
import torch

from ksdraft_amd.kernels import token_channel as tc

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(2097120, 9, 8), (2097121, 9, 8), (2200001, 15, 8), (4194241, 9, 16), (4300000, 20, 16)])
def test_many_tokens(M, N, K, dtype):
    g = torch.Generator().manual_seed(M)
    at = torch.cat([torch.arange(70), torch.randint(70, M - 70, (60,), generator=g).unique(), torch.arange(M - 70, M)]).to(DEV)
    px, pg = (torch.randn(len(at), c, generator=g).to(dtype).to(DEV) for c in (K, N))
    w, bias = torch.randn(N, K, generator=g).to(DEV), torch.randn(N, generator=g).to(DEV)
    x, dy = torch.zeros(M, K, dtype=dtype, device=DEV), torch.zeros(M, N, dtype=dtype, device=DEV)
    x[at], dy[at] = px, pg
    want_y, part = tc.token_channel_linear_train(px, w, bias)
    want_dx, want_dw, want_db = tc.token_channel_linear_backward(pg, part)
    y, saved = tc.token_channel_linear_train(x, w, bias)
    dx, dw, db = tc.token_channel_linear_backward(dy, saved)
    assert torch.equal(y[at], want_y) and torch.equal(dx[at], want_dx) and torch.equal(dw, want_dw)
    assert bool(((db - want_db).abs() <= 2 * len(at) * 2.0 ** -24 * pg.float().abs().sum(0)).all())
    y[at] = bias.to(dtype)
    dx[at] = 0
    assert torch.equal(y, bias.to(dtype).expand(M, N)) and not bool(dx.any())
