"""The operators on more than 2^31 elements of one tensor: parts of the results against calls on parts."""

import math

import pytest
import torch

from ksdraft_amd.kernels import token_channel as tc
from ksdraft_amd.kernels.embedding import embedding_gradient, embedding_lookup
from ksdraft_amd.train.clip import clip_gradients

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GiB of free device memory")
    yield
    torch.cuda.empty_cache()


def test_training_call():
    """A row of y and dX depends on its token alone, a row of dW on its channel's column of dY."""
    M, K, N = 16384, 64, 150144
    g = torch.Generator(device=DEV).manual_seed(0)
    x, w = torch.randn(M, K, device=DEV, generator=g).bfloat16(), torch.randn(N, K, device=DEV, generator=g)
    dy = torch.randn(M, N, device=DEV, generator=g, dtype=torch.bfloat16)
    bias = torch.randn(N, device=DEV, generator=g)
    y, saved = tc.token_channel_linear_train(x, w, bias)
    dx, dw, db = tc.token_channel_linear_backward(dy, saved)
    rows = torch.tensor([0, 1, 14302, 14303, 16382, 16383], device=DEV)  # around 2^31 elements, and the ends
    py, part = tc.token_channel_linear_train(x[rows], w, bias)
    assert torch.equal(y[rows], py) and torch.equal(dx[rows], tc.token_channel_linear_backward(dy[rows], part, need_dw=False)[0])
    cols = torch.tensor([0, 1, 77777, 150142, 150143], device=DEV)
    py, part = tc.token_channel_linear_train(x, w[cols], bias[cols])
    _, pdw, pdb = tc.token_channel_linear_backward(dy[:, cols], part, need_dx=False)
    assert torch.equal(y[:, cols], py) and torch.equal(dw[cols], pdw)
    size = dy[:, cols].float().abs().sum(0)
    assert bool(((db[cols] - pdb).abs() <= 2 * M * 2.0 ** -24 * size).all())


def test_clipping():
    n = (1 << 31) + 8193
    t = torch.full((n,), 0.25, dtype=torch.bfloat16, device=DEV)
    norm = clip_gradients([t], 0.125 * math.sqrt(n))
    assert abs(norm.item() - 0.25 * math.sqrt(n)) <= 3 * 2.0 ** -24 * norm.item()
    for i in range(0, n, 1 << 28):
        assert bool((t[i:i + (1 << 28)] == 0.125).all())


@pytest.mark.parametrize("n", [300, 5000, 70000])
def test_table(n):
    """A table of 2^31 elements and more, tokens at both ends of it."""
    V, d = 1 << 20, 2056
    g = torch.Generator().manual_seed(n)
    ids = torch.cat([torch.tensor([0, V - 1, V - 1]), torch.randint(V - 5000, V, (n - 3,), generator=g)]).to(DEV)
    rows = torch.randint(-8, 9, (n, 1), generator=g).float().to(DEV).expand(n, d).contiguous()
    dw = embedding_gradient(rows, ids, V)
    sums = torch.zeros(V, device=DEV).index_add_(0, ids, rows[:, 0])  # whole numbers: exact in any order
    for v in range(0, V, 1 << 16):
        assert torch.equal(dw[v:v + (1 << 16)], sums[v:v + (1 << 16), None].expand(-1, d))
    assert torch.equal(embedding_lookup(dw, ids, 2.0), 2 * sums[ids][:, None].expand(n, d))
