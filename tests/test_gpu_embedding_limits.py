"""The table gradient beside the 2^32 threads that one launch holds: a 64 GiB table whose clearing fits a launch
with the 128 workgroups that count 4096 tokens and not with the 512 that count 8192."""

import math

import pytest
import torch

from ksdraft_amd.kernels.embedding import embedding_gradient

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,V,d", [(8192, 23, 40), (4096, 524276, 32768), (8192, 524276, 32768)])
def test_clearing_beside_counting(n, V, d):
    if V > 23:
        torch.cuda.empty_cache()
        if torch.cuda.mem_get_info()[0] < 80 << 30:
            pytest.skip("needs 80 GiB of free device memory")
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[0], ids[1] = 0, V - 1
    rows = torch.randint(-8, 9, (n,), generator=g)  # small whole numbers: every sum is exact
    grad = (rows.to(DEV).float()[:, None] * (1 + torch.arange(d, device=DEV) % 7)).to(torch.bfloat16)
    out = torch.full((V, d), math.nan, device=DEV)
    embedding_gradient(grad, ids.to(DEV), V, out=out)
    sums = torch.zeros(V, dtype=torch.int64).index_add_(0, ids, rows).to(DEV).float()
    scale = (1 + torch.arange(d, device=DEV) % 7).float()
    for v in range(0, V, 1 << 14):
        assert torch.equal(out[v:v + (1 << 14)], sums[v:v + (1 << 14), None] * scale)
