"""Gradients of an adapted layer's fp32 parameters in 16-bit models, against fp64 on the CPU: sums in fp32, not rounded to the
layer's type, also past fp16's range.

Bound, u = 2^-24: a sum of k products in any order is off by at most k u of the sum of magnitudes, twice that allowed for
sums inside an instruction; a product of two such sums adds theirs."""

import pytest
import torch

from ksdraft_amd.model.adapters import AdaptedLinear, AdapterSelection

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1.0, 64.0])
def test_gradients(dtype, size):
    torch.manual_seed(2)
    M, K, N, n, r = 600, 96, 72, 3, 8
    lin = AdaptedLinear(torch.nn.Linear(K, N, dtype=dtype).requires_grad_(False), n, r, AdapterSelection(), alpha=16.0).to(DEV)
    with torch.no_grad():
        lin.adapter_a.abs_()
        lin.adapter_b.uniform_(0, 1)
    index = torch.randint(-1, n, (M,))
    lin.selection.index = index.to(DEV)
    x = (torch.rand(M, K) * size ** 0.5).to(dtype)
    dy = (torch.rand(M, N) * size).to(dtype)
    lin(x.to(DEV)).backward(dy.to(DEV))
    a, b = (p.detach().to(dtype).double().cpu() for p in (lin.adapter_a, lin.adapter_b))  # as the layer uses them
    x, dy = x.double(), dy.double()
    top = 0.0
    for i in range(n):
        at = index == i
        da, db = (dy[at] @ b[i]).t() @ x[at] * 2.0, dy[at].t() @ (x[at] @ a[i].t()) * 2.0
        for got, want, k in ((lin.adapter_a.grad[i], da, N), (lin.adapter_b.grad[i], db, K)):
            assert got.dtype == torch.float32
            assert bool(((got.double().cpu() - want).abs() <= 2 * (k + M + 8) * U * want).all())  # all terms are positive
            top = max(top, float(want.max()))
    assert (top > 65504) == (size > 1)
