"""Gradients of ``adapt`` and ``dropout`` with a seed on the device where saved tensors leave the device or are made again: the
same bits as without."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from ksdraft_amd.kernels.adapters import adapt
from ksdraft_amd.kernels.dropout import dropout

pytestmark = pytest.mark.gpu
DEV = "cuda"


def both(f, *leaves):
    """Outputs and gradients of f() plainly, under saved tensors kept on the CPU, and recomputed."""
    runs = []
    for kind in ("plain", "cpu", "again"):
        for t in leaves:
            t.grad = None
        if kind == "cpu":
            with torch.autograd.graph.save_on_cpu():
                y = f()
        else:
            y = checkpoint(f, use_reentrant=False) if kind == "again" else f()
        junk = [torch.full((1,), 1000 + i, device=DEV) for i in range(64)]  # what the forward freed holds other values now
        (y.float() * torch.arange(y.shape[-1], device=DEV)).sum().backward()
        runs.append([y.detach()] + [t.grad.clone() for t in leaves])
        del junk
    for other in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], other))
    return runs[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,n", [(37, 3), (900, 5)])
def test_adapt(M, n, dtype):
    g = torch.Generator(DEV).manual_seed(1)

    def leaf(*shape):
        return torch.randn(*shape, device=DEV, generator=g).to(dtype).requires_grad_()
    x, a, b, base = leaf(M, 200), leaf(n, 12, 200), leaf(n, 136, 12), leaf(M, 136)
    index = torch.randint(-1, n, (M,), device=DEV, generator=g)
    seed = torch.tensor([31], device=DEV)
    grads = both(lambda: adapt(x, a, b, index, None, base, 0.3, seed, 4), x, a, b, base)
    seed.fill_(32)
    other = both(lambda: adapt(x, a, b, index, None, base, 0.3, seed, 4), x, a, b, base)
    assert not torch.equal(grads[1], other[1])


def test_dropout():
    x = torch.randn(50, 77, device=DEV, requires_grad=True)
    seed = torch.tensor([5], device=DEV)
    both(lambda: dropout(x, 0.4, seed, 1), x)
