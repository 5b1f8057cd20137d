"""Kernels that write into a caller's tensors count in their versions, as torch's in-place operations do."""

import pytest
import torch

from ksdraft_amd.kernels.embedding import embedding_gradient
from ksdraft_amd.kernels import Int8Linear
from ksdraft_amd.train import AdamWRequant, adamw_requant_, adamw_requant_multi_
from ksdraft_amd.train.clip import clip_grad_norm_, clip_gradients, gradient_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def versions(ts):
    return [t._version for t in ts]


def test_clipping():
    ts = [torch.ones(5, device=DEV), torch.ones(70, 3, device=DEV)]
    out = [torch.zeros_like(t) for t in ts]
    was, outs = versions(ts), versions(out)
    gradient_norm(ts)
    clip_gradients(ts, 1.0, out=out)
    assert versions(ts) == was and all(a > b for a, b in zip(versions(out), outs))
    clip_gradients(ts, 1.0)
    assert all(a > b for a, b in zip(versions(ts), was))
    p = torch.nn.Parameter(torch.ones(4, device=DEV))
    p.grad = torch.ones(4, device=DEV)
    was = p.grad._version
    clip_grad_norm_(p, 1.0)
    assert p.grad._version > was


def test_backward_refuses_clipped_values():
    x = torch.ones(8, device=DEV, requires_grad=True)
    kept = torch.full((8,), 3.0, device=DEV)
    y = (x * kept).sum()
    clip_gradients([kept], 1.0)
    with pytest.raises(RuntimeError):
        y.backward()


def test_embedding_gradient():
    g, ids = torch.ones(2, 8, device=DEV), torch.tensor([1, 2], device=DEV)
    out = torch.zeros(5, 8, device=DEV)
    for accumulate in (False, True):
        was = out._version
        embedding_gradient(g, ids, 5, out=out, accumulate=accumulate)
        assert out._version > was


@pytest.mark.parametrize("multi", [False, True])
@pytest.mark.parametrize("quantize", [False, True])
def test_optimizer_kernels(multi, quantize):
    p, g, m, v = (torch.ones(8, 128, device=DEV) for _ in range(4))
    was = versions([p, g, m, v])
    if multi:
        adamw_requant_multi_([(p, g, m, v, 1, quantize)], 1e-3)
    else:
        adamw_requant_(p, g, m, v, 1, 1e-3, quantize=quantize)
    now = versions([p, g, m, v])
    assert [a > b for a, b in zip(now, was)] == [True, False, True, True]


def test_optimizer_step():
    """Fused masters and torch's small ones alike; the registered layer's codes stay current, those of
    another layer on the same master do not."""
    lin, tied = Int8Linear(256, 512).to(DEV), Int8Linear(256, 512, bias=False).to(DEV)
    tied.weight = lin.weight
    plain = torch.nn.Parameter(torch.ones(1 << 17, device=DEV))
    opt = AdamWRequant([*lin.parameters(), plain], lr=1e-2)
    opt.register_int8(tied)
    opt.register_int8(lin)
    params = [lin.weight, lin.bias, plain]
    for _ in range(2):
        for p in params:
            p.grad = torch.ones_like(p)
        was = versions(params)
        opt.step()
        assert all(a > b for a, b in zip(versions(params), was))
        assert lin._codes_current() and not tied._codes_current()


def test_inference_tensors():
    """They have no version: clipped all the same, beside ordinary ones."""
    with torch.inference_mode():
        a = torch.full((4,), 3.0, device=DEV)
    b = torch.full((4,), 3.0, device=DEV)
    was = b._version
    with torch.inference_mode():
        clip_gradients([b, a], 0.5)
        embedding_gradient(torch.ones(1, 4, device=DEV), torch.tensor([0], device=DEV), 1, out=a.view(1, 4), accumulate=True)
    assert b._version > was and bool((b < 1).all()) and bool((a > 1).all())
