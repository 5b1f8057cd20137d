"""Clipping where tensors are listed twice or meet in memory: a tied parameter counts and is scaled once,
written memory that two tensors share is refused before it is written, neighbours are not.

The bounds are those of a clipped gradient: a factor of four fp32 operations and one product."""

import math

import pytest
import torch

from ksdraft_amd.train.clip import clip_grad_norm_, clip_gradients, gradient_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_tied_parameter_listed_twice():
    g = torch.Generator().manual_seed(0)
    tied, other = (torch.nn.Parameter(torch.zeros(300, 70, device=DEV)) for _ in range(2))
    tied.grad, other.grad = (torch.randn(300, 70, generator=g).to(DEV) for _ in range(2))
    was = [p.grad.double() for p in (tied, other)]
    total = math.sqrt(sum(float(t.pow(2).sum()) for t in was))
    # 97 entries and more: the repeated ones would lie in one launch, and in two
    few = [torch.nn.Parameter(torch.zeros(1, device=DEV)) for _ in range(100)]
    norm = clip_grad_norm_(iter([tied, other, tied, *few, tied]), 1.0)
    assert abs(norm.item() - total) <= 3 * 2.0 ** -24 * total
    for p, t in zip((tied, other), was):
        ref = t / (total + 1e-6)
        assert bool(((p.grad.double() - ref).abs() <= 13 * 2.0 ** -24 * ref.abs()).all())


def test_shared_memory_is_refused_unwritten():
    t, u = torch.full((50000,), 3.0, device=DEV), torch.full((50000,), 4.0, device=DEV)
    out = torch.full((50000,), 7.0, device=DEV)
    with pytest.raises(ValueError):
        clip_gradients([t, t], 1.0)
    with pytest.raises(ValueError):
        clip_gradients([t[:30000], u, t[29999:]], 1.0)
    with pytest.raises(ValueError):
        clip_gradients([t, u], 1.0, out=[out, out])
    with pytest.raises(ValueError):
        clip_gradients([t, u], 1.0, out=[u, out])
    assert bool((t == 3).all() and (u == 4).all() and (out == 7).all())
    # nothing is written by the norm: a list may repeat itself there
    assert abs(gradient_norm([t, t])[0].item() - 3 * math.sqrt(100000)) <= 1e-3


def test_neighbours_in_any_order():
    flat = torch.full((90000,), 2.0, device=DEV)
    parts = list(flat.split([7, 40000, 1, 30000, 19992]))
    parts = [parts[i] for i in (3, 0, 4, 2, 1)]
    out = torch.zeros(90000, device=DEV)
    outs = [out[10:][sum(p.numel() for p in parts[:k]):][:p.numel()] for k, p in enumerate(parts[:4])] + [parts[4]]
    norm = clip_gradients(parts, 1.0, out=outs)  # the last one in place, the others not
    total = 2 * math.sqrt(90000)
    assert abs(norm.item() - total) <= 3 * 2.0 ** -24 * total
    want = 2 / (total + 1e-6)
    n = 90000 - parts[4].numel()
    assert bool(((out[10:10 + n] - want).abs() <= 13 * 2.0 ** -24 * want).all()) and not bool(out[:10].any())
    assert bool(((parts[4] - want).abs() <= 13 * 2.0 ** -24 * want).all()) and bool((flat[:7] == 2).all())
    clip_gradients([p.zero_() for p in parts], 1.0)
    assert not bool(flat.any())
