"""Gradient norm and clipping against 64-bit sums.

The squares and sums are fp64, so the norm is its rounding to fp32 (2^-24 relative, doubled for the
division by the loss scale and the comparison's own rounding). The factor takes four fp32
operations, a clipped gradient one product and one rounding to its type."""

import math

import pytest
import torch

from ksdraft_amd.train import AdamWRequant
from ksdraft_amd.train.clip import clip_grad_norm_, clip_gradients, gradient_norm

DEV = "cuda"
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def tensors(shapes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*s, generator=g) * scale).to(dtypes[i % len(dtypes)]).to(DEV) for i, s in enumerate(shapes)]


def reference(ts, max_norm, loss_scale=1.0, inf=False):
    if inf:
        total = max(float(t.double().abs().max()) for t in ts if t.numel()) / loss_scale
    else:
        total = math.sqrt(sum(float(t.double().pow(2).sum()) for t in ts)) / loss_scale
    return total, min(1.0, max_norm / (total + 1e-6)) / loss_scale


SETS = [
    [(1,)],
    [(7,), (3, 5), (0, 4), (129,)],
    [(16384,), (16385,), (16383,), (1,)],
    [(257, 513), (1000001,), (5,)],
    [(i % 37 + 1,) for i in range(300)],
    [(3, i + 1) for i in range(97)],
]
TYPES = [[torch.float32], [torch.bfloat16], [torch.float16], [torch.float32, torch.bfloat16, torch.float16]]


@pytest.mark.gpu
@pytest.mark.parametrize("types", range(4))
@pytest.mark.parametrize("which", range(len(SETS)))
@pytest.mark.parametrize("max_norm,loss_scale", [(1.0, 1.0), (0.3, 1024.0), (1e6, 1.0), (1e6, 8.0)])
def test_clip(which, types, max_norm, loss_scale):
    ts = tensors(SETS[which], TYPES[types], seed=which)
    was = [t.clone() for t in ts]
    total, factor = reference(ts, max_norm, loss_scale)
    out = [torch.full_like(t, math.nan) for t in ts]
    norm = clip_gradients(ts, max_norm, out=out, loss_scale=loss_scale)
    assert abs(norm.item() - total) <= 3 * 2.0 ** -24 * total
    assert all(torch.equal(a, b) for a, b in zip(ts, was))
    for t, o in zip(was, out):
        ref = t.double() * factor
        bound = 12 * 2.0 ** -24 * ref.abs()
        bound = bound + EPS[t.dtype] * (ref.abs() + bound) + (2.0 ** -25 if t.dtype == torch.float16 else 1e-45)
        assert bool(((o.double() - ref).abs() <= bound).all())
    norm2 = clip_gradients(ts, max_norm, loss_scale=loss_scale)  # in place
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(ts, out))


@pytest.mark.gpu
def test_inf_norm_views_and_alignment():
    flat = tensors([(100000,)], [torch.bfloat16])[0]
    ts = [flat[1:5000], flat[5003:5004], flat[6001:90000]]
    total, _ = reference(ts, 1.0, inf=True)
    norm, factor = gradient_norm(ts, 1.0, norm_type=math.inf)
    assert norm.item() == total and abs(factor.item() - 1 / (total + 1e-6)) <= 4 * 2.0 ** -24
    before = flat.clone()
    clip_gradients(ts, 0.5)
    assert torch.equal(flat[5000:5003], before[5000:5003]) and torch.equal(flat[90000:], before[90000:])
    total, f = reference([before[1:5000], before[5003:5004], before[6001:90000]], 0.5)
    assert (flat[6001:90000].double() - before[6001:90000].double() * f).abs().max().item() <= 2.0 ** -8 * 5 * f


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e30, 3e38])
def test_extremes(scale):
    """Squares outside the fp32 range."""
    ts = [torch.full((1000,), scale, device=DEV), torch.full((3,), -scale, device=DEV)]
    total, factor = reference(ts, 1.0)
    norm = clip_gradients(ts, 1.0)
    if total > torch.finfo(torch.float32).max:
        assert math.isinf(norm.item()) and not bool(ts[0].any())
    else:
        assert abs(norm.item() - total) <= 3 * 2.0 ** -24 * total
        assert abs(ts[0][0].item() - scale * factor) <= 12 * 2.0 ** -24 * scale * factor


@pytest.mark.gpu
def test_nonfinite_as_torch():
    for bad in (math.nan, math.inf):
        ts = tensors([(50,), (20000,)], [torch.float32])
        ts[1][777] = bad
        params = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
        for p, t in zip(params, ts):
            p.grad = t.clone()
        ref = torch.nn.utils.clip_grad_norm_(params, 1.0)
        norm = clip_gradients(ts, 1.0)
        assert torch.equal(norm.isnan(), ref.isnan()) and torch.equal(norm.isinf(), ref.isinf())
        for p, t in zip(params, ts):
            assert torch.equal(p.grad.isnan(), t.isnan()) and torch.equal(p.grad.nan_to_num(5.0), t.nan_to_num(5.0))


@pytest.mark.gpu
def test_parameters_and_optimizer():
    """clip_grad_norm_ on parameters, and the factor handed to AdamWRequant instead."""
    def params():
        ps = [torch.nn.Parameter(t) for t in tensors([(300, 256), (256,), (70, 3)], [torch.float32], 1)]
        for p, g in zip(ps, tensors([(300, 256), (256,), (70, 3)], [torch.float32], 2)):
            p.grad = g
        return ps
    a, b = params(), params()
    extra = torch.nn.Parameter(torch.zeros(4, device=DEV))  # no gradient
    norm = clip_grad_norm_(a + [extra], 1.0)
    AdamWRequant(a, lr=0.1).step()
    n2, factor = gradient_norm([p.grad for p in b], 1.0)
    AdamWRequant(b, lr=0.1).step(clip_coef=factor)
    assert torch.equal(norm, n2)
    for p, q in zip(a, b):
        assert (p - q).abs().max().item() <= 1e-6 * 3
    assert clip_grad_norm_([extra], 1.0).item() == 0.0


@pytest.mark.gpu
def test_gradients_of_other_layouts():
    """A transposed gradient, an empty one, and one tensor as the parameters."""
    p = torch.nn.Parameter(torch.zeros(50, 70, device=DEV))
    g = tensors([(70, 50)], [torch.float32])[0].t()
    p.grad = torch.empty(70, 50, device=DEV).t()
    p.grad.copy_(g)
    assert not p.grad.is_contiguous()
    e = torch.nn.Parameter(torch.zeros(0, 3, device=DEV))
    e.grad = torch.zeros(0, 3, device=DEV)
    total, factor = reference([g], 1.0)
    norm = clip_grad_norm_([p, e], 1.0)
    assert abs(norm.item() - total) <= 3 * 2.0 ** -24 * total
    assert (p.grad.double() - g.double() * factor).abs().max().item() <= 12 * 2.0 ** -24 * 5 * factor
    assert abs(clip_grad_norm_(p, 2.0).item() - 1.0) <= 1e-5
    assert clip_grad_norm_(e, 1.0).item() == 0.0


@pytest.mark.gpu
def test_refusals():
    t = torch.ones(4, 4, device=DEV)
    with pytest.raises(ValueError):
        clip_gradients([], 1.0)
    with pytest.raises(ValueError):
        clip_gradients([t], 1.0, norm_type=3)
    with pytest.raises(ValueError):
        clip_gradients([t], 1.0, loss_scale=0.0)
    with pytest.raises(ValueError):
        clip_gradients([t], 1.0, out=[t, t])
    with pytest.raises(ValueError):
        clip_gradients([t], 1.0, out=[t.bfloat16()])
    with pytest.raises(ValueError):
        clip_gradients([t.t()[:, :2]], 1.0)
    with pytest.raises(ValueError):
        clip_gradients([t.to_sparse()], 1.0)
    with pytest.raises(TypeError):
        clip_gradients([t.double()], 1.0)
    with pytest.raises(RuntimeError):
        clip_gradients([t.cpu()], 1.0)
