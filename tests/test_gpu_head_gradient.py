"""The gradients of a converted model's vocabulary head (TokenChannelLinear with group_gradient) under cross
entropy against the float gradients of the same dY.

A code is within half a step of its value, and a value below half a step becomes 0, so it is off by at most
min(|v|, step / 2); a step is the group's largest magnitude / 127, rounded to fp16 (2^-11, and 2^-25 below its
normal numbers, which 127 codes see; dY is brought to 2^20 before). W and X pass two such roundings, the second
one over the first one's result. The products add at most one fp32 rounding per group and operation."""

import math

import pytest
import torch
import torch.nn.functional as F

from ksdraft_amd.config import KSDraftConfig
from ksdraft_amd.kernels import Int8Linear, TokenChannelLinear
from ksdraft_amd.kernels.linear import w8a8_linear_backward
from ksdraft_amd.kernels.quant import quantize_dual
from ksdraft_amd.model import KSDraftModel, to_token_channel

pytestmark = pytest.mark.gpu
DEV = "cuda"
UP = 1 + 2.0 ** -11


def steps(t, least):
    """Each value's step: its group of 128 in the row, in fp64 on the CPU."""
    rows, n = t.shape
    a = F.pad(t.abs(), (0, -n % 128)).view(rows, -1, 128).amax(2) / 127 * UP + 2 * 127 * least
    return a.repeat_interleave(128, 1)[:, :n]


def off(v):
    return torch.minimum(v.abs(), steps(v, 2.0 ** -25 * v.abs().max() / 2.0 ** 20) / 2)


def twice(t):
    """How far an operand (rows contracted) is off after the rounding along its rows and then its columns."""
    first = steps(t, 2.0 ** -25) / 2
    return first + steps((t.abs() + first).t(), 2.0 ** -25).t() / 2


def bounds(dy, x, w):
    """dX and dW in fp64, and how far int8 ones may be off."""
    ew, ex, gx, gw = twice(w), twice(x), off(dy), off(dy.t()).t()
    dx, dw = dy @ w, dy.t() @ x
    bx = gx @ (w.abs() + ew) + dy.abs() @ ew
    bw = gw.t() @ (x.abs() + ex) + dy.t().abs() @ ex
    n = (dy.shape[1] + dy.shape[0]) / 128 + 8
    return dx, dw, bx + n * 2.0 ** -24 * (dy.abs() @ w.abs() + bx), bw + n * 2.0 ** -24 * (dy.abs().t() @ x.abs() + bw)


def head_of(V, d, seed):
    """A converted model's head: rows of the table share a direction, as a trained one's do."""
    g = torch.Generator().manual_seed(seed)
    model = KSDraftModel(KSDraftConfig(vocab_size=V, layers=1, d_model=d, rosa_streams=32, ks3_charts=128)).to(DEV)
    head = to_token_channel(model).head
    with torch.no_grad():
        head.weight.copy_((torch.randn(V, d, generator=g) + torch.randn(d, generator=g)) * 0.02)
    return head, g


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -13, 1e-30])
@pytest.mark.parametrize("M,V,d", [(200, 20000, 256), (65, 30011, 192), (1, 20000, 256)])
def test_cross_entropy(M, V, d, scale):
    head, g = head_of(V, d, M)
    x = (F.layer_norm(torch.randn(M, d, generator=g), (d,)) + torch.randn(d, generator=g) / 2).to(DEV).requires_grad_(True)
    tgt = torch.randint(0, V, (M,), generator=g).to(DEV)
    y = head(x)
    y.retain_grad()
    (F.cross_entropy(y, tgt, reduction="sum") * scale).backward()
    dy, xc, w = (t.detach().double().cpu() for t in (y.grad, x, head.weight))
    dx, dw, bx, bw = bounds(dy, xc, w)
    # the probabilities' part is far above the bound, so a gradient without it does not pass
    soft = dx + w[tgt.cpu()] * -dy.gather(1, tgt.cpu()[:, None])
    assert bx.mean() < 0.25 * soft.abs().mean()
    assert bool(((x.grad.double().cpu() - dx).abs() <= bx).all())
    assert bool(((head.weight.grad.double().cpu() - dw).abs() <= bw).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead,K,N", [((1,), 128, 1), ((2, 33), 200, 77), ((300,), 512, 640), ((129,), 17, 20)])
def test_as_the_group_scaled_layer(lead, K, N, dtype):
    """The gradients are those of the group-128 operands of dY brought to 2^20, brought back."""
    g = torch.Generator().manual_seed(N)
    lin = TokenChannelLinear.from_float(torch.nn.Linear(K, N).to(DEV), group_gradient=True)
    plain = TokenChannelLinear.from_float(lin)
    x = torch.randn(*lead, K, generator=g).to(dtype).to(DEV).requires_grad_(True)
    res = torch.randn(*lead, N, generator=g).to(dtype).to(DEV).requires_grad_(True)
    y = lin(x, residual=res)
    assert torch.equal(y, plain(x, residual=res))
    dy = (torch.randn(*lead, N, generator=g) * 2.0 ** -torch.randint(0, 12, (*lead, N), generator=g)).to(dtype).to(DEV)
    y.backward(dy)
    g2 = dy.reshape(-1, N)
    g2 = g2.float() if dtype == torch.float16 else g2
    s = 2.0 ** (20 - math.floor(math.log2(g2.abs().max().item())))
    xt, wt = quantize_dual(x.detach().reshape(-1, K), t_from_codes=True)[2:], quantize_dual(lin.weight.detach(), t_from_codes=True)[2:]
    dx, dw, db = w8a8_linear_backward(g2 * s, None, None, None, None, xt=xt, wt=wt, want_db=True)
    assert torch.equal(x.grad, (dx / s).to(dtype).reshape(x.shape)) and torch.equal(lin.weight.grad, dw / s)
    assert torch.equal(lin.bias.grad, db / s) and torch.equal(res.grad, dy)


def test_scale_of_the_gradient():
    """A power of two passes through; the group-scaled layer alone loses the small one."""
    lin = TokenChannelLinear.from_float(torch.nn.Linear(256, 384, bias=False).to(DEV), group_gradient=True)
    g = torch.Generator().manual_seed(0)
    x, dy = torch.randn(150, 256, generator=g).to(DEV), torch.randn(150, 384, generator=g).to(DEV)
    first = None
    for s in (1.0, 2.0 ** -60, 2.0 ** 60, 2.0 ** -100):
        xg = x.clone().requires_grad_(True)
        lin.weight.grad = None
        lin(xg).backward(dy * s)
        got = [xg.grad / s, lin.weight.grad / s]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nonfinite_gradients_are_not_hidden(bad):
    lin = TokenChannelLinear.from_float(torch.nn.Linear(256, 300).to(DEV), group_gradient=True)
    x = torch.randn(140, 256, generator=torch.Generator().manual_seed(0)).to(DEV).requires_grad_(True)
    dy = torch.ones(140, 300, device=DEV)
    dy[7, 9] = bad
    lin(x).backward(dy)
    assert all(bool(t.isnan().all()) for t in (x.grad, lin.weight.grad, lin.bias.grad))


def test_parts_and_empties():
    lin = TokenChannelLinear.from_float(torch.nn.Linear(128, 200).to(DEV), group_gradient=True)
    g = torch.Generator().manual_seed(0)
    x, dy = torch.randn(50, 128, generator=g).to(DEV), torch.randn(50, 200, generator=g).to(DEV)
    lin(xg := x.clone().requires_grad_(True)).backward(dy)
    whole = [xg.grad, lin.weight.grad, lin.bias.grad]
    lin.zero_grad()
    lin(x).backward(dy)  # dW and db alone
    assert torch.equal(lin.weight.grad, whole[1])
    lin.requires_grad_(False)
    lin(xg2 := x.clone().requires_grad_(True)).backward(dy)
    assert torch.equal(xg2.grad, whole[0])
    lin.requires_grad_(True)
    lin.weight.requires_grad_(False)
    lin.zero_grad()
    lin(x).backward(dy)  # db alone
    assert (lin.bias.grad - whole[2]).abs().max().item() <= 100 * 2.0 ** -24 * dy.abs().sum(0).max().item()
    lin.requires_grad_(True)
    lin.zero_grad()
    none = torch.empty(0, 128, device=DEV, requires_grad=True)
    lin(none).sum().backward()
    assert none.grad.shape == (0, 128) and not bool(lin.weight.grad.any()) and not bool(lin.bias.grad.any())
    lin.zero_grad()
    lin(xg := x.clone().requires_grad_(True)).backward(torch.zeros_like(dy))
    assert not bool(xg.grad.any()) and not bool(lin.weight.grad.any())
    with pytest.raises(RuntimeError):
        lin(xg).sum().backward(create_graph=True)
        xg.grad.sum().backward()


def test_master_changed_before_the_backward():
    """The backward reads the master: one that has changed since is refused."""
    lin = TokenChannelLinear.from_float(torch.nn.Linear(128, 200).to(DEV), group_gradient=True)
    y = lin(torch.ones(3, 128, device=DEV, requires_grad=True))
    with torch.no_grad():
        lin.weight.mul_(2)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_int8_head_agrees():
    """The group-scaled head's gradients from the same float head lie within the two bounds' sum."""
    head, g = head_of(20000, 256, 3)
    other = Int8Linear(256, 20000, bias=False).to(DEV)
    other.weight = head.weight
    x = torch.randn(90, 256, generator=g).to(DEV)
    dy = torch.randn(90, 20000, generator=g).to(DEV)
    grads = []
    for lin in (head, other):
        head.weight.grad = None
        xg = x.clone().requires_grad_(True)
        lin(xg).backward(dy)
        grads.append((xg.grad.double().cpu(), head.weight.grad.double().cpu()))
    _, _, bx, bw = bounds(dy.double().cpu(), x.double().cpu(), head.weight.detach().double().cpu())
    assert bool(((grads[0][0] - grads[1][0]).abs() <= 2 * bx).all()) and bool(((grads[0][1] - grads[1][1]).abs() <= 2 * bw).all())


def test_captured_step():
    """Captured, the layer's calls give the eager bits on every replay."""
    lin = TokenChannelLinear.from_float(torch.nn.Linear(256, 1000).to(DEV), group_gradient=True)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(300, 256, generator=g).to(DEV).requires_grad_(True)
    dy = torch.randn(300, 1000, generator=g).to(DEV)

    def step():
        y = lin(x)
        return [y.detach(), *torch.autograd.grad(y, [x, lin.weight, lin.bias], dy)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        dy.mul_(0.5)  # another lift each time
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))
        torch.cuda.synchronize()
