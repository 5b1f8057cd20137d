"""TokenChannelLinear against the float layer: y, dX and dW of ordinary values.

A code is within half a step of its value (a step is the row's largest magnitude / 127; two fp32 roundings add
2^-22 of it). y and dX carry the error of both operands of their products, dW too; the int32 sums are exact and
at most five fp32 roundings follow."""

import pytest
import torch

from ksdraft_amd.kernels import TokenChannelLinear

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def step(t):
    return t.abs().amax(1, keepdim=True) / 127 * (1 + 2.0 ** -20)


def check(got, a, b, ea, eb, dtype, extra=0.0):
    """got against a @ b.T + extra, whose operands are within ea and eb."""
    ref = a @ b.t() + extra
    bound = ea @ (b.abs() + eb).t() + a.abs() @ eb.t()
    bound = bound + 5 * 2.0 ** -24 * ((a.abs() + ea) @ (b.abs() + eb).t() + abs(extra))
    bound = bound + EPS[dtype] * (ref.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert bool(((got.double().cpu() - ref).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N", [(1, 64, 48), (5, 200, 31), (257, 512, 1536), (1000, 1536, 512), (2047, 333, 597)])
def test_against_float(M, K, N, dtype):
    g = torch.Generator().manual_seed(M)
    lin = TokenChannelLinear(K, N).to(DEV)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=g) * K ** -0.5)
        lin.bias.copy_(torch.randn(N, generator=g))
    x = torch.randn(M, K, generator=g).to(dtype).to(DEV).requires_grad_(True)
    # gradients whose size differs from token to token and from channel to channel
    dy = (torch.randn(M, N, generator=g) * 2.0 ** -torch.randn(M, 1, generator=g).abs() * 2.0 ** -torch.randn(N, generator=g).abs())
    dy = dy.to(dtype).to(DEV)
    y = lin(x)
    y.backward(dy)
    xc, w, d, b = (t.detach().double().cpu() for t in (x, lin.weight, dy, lin.bias))
    ew, ex = (step(w) / 2).expand_as(w), (step(xc) / 2).expand_as(xc)
    check(y, xc, w, ex, ew, dtype, b)
    sw, sx = step(w), step(xc)
    ones = torch.ones(1, dtype=torch.float64)
    # dY * sw is quantized per row, dY * sx per column; the products' other operand are the codes
    check(x.grad, d * sw.t(), (w / sw).t(), (step(d * sw.t()) / 2).expand_as(d), 0.5 * ones.expand(K, N), dtype)
    dsx = (d * sx).t()
    check(lin.weight.grad, dsx, (xc / sx).t(), (step(dsx) / 2).expand_as(dsx), 0.5 * ones.expand(K, M), torch.float32)
    assert bool(((lin.bias.grad.double().cpu() - d.sum(0)).abs() <= (M + 1) * 2.0 ** -24 * d.abs().sum(0)).all())
