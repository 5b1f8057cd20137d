"""Low-rank adapters, forward and backward, against the formulas in 64 bits on the CPU.

Bounds, u = 2^-24: a sum of k products in fp32 in any order is off by at most k u of the sum of magnitudes (twice that
is allowed: a matrix instruction may round its inner sums on its own). h enters the second product as two 16-bit
parts: (u_T)^2 of it is lost (bf16: 2^-16; fp16: 2^-22, and 2^-24 of the row's largest where the rest is
subnormal), fp32 nothing. The scale, the mask and base are one operation each; y is rounded once (u_T).
Magnitudes are propagated with the values: |A|, |B| and |x| in place of A, B and x."""

import math

import pytest
import torch

from ksdraft_amd.kernels.adapters import adapt, adapter_linear, adapter_linear_backward, adapter_linear_train
from ksdraft_amd.kernels.dropout import dropout
from tests.philox import mask

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24
UT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
PART = {torch.float32: U, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -21}


def case(M, K, N, r, n, dtype, seed=0, lead=None, none=True, outliers=True):
    g = torch.Generator().manual_seed(seed)
    dt = TYPES[dtype]

    def randn(*s, scale=1.0):
        return (torch.randn(*s, generator=g) * scale).to(dt)
    lead = lead or (M,)
    x = torch.randn(*lead, K, generator=g)
    if outliers:
        x = x * (1 + 9 * (torch.rand(K, generator=g) < 0.05))
    index = torch.randint(-1 if none else 0, n, lead, generator=g)
    return dict(x=x.to(dt), a=randn(n, r, K, scale=K ** -0.5), b=randn(n, N, r, scale=r ** -0.5), index=index,
                scales=0.5 + torch.rand(n, generator=g), base=randn(*lead, N), dy=randn(*lead, N), dx_base=randn(*lead, K))


def to(c, *names):
    return [None if c[k] is None else c[k].to(DEV) for k in names]


def forward(c, keep=None, value=lambda t: t):
    """h and y in fp64 of value(inputs); value = abs gives the magnitudes."""
    x = value(c["x"].double()).reshape(-1, c["x"].shape[-1])
    if keep is not None:
        x = x * keep
    M, n = x.shape[0], c["a"].shape[0]
    idx = c["index"].reshape(-1)
    idx = idx.repeat_interleave(M // max(1, idx.numel())) if idx.numel() != M else idx
    h = torch.zeros(M, c["a"].shape[1], dtype=torch.float64)
    y = torch.zeros(M, c["b"].shape[1], dtype=torch.float64)
    for i in range(n):
        at = idx == i
        s = 1.0 if c["scales"] is None else float(c["scales"][i])
        h[at] = x[at] @ value(c["a"][i].double()).t() * s
        y[at] = h[at] @ value(c["b"][i].double()).t()
    return x, idx, h, y


def close(got, want, bound, dt):
    """|got - want| <= bound + one rounding of the result."""
    got, want = got.double().cpu().reshape(want.shape), want
    bad = (got - want).abs() > bound * 1.001 + UT[dt] * (want.abs() + bound) + 1e-37
    if dt == torch.float16:  # below its normal range a half step is 2^-25
        bad &= (got - want).abs() > bound * 1.001 + 2.0 ** -25
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}, worst {float(((got - want).abs() / (bound + 1e-37)).max())}"


def spread(h):
    return h.abs().amax(1, keepdim=True) * 2.0 ** -23


def check_y(got, c, keep=None):
    dt = c["x"].dtype
    _, idx, h, y = forward(c, keep)
    _, _, hm, ym = forward(c, keep, torch.abs)
    K, r = c["a"].shape[2], c["a"].shape[1]
    bound = ym * (2 * (K + r + 4) * U + PART[dt])
    if dt == torch.float16:
        bm = c["b"].double().abs()
        pad = torch.zeros_like(bound)
        for i in range(bm.shape[0]):
            pad[idx == i] = spread(hm[idx == i]) * bm[i].sum(1)
        bound = bound + pad
    if c["base"] is not None:
        base = c["base"].double().reshape(y.shape)
        y, bound = y + base, bound + 2 * U * (ym + base.abs())
    none = (idx < 0) | (idx >= c["a"].shape[0])
    assert torch.equal(got.cpu().reshape(y.shape)[none], (torch.zeros_like(y, dtype=dt) if c["base"] is None else
                                                          c["base"].reshape(y.shape))[none])
    close(got, y, bound, dt)


SHAPES = [(1, 1, 1, 1, 1), (1, 64, 64, 8, 3), (3, 33, 65, 4, 2), (17, 597, 130, 16, 4), (40, 256, 1792, 16, 40), (5, 1536, 512, 32, 2),
          (64, 100, 70, 24, 7), (33, 130, 257, 64, 3), (9, 72, 200, 128, 2), (300, 128, 96, 16, 3), (513, 96, 193, 65, 5), (31, 4, 3, 7, 2)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,N,r,n", SHAPES)
def test_forward(M, K, N, r, n, dtype):
    c = case(M, K, N, r, n, dtype, seed=M + K)
    check_y(adapter_linear(*to(c, "x", "a", "b", "index", "scales", "base")), c)
    c["base"] = c["scales"] = None
    check_y(adapter_linear(*to(c, "x", "a", "b"), c["index"].int().to(DEV)), c)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_sequences_and_many_rows(dtype):
    c = case(0, 200, 150, 16, 3, dtype, seed=2, lead=(6, 37))
    c["index"] = torch.tensor([0, 2, -1, 1, 1, 5])  # 5: none
    check_y(adapter_linear(*to(c, "x", "a", "b", "index", "scales", "base")), c)
    c = case(9000, 64, 72, 8, 2, dtype, seed=3)
    check_y(adapter_linear(*to(c, "x", "a", "b", "index", "scales", "base")), c)
    c = case(0, 64, 72, 8, 5, dtype, seed=4, lead=(3, 5, 7))
    c["index"] = c["index"][:, :, 0]
    check_y(adapter_linear(*to(c, "x", "a", "b", "index", "scales", "base")), c)


# tokens listed by adapter; a narrow product in parts; 32 rows a workgroup, with and without lists, at each block of ranks;
# rows in parts of their columns; more adapters than tokens; odd widths of each
FORMS = [(700, 300, 1000, 24, 5), (701, 301, 1001, 24, 5), (700, 301, 1000, 4, 200), (1500, 130, 515, 100, 3), (40, 4500, 130, 8, 2),
         (300, 4097, 257, 16, 1), (130, 5000, 1793, 40, 3), (8200, 72, 136, 16, 1), (8200, 71, 135, 16, 1), (8200, 40, 72, 30, 1),
         (8200, 40, 72, 64, 1), (9000, 130, 170, 16, 3), (9000, 131, 171, 33, 3), (70, 256, 1792, 16, 1), (100, 64, 6869, 7, 300),
         (2, 5000, 3000, 16, 3)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,N,r,n", FORMS)
def test_forms(M, K, N, r, n, dtype):
    c = case(M, K, N, r, n, dtype, seed=M + r)
    check_y(adapter_linear(*to(c, "x", "a", "b", "index", "scales", "base")), c)
    backward_case(c, 0.2 if M % 2 else 0.0, seed=5, stream=M)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_odd_addresses(dtype, offset):
    """Tensors that begin on each half word, at even and odd widths."""
    for K, N, r in ((64, 70, 8), (65, 71, 8), (64, 71, 3), (65, 70, 16)):
        c = case(37, K, N, r, 3, dtype, seed=offset + K + N, none=True)
        moved = {}
        for k in ("x", "a", "b", "base"):
            t = c[k]
            room = torch.full((t.numel() + 8,), math.nan, dtype=t.dtype, device=DEV)
            moved[k] = room[offset:offset + t.numel()].view(t.shape)
            moved[k].copy_(t)
        index, scales = to(c, "index", "scales")
        room = torch.full((37 * N + 8,), 7.0, dtype=c["x"].dtype, device=DEV)
        out = room[offset:offset + 37 * N].view(37, N)
        check_y(adapter_linear(moved["x"], moved["a"], moved["b"], index, scales, moved["base"], out=out), c)
        assert bool((room[:offset] == 7).all()) and bool((room[offset + 37 * N:] == 7).all())
        y, saved = adapter_linear_train(moved["x"], moved["a"], moved["b"], index, scales, moved["base"])
        check_y(y, c)
        room = torch.full((37 * N + 8,), math.nan, dtype=c["x"].dtype, device=DEV)
        dy = room[offset:offset + 37 * N].view(37, N)
        dy.copy_(c["dy"])
        plain = adapter_linear_backward(c["dy"].to(DEV), saved)
        for p, q in zip(adapter_linear_backward(dy, saved), plain):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_an_adapter_is_its_own(dtype):
    """NaN and inf in one adapter, or one token, reach nobody else's rows."""
    c = case(70, 96, 80, 16, 4, dtype, seed=5)
    want = adapter_linear(*to(c, "x", "a", "b", "index", "scales", "base")).cpu()
    bad = {k: v.clone() for k, v in c.items()}
    bad["a"][1], bad["b"][2] = math.nan, math.inf
    bad["x"][7] = math.inf
    got = adapter_linear(*to(bad, "x", "a", "b", "index", "scales", "base")).cpu()
    fine = (c["index"] != 1) & (c["index"] != 2)
    fine[7] = False
    assert torch.equal(got[fine], want[fine]) and bool(fine.any())
    assert not bool(torch.isfinite(got[(c["index"] == 1)].float()).any())
    # the gradients of the others too
    x, a, b, index, scales = to(bad, "x", "a", "b", "index", "scales")
    x[7] = 0
    _, saved = adapter_linear_train(x, a, b, index, scales)
    dx, da, db = adapter_linear_backward(bad["dy"].to(DEV), saved)
    for i in (0, 3):
        assert bool(torch.isfinite(da[i]).all()) and bool(torch.isfinite(db[i]).all())
    assert bool(torch.isfinite(dx[fine.to(DEV)].float()).all())


def test_large_and_small_values():
    """fp16 rows whose h is far past fp16's range, and far below it."""
    c = case(40, 64, 48, 16, 2, "fp16", seed=6, none=False, outliers=False)
    c["x"] = (c["x"].float() * torch.logspace(-6, 3.5, 40)[:, None]).half()
    c["a"] = (c["a"].float() * 2000).half()
    c["b"] = (c["b"].float() * 1e-4).half()
    check_y(adapter_linear(*to(c, "x", "a", "b", "index", "scales", "base")), c)
    c = case(8, 64, 48, 16, 2, "bf16", seed=6, none=False)
    c["x"] = (c["x"].float() * 1e20).bfloat16()
    check_y(adapter_linear(*to(c, "x", "a", "b", "index", "scales", "base")), c)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_layouts(dtype):
    c = case(50, 64, 72, 8, 3, dtype, seed=8)
    x, a, b, index, scales, base = to(c, "x", "a", "b", "index", "scales", "base")
    want = adapter_linear(x, a, b, index, scales, base)
    wide = torch.zeros(50, 75, dtype=x.dtype, device=DEV)
    wide[:, 5:69] = x
    assert torch.equal(adapter_linear(wide[:, 5:69], a, b, index, scales, base), want)
    assert torch.equal(adapter_linear(x.t().contiguous().t(), a.transpose(1, 2).contiguous().transpose(1, 2), b, index,
                                      scales, base), want)
    wb = torch.zeros(50, 80, dtype=x.dtype, device=DEV)
    wb[:, 1:73] = base
    assert torch.equal(adapter_linear(x, a, b, index, scales, wb[:, 1:73]), want)
    out = base.clone()
    was = out._version
    assert adapter_linear(x, a, b, index, scales, out, out=out) is out and torch.equal(out, want) and out._version > was
    assert adapter_linear(x[:0], a, b, index[:0], scales, base[:0]).shape == (0, 72)
    assert torch.equal(adapter_linear(x, a, b, index, scales, base), want)  # the same bits


def backward_case(c, p=0.0, seed=0, stream=0, base=True):
    dt = c["x"].dtype
    x2 = c["x"].reshape(-1, c["x"].shape[-1])
    M, K = x2.shape
    n, N, r = c["b"].shape
    keep = mask(M, K, p, seed, stream).double() if p else None
    y, saved = adapter_linear_train(*to(c, "x", "a", "b", "index", "scales", "base"), dropout=p, seed=seed, stream=stream)
    check_y(y, c, keep)
    dx, da, db = adapter_linear_backward(c["dy"].to(DEV), saved, base=c["dx_base"].to(DEV) if base else None)
    out = {}
    for name, value in (("value", lambda t: t), ("size", torch.abs)):
        x, idx, h, _ = forward(c, keep, value)
        dy = value(c["dy"].double()).reshape(M, N)
        g = torch.zeros(M, r, dtype=torch.float64)
        wx, wa, wb = torch.zeros(M, K, dtype=torch.float64), torch.zeros(n, r, K, dtype=torch.float64), torch.zeros(n, N, r, dtype=torch.float64)
        for i in range(n):
            at = idx == i
            s = 1.0 if c["scales"] is None else float(c["scales"][i])
            g[at] = dy[at] @ value(c["b"][i].double()) * s
            wx[at] = g[at] @ value(c["a"][i].double())
            wa[i], wb[i] = g[at].t() @ x[at], dy[at].t() @ h[at]
        out[name] = (wx * keep if p else wx, wa, wb, g, idx)
    (wx, wa, wb, g, idx), (sx, sa, sb, gm, _) = out["value"], out["size"]
    bound = sx * (2 * (N + r + 5) * U + PART[dt])
    if dt == torch.float16:
        am = c["a"].double().abs()
        for i in range(n):
            at = idx == i
            pad = spread(gm[at]) * am[i].sum(0)
            bound[at] += pad * keep[at] if p else pad
    if base:
        db0 = c["dx_base"].double().reshape(M, K)
        wx, bound = wx + db0, bound + 2 * U * (sx + db0.abs())
    close(dx, wx, bound, dt)
    # the parts of g and h that enter these products keep at least 24 bits
    close(da, wa, sa * 2 * (N + M + 8) * U, torch.float32)
    close(db, wb, sb * 2 * (K + M + 8) * U, torch.float32)
    return saved


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("M,K,N,r,n", SHAPES)
def test_backward(M, K, N, r, n, p, dtype):
    backward_case(case(M, K, N, r, n, dtype, seed=M + N), p, seed=(1 << 63) + 5, stream=9, base=M != 17)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_backward_many_rows(dtype):
    """Lists of several pieces, one token's, none's, and exactly one piece."""
    c = case(1500, 40, 72, 8, 6, dtype, seed=12)
    index = torch.full((1500,), -1)
    index[100:700], index[700:956], index[1000], index[1001:1258] = 1, 3, 4, 5
    c["index"] = index[torch.randperm(1500, generator=torch.Generator().manual_seed(0))]
    backward_case(c, 0.1, seed=77)
    c["index"] = index
    backward_case(c)
    c = case(0, 40, 72, 8, 3, dtype, seed=13, lead=(4, 300))
    c["index"] = torch.tensor([1, 1, -1, 0])
    backward_case(c, 0.5, seed=3)
    c["scales"] = None
    c["index"][:] = -1
    saved = backward_case(c)
    _, da, db = adapter_linear_backward(c["dy"].to(DEV), saved)
    assert not bool(da.any()) and not bool(db.any())


def test_backward_parts_and_empty():
    c = case(90, 64, 48, 8, 2, "bf16", seed=14)
    x, a, b, index, scales, dy = to(c, "x", "a", "b", "index", "scales", "dy")
    _, saved = adapter_linear_train(x, a, b, index, scales)
    dx, da, db = adapter_linear_backward(dy, saved)
    only = adapter_linear_backward(dy, saved, need_dab=False)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None
    only = adapter_linear_backward(dy, saved, need_dx=False)
    assert only[0] is None and torch.equal(only[1], da) and torch.equal(only[2], db)
    assert adapter_linear_backward(dy, saved, need_dx=False, need_dab=False) == (None, None, None)
    wide = torch.zeros(90, 61, dtype=dy.dtype, device=DEV)
    wide[:, 6:54] = dy
    again = adapter_linear_backward(wide[:, 6:54], saved)
    for p, q in zip(again, (dx, da, db)):
        assert torch.equal(p, q)
    _, saved = adapter_linear_train(x[:0], a, b, index[:0], scales)
    dx, da, db = adapter_linear_backward(dy[:0], saved)
    assert dx.shape == (0, 64) and not bool(da.any()) and not bool(db.any())


def test_gradients_against_differences():
    """adapt is linear in x, in a and in b, so a difference of outputs is the derivative up to the outputs'
    roundings: with fp32, steps as large as the values and sums of 72 outputs, 1e-4 of the magnitudes."""
    c = case(50, 64, 72, 8, 3, "fp32", seed=15)
    x, a, b, base = (t.requires_grad_() for t in to(c, "x", "a", "b", "base"))
    index, scales, dy = to(c, "index", "scales", "dy")

    def f(x, a, b, base):
        return (adapt(x, a, b, index, scales, base, 0.25, 31, 2).double() * dy.double()).sum()
    grads = torch.autograd.grad(f(x, a, b, base), (x, a, b, base))
    g = torch.Generator().manual_seed(1)
    for k in range(4):
        args = [x.detach(), a.detach(), b.detach(), base.detach()]
        step = torch.randn(args[k].shape, generator=g).to(DEV) * args[k].std()
        moved = list(args)
        moved[k] = args[k] + step
        with torch.no_grad():
            diff = float(f(*moved) - f(*args))
        want = float((grads[k].double() * step.double()).sum())
        size = float((grads[k].double() * step.double()).abs().sum()) + float((dy.abs().double() * (1 + c["base"].to(DEV).abs().double())).sum())
        assert abs(diff - want) <= 1e-4 * size, k


def test_dropout_is_the_operator():
    """x~ is kernels.dropout's: an adapter that passes x through shows it."""
    for dtype, dt in TYPES.items():
        x = torch.randn(33, 24, generator=torch.Generator().manual_seed(1)).to(dt).to(DEV)
        eye = torch.eye(24, dtype=dt, device=DEV)[None]
        y, _ = adapter_linear_train(x, eye, eye, torch.zeros(33, dtype=torch.int64, device=DEV), dropout=0.4, seed=9, stream=4)
        want = dropout(x, 0.4, 9, 4)
        assert torch.equal(y == 0, want == 0)
        assert bool(((y - want).abs() <= 3 * UT[dt] * want.abs()).all())


def test_captured_step():
    c = case(70, 64, 48, 8, 3, "bf16", seed=16)
    x, index, scales, dy = to(c, "x", "index", "scales", "dy")
    a, b = (t.requires_grad_() for t in to(c, "a", "b"))
    seed = torch.tensor([3], device=DEV)

    def step():
        y = adapt(x, a, b, index, scales, None, 0.2, seed, 1)
        seed.add_(1)
        return (y.detach(), *torch.autograd.grad(y, (a, b), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for n in range(4):
        at = int(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert int(seed) == at + 1
        y = adapt(x, a, b, index, scales, None, 0.2, at, 1)
        for p, q in zip(kept, (y, *torch.autograd.grad(y, (a, b), dy))):
            assert torch.equal(p, q)
        x.add_(0.125)


def test_two_graphs_and_streams():
    cs = [case(65, 96, 80, 16, 3, "bf16", seed=s) for s in (20, 21)]
    args = [to(c, "x", "a", "b", "index", "scales", "base") for c in cs]
    want = [adapter_linear(*a) for a in args]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = adapter_linear(*args[1])
    mine = adapter_linear(*args[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(mine, want[0]) and torch.equal(other, want[1])
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, a in zip(graphs, args):
        with torch.cuda.graph(g):
            outs.append(adapter_linear(*a))
    for _ in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_refusals():
    c = case(6, 16, 24, 4, 2, "fp32")
    x, a, b, index, scales, base = to(c, "x", "a", "b", "index", "scales", "base")
    big = torch.zeros(1, 129, 16, device=DEV), torch.zeros(1, 24, 129, device=DEV)
    for f in (lambda: adapter_linear(x[0], a, b, index[:0]), lambda: adapter_linear(x, a[:1], b, index), lambda: adapter_linear(x, a, b[:, :, :3], index),
              lambda: adapter_linear(x[:, :8], a, b, index), lambda: adapter_linear(x, a, b, index[:5]), lambda: adapter_linear(x, a, b, index, scales[:1]),
              lambda: adapter_linear(x, a, b, index, scales.double()), lambda: adapter_linear(x, a, b, index, scales, base[:, :8]),
              lambda: adapter_linear(x, a, b, index, scales, base.half()), lambda: adapter_linear(x, *big, index),
              lambda: adapter_linear(x, a[:0], b[:0], index), lambda: adapter_linear(x, a, b, index, out=base[:, :8]),
              lambda: adapter_linear(base[:, :16], a, b, index, out=base), lambda: adapter_linear_train(x, a, b, index, dropout=1.5)):
        with pytest.raises(ValueError):
            f()
    flat = torch.zeros(6 * 24 + 24, device=DEV)
    with pytest.raises(ValueError):  # base one row further than out
        adapter_linear(x, a, b, index, base=flat[24:].view(6, 24), out=flat[:144].view(6, 24))
    for f in (lambda: adapter_linear(x, a.half(), b.half(), index), lambda: adapter_linear(x, a, b, index.float()),
              lambda: adapter_linear(x.double(), a.double(), b.double(), index)):
        with pytest.raises(TypeError):
            f()
    _, saved = adapter_linear_train(x, a, b, index)
    with pytest.raises(ValueError):
        adapter_linear_backward(base[:, :8], saved)
    with pytest.raises(ValueError):
        adapter_linear_backward(base.half(), saved)
    with pytest.raises(ValueError):
        adapter_linear_backward(base, saved, base=base)
    with pytest.raises(RuntimeError):
        adapter_linear(x.cpu(), a, b, index)


@pytest.mark.parametrize("M", [70, 900])  # rows one by one, and by lists
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_autograd_layouts(M, dtype):
    """Strided inputs, a broadcast gradient and a graph that is kept: the dense tensors' bits, twice."""
    c = case(M, 1200, 1300, 8, 3, dtype, seed=21)
    c["x"] = c["x"].reshape(2, M // 2, 1200)
    c["base"] = c["base"].reshape(2, M // 2, 1300)
    c["index"] = c["index"].reshape(2, M // 2)
    x, a, b, index, scales, base = to(c, "x", "a", "b", "index", "scales", "base")

    def run(x, a, b, base, index, w):
        x, a, b, base = (t.detach().requires_grad_() for t in (x, a, b, base))
        y = adapt(x, a, b, index, scales, base, 0.25, 5, 2)
        first = torch.autograd.grad(y, (x, a, b, base), w, retain_graph=True)
        again = torch.autograd.grad(y, (x, a, b, base), w)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
        return (y.detach(), *first)
    w = torch.randn(1300, generator=torch.Generator().manual_seed(2)).to(x.dtype).to(DEV).expand(2, M // 2, 1300)
    want = run(x, a, b, base, index, w.contiguous())
    flip = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, base, index)]
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (a, b)]
    got = run(flip[0], *turned, flip[1], flip[2], w)
    for p, q in zip(want, got):
        assert torch.equal(p, q)
    assert torch.equal(got[4], w)


@pytest.mark.parametrize("dtype,K,N,p", [("bf16", 4096, 4104, 0.0), ("fp32", 4104, 4160, 0.25), ("fp16", 4099, 4104, 0.0)])
def test_large_banks(dtype, K, N, p):
    """32 rows of one adapter and a narrow product in parts, both ways; 16 rows where they lie on odd half words."""
    c = case(4200, K, N, 32, 2, dtype, seed=22, lead=(2, 2100))
    c["index"] = torch.tensor([1, 0])
    backward_case(c, p, seed=3)


@pytest.mark.parametrize("M,K,N,r", [(40, 300, 200, 32), (130, 96, 1000, 64), (208, 1471, 650, 64), (70, 64, 600, 128)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ranks_choose_rows(M, K, N, r, dtype):
    """A sequence's rows, more of them to a workgroup for larger ranks."""
    c = case(M, K, N, r, 3, dtype, seed=23, lead=(2, M // 2))
    c["index"] = torch.tensor([2, -1])
    backward_case(c, 0.25, seed=4)
