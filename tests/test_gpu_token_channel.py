"""W8A8 with scales per token and channel against 64-bit arithmetic on the same codes.

Codes and scales are defined by single fp32 operations, so they are compared bit for bit with the
same operations on the CPU. A product's value passes at most five fp32 roundings (the int32 sum,
two scales, bias, residual), each at most 2^-24 of the largest magnitude that it meets, and one
rounding to the output type (2^-24, 2^-11 or 2^-8 relative for fp32, fp16 and bf16; 2^-25 absolute
for fp16's subnormals)."""

import ctypes
import math

import pytest
import torch

from ksdraft_amd import _lib
from ksdraft_amd.kernels import token_channel as tc

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rows_cpu(x):
    """The row quantization's definition, in fp32 on the CPU."""
    x = x.float().cpu()
    a = x.abs().amax(1)
    bad = ~torch.isfinite(a)
    live = (a >= 2.0 ** -100) & ~bad
    safe = torch.where(live, a, torch.ones(()))
    top = torch.full_like(safe, 127.0)  # a tensor: torch's 127 / t is a reciprocal and a product
    scale = torch.where(live, safe / top, torch.zeros(()))
    inv = torch.where(live, top / safe, torch.zeros(()))
    codes = torch.where(live[:, None], torch.round(x * inv[:, None]), torch.zeros(()))
    return codes.to(torch.int8), torch.where(bad, torch.full((), math.nan), scale)


def close(y, ref, size, dtype, n_ops=5):
    """|y - ref| within n_ops fp32 roundings of `size` and one to dtype."""
    y, ref, size = y.double().cpu(), ref.double().cpu(), size.double().cpu()
    bound = n_ops * 2.0 ** -24 * size
    bound = bound + EPS[dtype] * (ref.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 1e-45)
    off = (y - ref).abs() > bound
    assert not bool(off.any()), f"{int(off.sum())} of {y.numel()} off, worst {float(((y - ref).abs() / bound).max()):.2f} bounds"


def data(M, K, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * scale
    return x.to(TYPES[dtype]).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 16), (4, 129), (7, 512), (2, 513), (9, 597), (6, 1536), (3, 1537),
                                 (2, 8192), (2, 8200), (3, 20011), (257, 64)])
def test_quantize_rows(M, K, dtype):
    x = data(M, K, dtype, M * 1000 + K)
    if M > 2:
        x[1] = 0
        x[2, K // 2] = 8
    q, s = tc.quantize_rows(x)
    eq, es = rows_cpu(x)
    assert torch.equal(s.cpu(), es)
    assert torch.equal(q.cpu(), eq)
    pad = torch.as_strided(q, (M, -(-K // 16) * 16), (q.stride(0) if M > 1 else -(-K // 16) * 16, 1))
    assert not bool(pad[:, K:].any())


@pytest.mark.gpu
def test_quantize_rows_edges():
    """Ties, rows of tiny, infinite and NaN values, strided and unaligned rows."""
    x = torch.zeros(8, 40)
    x[0] = torch.linspace(-127, 127, 40)
    x[0, 0] = 127.0
    x[0, 1:5] = torch.tensor([0.5, 1.5, -2.5, 3.5])  # scale 1: ties go to the even code
    x[1] = 2.0 ** -101
    x[2] = 2.0 ** -100
    x[3] = 1.0
    x[3, 5] = math.inf
    x[4] = 1.0
    x[4, 39] = math.nan
    x[5] = torch.finfo(torch.float32).max
    x[6] = -3.0e-30
    q, s = tc.quantize_rows(x.to(DEV))
    eq, es = rows_cpu(x)
    assert torch.equal(q.cpu(), eq) and torch.equal(s.cpu().isnan(), es.isnan())
    assert torch.equal(s.cpu().nan_to_num(7.0), es.nan_to_num(7.0))
    assert q[0, 1:5].tolist() == [0, 2, -2, 4] and s[0].item() == 1.0
    assert q[3].abs().sum().item() == 0 and math.isnan(s[3].item()) and math.isnan(s[4].item())
    base = data(6, 300, "bf16", 3)
    for view in (base[:, 1:290], base[1::2, 3:], base.t()[5:]):
        q, s = tc.quantize_rows(view)
        eq, es = rows_cpu(view)
        assert torch.equal(q.cpu(), eq) and torch.equal(s.cpu(), es)


SHAPES = [(1, 1, 1), (1, 512, 1536), (3, 5, 7), (4, 1000, 129), (16, 64, 1536), (17, 33, 2048), (64, 130, 597),
          (2, 40, 20011), (32, 50, 2500), (33, 48, 1537), (31, 2000, 100), (129, 127, 16), (130, 257, 1000), (300, 1536, 512), (515, 384, 4099), (1021, 777, 333)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_linear(M, N, K, dtype):
    x = data(M, K, dtype, 1)
    wq, ws = tc.quantize_rows(data(N, K, "fp32", 2, K ** -0.5))
    bias = data(1, N, "fp32", 3)[0] if (M + N) % 2 else None
    res = data(M, N, dtype, 4) if (M + K) % 2 else None
    y = tc.token_channel_linear(x, wq, ws, bias, res)
    assert y.dtype == TYPES[dtype] and y.shape == (M, N)
    xq, xs = rows_cpu(x)
    main = (xq.double() @ wq.cpu().double().t()) * xs.double()[:, None] * ws.cpu().double()
    ref, size = main.clone(), main.abs()
    for extra in (bias, res):
        if extra is not None:
            ref = ref + extra.cpu().double()
            size = size + extra.cpu().double().abs()
    close(y, ref, size, TYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 17, 133200), (130, 40, 300000), (20, 300, 200016)])
def test_long_sums(M, N, K):
    """Codes of one sign and full size over reductions whose sum passes 32 bits."""
    a = torch.full((M, K), 127, dtype=torch.int8, device=DEV)
    w = torch.full((N, K), 127, dtype=torch.int8, device=DEV)
    a[0, ::3] = -5
    sa, sw = torch.full((M,), 0.5, device=DEV), torch.full((N,), 2.0, device=DEV)
    y = tc.token_channel_gemm(a, sa, w, sw)
    ref = (a.double() @ w.double().t()).cpu()
    close(y, ref, ref.abs(), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES + [(2047, 300, 257), (5, 3000, 64)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_training(M, N, K, dtype):
    """y, dX, dW and db against the formulas on the codes."""
    dt = TYPES[dtype]
    x, w, g = data(M, K, dtype, 5), data(N, K, "fp32", 6, K ** -0.5), data(M, N, dtype, 7)
    if M > 3:
        x[2] = 0   # a token of zeros: scale 0
        g[1] = 0   # a token without gradient
    if N > 3:
        w[2] = 0
        g[:, 1] = 0
    bias = data(1, N, "fp32", 8)[0]
    y, saved = tc.token_channel_linear_train(x, w, bias)
    dx, dw, db = tc.token_channel_linear_backward(g, saved)
    xq, xs = rows_cpu(x)
    wq, ws = rows_cpu(w)
    main = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    close(y, main + bias.cpu().double(), main.abs() + bias.cpu().double().abs(), dt)
    gf = g.float().cpu()
    q, e = rows_cpu(gf * ws)
    main = (q.double() @ wq.double()) * e.double()[:, None]
    close(dx, main, main.abs(), dt)
    c, f = rows_cpu((gf * xs[:, None]).t())
    main = (c.double() @ xq.double()) * f.double()[:, None]
    close(dw, main, main.abs(), torch.float32)
    close(db, gf.double().sum(0), gf.double().abs().sum(0), torch.float32, n_ops=M)
    assert dx.dtype == dt and dw.dtype == db.dtype == torch.float32


# (M, N, K) and the tile (rows, columns, workgroups per CU) that one of its products gets: 0 the forward
# (M, N, K), 1 dX (M, K, N), 2 dW (N, K, M)
TILED = [(2617, 4477, 134, 0, (256, 256, 1)), (2574, 128, 4458, 1, (256, 256, 1)), (133, 4909, 2587, 2, (256, 256, 1)),
         (4625, 1686, 131, 0, (256, 192, 1)), (2342, 128, 3512, 1, (256, 192, 1)), (128, 1808, 4725, 2, (256, 192, 1)),
         (4685, 801, 129, 0, (128, 128, 2)), (961, 130, 4143, 1, (128, 128, 2)), (132, 3694, 1048, 2, (128, 128, 2)),
         (4133, 479, 4157, 0, (128, 128, 1)), (523, 4305, 3639, 1, (128, 128, 1)), (4330, 4726, 394, 2, (128, 128, 1)),
         (389, 4785, 137, 0, (64, 128, 2)), (840, 131, 2315, 1, (64, 128, 2)), (131, 4862, 387, 2, (64, 128, 2)),
         (135, 5902, 5951, 0, (64, 128, 2)), (135, 128, 2952, 0, (64, 64, 2)), (141, 2855, 134, 1, (64, 64, 2)),
         (2878, 131, 156, 2, (64, 64, 2)), (4600, 4700, 140, 0, (256, 192, 1)), (5003, 5009, 140, 0, (256, 256, 1))]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,which,tile", TILED)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_products_of_every_tile(M, N, K, which, tile, dtype):
    """All three products at shapes that take each tile form, ragged at every edge, four of them with the
    reduction in parts, the last two with several tiles to a workgroup: on the codes as they are, exact up to
    the output's rounding."""
    v = [ctypes.c_int() for _ in range(4)]
    _lib.call("ksd_tc_gemm_form", *((M, N, K), (M, K, N), (N, K, M))[which], *[ctypes.byref(x) for x in v])
    assert tuple(x.value for x in v[:3]) == tile
    g = torch.Generator().manual_seed(M)
    a = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8).to(DEV)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8).to(DEV)
    sa, sw = torch.rand(M, generator=g).to(DEV) + 0.5, torch.rand(N, generator=g).to(DEV) + 0.5
    bias, res = data(1, N, "fp32", 3)[0], data(M, N, dtype, 4)
    y = tc.token_channel_gemm(a, sa, w, sw, bias, res, TYPES[dtype])
    main = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()
    size = main.abs() + bias.double().abs() + res.double().abs()
    close(y, main + bias.double() + res.double(), size, TYPES[dtype])
    x, wt, up = data(M, K, dtype, 5), data(N, K, "fp32", 6), data(M, N, dtype, 7)
    _, s = tc.token_channel_linear_train(x, wt)
    dx, dw, _ = tc.token_channel_linear_backward(up, s)
    xq, wq, xs, ws = s.xq[:, :K].double(), s.wq[:, :K].double(), s.xs, s.ws
    q, e = rows_cpu(up.float().cpu() * ws.cpu())
    main = (q.to(DEV).double() @ wq) * e.to(DEV).double()[:, None]
    close(dx, main, main.abs(), TYPES[dtype])
    c, f = rows_cpu((up.float().cpu() * xs.cpu()[:, None]).t())
    main = (c.to(DEV).double() @ xq) * f.to(DEV).double()[:, None]
    close(dw, main, main.abs(), torch.float32)


@pytest.mark.gpu
def test_training_nonfinite():
    """A NaN or inf stays in the rows that it reaches: y's and dX's token, dW's channel."""
    M, N, K = 70, 90, 200
    x, w, g = data(M, K, "fp32", 1), data(N, K, "fp32", 2), data(M, N, "fp32", 3)
    g[5, 7] = math.nan
    g[9, 11] = math.inf
    y, saved = tc.token_channel_linear_train(x, w)
    dx, dw, _ = tc.token_channel_linear_backward(g, saved)
    rows, cols = torch.zeros(M, dtype=torch.bool), torch.zeros(N, dtype=torch.bool)
    rows[[5, 9]] = True
    cols[[7, 11]] = True
    assert torch.equal(dx.isnan().cpu(), rows[:, None].expand(M, K))
    assert torch.equal(dw.isnan().cpu(), cols[:, None].expand(N, K))
    x[3, 1] = math.nan
    y, _ = tc.token_channel_linear_train(x, w)
    rows.zero_()
    rows[3] = True
    assert torch.equal(y.isnan().cpu(), rows[:, None].expand(M, N))


@pytest.mark.gpu
def test_gradient_by_differences():
    """On values that the codes hold exactly (integers with a row maximum of 127), the layer is the
    plain linear map, whose differences are exact in fp64."""
    g = torch.Generator().manual_seed(0)

    def ints(r, c):
        t = torch.randint(-126, 127, (r, c), generator=g).float()
        t[torch.arange(r), torch.arange(r) % c] = 127.0
        return t
    M, N, K = 12, 10, 14
    x, w = ints(M, K), ints(N, K)
    up = torch.zeros(M, N)
    up[torch.arange(M), torch.arange(M) % N] = 1.0  # one channel per token: its codes are exact too
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV)
    lin = tc.TokenChannelLinear(K, N, bias=True).to(DEV)
    with torch.no_grad():
        lin.weight.copy_(wd)
    (lin(xd) * up.to(DEV)).sum().backward()

    def loss(xv, wv, bv):
        return float(((xv.double() @ wv.double().t() + bv) * up.double()).sum())
    zero = torch.zeros(N, dtype=torch.float64)
    for i, k in [(0, 0), (3, 5), (11, 13)]:
        d = torch.zeros_like(x)
        d[i, k] = 1.0
        num = (loss(x + d, w, zero) - loss(x - d, w, zero)) / 2
        assert abs(xd.grad[i, k].item() - num) <= 4 * 2.0 ** -24 * abs(num)
    for n, k in [(0, 0), (9, 3), (4, 13)]:
        d = torch.zeros_like(w)
        d[n, k] = 1.0
        num = (loss(x, w + d, zero) - loss(x, w - d, zero)) / 2
        # dW's codes round dY (0 or 1 here, several tokens of one channel): all are 127 or 0
        assert abs(lin.weight.grad[n, k].item() - num) <= 4 * 2.0 ** -24 * 127 * M
    assert torch.equal(lin.bias.grad.cpu(), up.sum(0))


@pytest.mark.gpu
def test_module_and_strides():
    lin = torch.nn.Linear(200, 77).to(DEV)
    mod = tc.TokenChannelLinear.from_float(lin)
    x = data(30, 400, "bf16", 1)[:, ::2].reshape(5, 6, 200)
    with torch.no_grad():
        y = mod(x)
        assert torch.equal(y, mod.pack()(x)) and y.shape == (5, 6, 77)
        assert mod.unpack()._packed is None
        ref = torch.nn.functional.linear(x.float(), lin.weight, lin.bias)
        assert ((y.float() - ref).norm() / ref.norm()).item() < 0.03
        # codes in a buffer of another pitch, and a residual
        q, s = tc.quantize_rows(lin.weight)
        tight = q.contiguous()
        r = data(30, 77, "bf16", 2).reshape(5, 6, 77)
        a = tc.token_channel_linear(x, q, s, lin.bias, r)
        assert torch.equal(a, tc.token_channel_linear(x, tight, s, lin.bias, r))
    xg = x.clone().requires_grad_(True)
    rg = r.clone().requires_grad_(True)
    out = mod(xg, residual=rg)
    g = torch.ones_like(out)
    out.backward(g)
    assert torch.equal(rg.grad, g) and xg.grad.shape == x.shape and mod.weight.grad.shape == (77, 200)
    assert mod._packed is None
    # an expanded upstream gradient (the backward of a sum) has zero strides
    mod.zero_grad()
    xg.grad = None
    first = None
    out = mod(xg)
    out.backward(torch.ones((), device=DEV, dtype=out.dtype).expand(out.shape))
    first = mod.weight.grad.clone()
    mod.zero_grad()
    mod(xg).backward(torch.ones_like(out))
    assert torch.equal(first, mod.weight.grad)


@pytest.mark.gpu
def test_module_dtypes():
    """Half precision masters, and a residual of another dtype."""
    mod = tc.TokenChannelLinear.from_float(torch.nn.Linear(96, 50).to(DEV)).to(torch.bfloat16)
    x = data(20, 96, "bf16", 1).requires_grad_(True)
    r = data(20, 50, "fp32", 2)
    with torch.no_grad():
        plain = mod(x)
        assert torch.equal(mod(x, residual=r), r + plain)
    mod(x).backward(torch.ones(20, 50, device=DEV, dtype=torch.bfloat16))
    assert mod.weight.grad.dtype == mod.bias.grad.dtype == torch.bfloat16 and x.grad.dtype == torch.bfloat16
    assert torch.equal(mod.bias.grad, torch.full((50,), 20.0, device=DEV, dtype=torch.bfloat16))


@pytest.mark.gpu
def test_graph():
    """A captured step (products, both gradients, embedding gradient, clipping), replayed between eager
    work: every replay gives the eager bits."""
    from ksdraft_amd.kernels.embedding import embedding_gradient, embedding_lookup
    from ksdraft_amd.train.clip import clip_gradients
    table, w = data(900, 256, "fp32", 1), data(384, 256, "fp32", 2)
    ids = torch.randint(0, 900, (3000,), generator=torch.Generator().manual_seed(3)).to(DEV)
    up = data(3000, 384, "fp32", 4)

    def step():
        x = embedding_lookup(table, ids, 16.0, check_ids=False)
        y, s = tc.token_channel_linear_train(x, w)
        few = tc.token_channel_linear(x[:4], s.wq[:, :256], s.ws)
        dx, dw, db = tc.token_channel_linear_backward(up, s, need_db=True)
        dt = embedding_gradient(dx, ids, 900, 16.0, check_ids=False)
        out = [torch.empty_like(dw), torch.empty_like(dt)]
        return [y, few, dx, dw, db, dt, clip_gradients([dw, dt], 1.0, out=out), *out]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        eager = [t.clone() for t in step()]
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))
        step()
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_operands_with_unknown_padding():
    """Bytes between a caller's rows take no part."""
    buf = torch.full((20, 48), 77, dtype=torch.int8, device=DEV)
    wbuf = torch.full((30, 64), 55, dtype=torch.int8, device=DEV)
    a, w = buf[:, :37], wbuf[:, :37]
    a.copy_(torch.randint(-127, 128, (20, 37), generator=torch.Generator().manual_seed(0)))
    w.copy_(torch.randint(-127, 128, (30, 37), generator=torch.Generator().manual_seed(1)))
    one_a, one_w = torch.ones(20, device=DEV), torch.ones(30, device=DEV)
    for m in (1, 20):
        y = tc.token_channel_gemm(a[:m], one_a[:m], w, one_w)
        assert torch.equal(y.cpu().double(), a[:m].cpu().double() @ w.cpu().double().t())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(16, 33, 2048), (17, 33, 2048), (13, 20000, 129), (12, 40, 2730), (8, 50, 4096), (8, 50, 4097),
                                   (5, 17, 3001), (4, 21, 8192), (4, 21, 8193), (1, 16500, 70)])
def test_few_tokens(M, N, K):
    """Either side of the one-launch form: the same bits as the quantizer and the product apart."""
    x = data(M, K, "bf16", 1)
    wq, ws = tc.quantize_rows(data(N, K, "fp32", 2, K ** -0.5))
    bias, res = data(1, N, "fp32", 3)[0], data(M, N, "bf16", 4)
    q, s = tc.quantize_rows(x)
    y = tc.token_channel_linear(x, wq, ws, bias, res)
    assert torch.equal(y, tc.token_channel_gemm(q, s, wq, ws, bias, res, out_dtype=torch.bfloat16))
    sums = (q.cpu().double() @ wq.cpu().double().t()).float()
    exact = ((sums * s.cpu()[:, None] * ws.cpu()) + bias.cpu() + res.float().cpu()).bfloat16()
    assert torch.equal(y.cpu(), exact)


@pytest.mark.gpu
def test_empty_and_repeat():
    wq, ws = tc.quantize_rows(data(40, 64, "fp32", 1))
    x = torch.empty(0, 64, device=DEV)
    assert tc.token_channel_linear(x, wq, ws).shape == (0, 40)
    y, s = tc.token_channel_linear_train(x, data(40, 64, "fp32", 1))
    dx, dw, db = tc.token_channel_linear_backward(torch.empty(0, 40, device=DEV), s, need_db=True)
    assert dx.shape == (0, 64) and not bool(dw.any()) and not bool(db.any())
    x, w, g = data(333, 500, "fp32", 2), data(200, 500, "fp32", 3), data(333, 200, "fp32", 4)
    outs = []
    for _ in range(2):
        y, s = tc.token_channel_linear_train(x, w)
        outs.append([y, *tc.token_channel_linear_backward(g, s, need_db=True)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    dx, dw, db = tc.token_channel_linear_backward(g, s, need_dx=False)
    assert dx is None and db is None and torch.equal(dw, outs[0][2])
    dx, dw, db = tc.token_channel_linear_backward(g, s, need_dw=False)
    assert dw is None and torch.equal(dx, outs[0][1])


@pytest.mark.gpu
def test_other_stream():
    x, w = data(300, 256, "bf16", 1), data(256, 256, "fp32", 2)
    wq, ws = tc.quantize_rows(w)
    y = tc.token_channel_linear(x, wq, ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        z = tc.token_channel_linear(x, wq, ws)
    side.synchronize()
    assert torch.equal(y, z)


@pytest.mark.gpu
def test_refusals():
    x = data(4, 64, "fp32")
    wq, ws = tc.quantize_rows(data(8, 64, "fp32"))
    with pytest.raises(ValueError):
        tc.token_channel_linear(x[:, :63], wq, ws)
    with pytest.raises(ValueError):
        tc.token_channel_linear(x, wq, ws[:7])
    with pytest.raises(ValueError):
        tc.token_channel_linear(x, wq, ws, bias=torch.zeros(8, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        tc.token_channel_linear(x, wq.float(), ws)
    with pytest.raises(TypeError):
        tc.token_channel_linear(x.double(), wq, ws)
    with pytest.raises(TypeError):
        tc.token_channel_linear(x, wq, ws, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        tc.token_channel_linear(x, wq, ws, residual=torch.zeros(4, 8, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        tc.token_channel_gemm(wq[:4], ws[:4], wq[:, :32], ws)
    with pytest.raises(ValueError):
        tc.quantize_rows(torch.zeros(3, 0, device=DEV))
    with pytest.raises(RuntimeError):
        tc.token_channel_linear(x.cpu(), wq, ws)
    _, s = tc.token_channel_linear_train(x, data(8, 64, "fp32"))
    with pytest.raises(ValueError):
        tc.token_channel_linear_backward(torch.zeros(4, 9, device=DEV), s)
