"""The scaled lookup and the gradient by sorted tokens against 64-bit sums.

A lookup is one fp32 product and one rounding. A gradient entry is a sum of c terms in fp32 (at
most c roundings of the running sum, bounded by the sum of magnitudes), one product with the scale
and one rounding to the output type."""

import math

import pytest
import torch

from ksdraft_amd.kernels.embedding import ScaledEmbedding, embedding_gradient, embedding_lookup

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def randn(*shape, dtype="fp32", seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(TYPES[dtype]).to(DEV)


def ids_of(n, V, seed=0, how="zipf"):
    g = torch.Generator().manual_seed(seed)
    if how == "uniform":
        return torch.randint(0, V, (n,), generator=g).to(DEV)
    if how == "one":
        return torch.full((n,), V - 1, dtype=torch.int64).to(DEV)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    return ((V + 1) ** u).long().sub(1).clamp(0, V - 1).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("out", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (5, 9, 7), (33, 100, 129), (64, 1000, 1536), (3, 50, 2051)])
def test_lookup(n, V, d, dtype, out):
    w, ids = randn(V, d, dtype=dtype), ids_of(n, V, 1)
    y = embedding_lookup(w, ids, 0.3, out_dtype=TYPES[out])
    ref = (w.float().cpu()[ids.cpu()] * torch.tensor(0.3)).to(TYPES[out])
    assert torch.equal(y.cpu(), ref)
    assert torch.equal(embedding_lookup(w, ids.int().reshape(1, n), 0.3, out_dtype=TYPES[out])[0].cpu(), ref)


@pytest.mark.gpu
def test_lookup_edges():
    w = randn(10, 24)
    strided = randn(10, 50)[:, 3:27]
    ids = torch.tensor([[0, 9], [3, 3]], device=DEV)
    assert torch.equal(embedding_lookup(strided, ids), strided[ids])
    assert torch.equal(embedding_lookup(w.t().contiguous().t(), ids), w[ids])
    bad = torch.tensor([-1, 10, 2, 1 << 40], device=DEV)
    y = embedding_lookup(w, bad, 2.0, check_ids=False)
    assert not bool(y[[0, 1, 3]].any()) and torch.equal(y[2], w[2] * 2)
    with pytest.raises(IndexError):
        embedding_lookup(w, bad)
    assert embedding_lookup(w, bad[:0]).shape == (0, 24)
    w[4, 5] = math.inf
    assert math.isinf(embedding_lookup(w, torch.tensor([4], device=DEV))[0, 5].item())


def check_gradient(got, g, ids, V, scale, pad, dtype, was=None):
    gd, idc = g.double().cpu().reshape(-1, g.shape[-1]), ids.cpu().reshape(-1).long()
    keep = (idc >= 0) & (idc < V)
    if pad is not None:
        keep &= idc != pad % V
    d = gd.shape[1]
    ref = torch.zeros(V, d, dtype=torch.float64).index_add_(0, idc[keep], gd[keep])
    size = torch.zeros(V, d, dtype=torch.float64).index_add_(0, idc[keep], gd[keep].abs())
    count = torch.zeros(V, dtype=torch.float64).index_add_(0, idc[keep], torch.ones(int(keep.sum()), dtype=torch.float64))
    bound = (count[:, None] + 2) * 2.0 ** -24 * size * abs(scale)
    ref = ref * scale
    if was is not None:
        ref = ref + was.double().cpu()
        bound = bound + 2.0 ** -24 * ref.abs()
    bound = bound + EPS[dtype] * (ref.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 1e-45)
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.2f} bounds"
    untouched = count == 0
    assert torch.equal(got.cpu()[untouched], (torch.zeros_like(got) if was is None else was).cpu()[untouched])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,V,d,how,pad", [(1, 1, 1, "one", None), (1, 5, 8, "one", 4), (7, 3, 5, "zipf", 0), (32, 300, 64, "uniform", None),
                                           (33, 2, 129, "one", None), (1024, 40, 130, "zipf", None), (2048, 5, 33, "zipf", None), (2049, 3000, 20, "zipf", 1), (900, 1 << 20, 4, "uniform", None), (5000, 1 << 20, 4, "zipf", None), (5000, 600000, 3, "uniform", 7), (8192, 20000, 1030, "zipf", None), (500, 255, 1001, "zipf", None), (2048, 256, 24, "zipf", 255),
                                           (2049, 257, 40, "one", 0), (3000, 70000, 36, "zipf", None),
                                           (8192, 150144, 8, "uniform", -1), (8193, 65536, 33, "zipf", 0), (20000, 11, 2056, "zipf", None),
                                           (100003, 40000, 16, "zipf", 0), (140001, 700, 12, "zipf", None)])
def test_gradient(n, V, d, how, pad, dtype):
    g, ids = randn(n, d, dtype=dtype, seed=2), ids_of(n, V, 3, how)
    got = embedding_gradient(g, ids, V, 1.5, padding_idx=pad)
    check_gradient(got, g, ids, V, 1.5, pad, torch.float32)
    assert torch.equal(got, embedding_gradient(g, ids.int(), V, 1.5, padding_idx=pad))


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,d,how", [(1, 600, 70, "one"), (512, 300, 33, "zipf"), (513, 300, 33, "zipf"), (512, 9000, 132, "one"),
                                       (40, 131101, 513, "zipf"), (511, 70001, 1025, "uniform"), (514, 524287, 3, "one"), (1025, 524287, 2, "uniform"),
                                       (2047, 800, 60, "zipf"), (2048, 40000, 19, "uniform"), (1999, 3, 258, "zipf"), (12000, 48000, 20, "zipf"),
                                       (12000, 47999, 20, "zipf"), (9000, 600000, 9, "uniform"), (16385, 70000, 5, "one"),
                                       (262144, 900, 6, "zipf"), (262145, 3, 70, "zipf"), (270001, 1, 258, "one")])
def test_gradient_written_once(n, V, d, how):
    """Tables of 256 MB and more, few and many tokens, one run through all: nothing of what `out` held stays."""
    g, ids = randn(n, d, seed=7), ids_of(n, V, 8, how)
    got = torch.full((V, d), math.nan, device=DEV)
    embedding_gradient(g, ids, V, 0.5, padding_idx=0 if V > 1 else None, out=got)
    if V * d < 1 << 24:
        check_gradient(got, g, ids, V, 0.5, 0 if V > 1 else None, torch.float32)
    else:
        rows = ids.unique()
        rows = rows[rows != 0]
        check_gradient(got[rows], g, torch.searchsorted(rows, ids) + (ids == 0) * len(rows), len(rows), 0.5, None, torch.float32)
        got[rows] = 0
        assert not bool(got.any())
    if V * d < 1 << 24:
        was = randn(V, d, seed=9)
        more = was.clone()
        embedding_gradient(g, ids, V, 0.5, padding_idx=0 if V > 1 else None, out=more, accumulate=True)
        check_gradient(more, g, ids, V, 0.5, 0 if V > 1 else None, torch.float32, was)


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["fp32", "bf16", "fp16"])
def test_gradient_accumulates(out):
    n, V, d = 700, 900, 52
    g, ids = randn(n, d, seed=4), ids_of(n, V, 5)
    was = randn(V, d, dtype=out, seed=6)
    got = was.clone()
    embedding_gradient(g, ids, V, 0.25, out=got, accumulate=True)
    check_gradient(got, g, ids, V, 0.25, None, TYPES[out], was)
    fresh = torch.full((V, d), math.nan, device=DEV, dtype=TYPES[out])
    embedding_gradient(g, ids, V, 0.25, out=fresh)
    check_gradient(fresh, g, ids, V, 0.25, None, TYPES[out])


@pytest.mark.gpu
def test_gradient_edges():
    g, ids = randn(40, 60)[:, 7:31], ids_of(40, 20)
    check_gradient(embedding_gradient(g, ids, 20), g, ids, 20, 1.0, None, torch.float32)
    bad = ids.clone()
    bad[3], bad[5] = -2, 20
    check_gradient(embedding_gradient(g, bad, 20, check_ids=False), g, bad, 20, 1.0, None, torch.float32)
    with pytest.raises(IndexError):
        embedding_gradient(g, bad, 20)
    assert not bool(embedding_gradient(g[:0], ids[:0], 20).any())
    only = torch.full((40,), 3, device=DEV)
    assert not bool(embedding_gradient(g, only, 20, padding_idx=3).any())
    # NaN and inf stay in their token's row and column
    h = g.clone()
    h[4, 2] = math.nan
    got = embedding_gradient(h, ids, 20)
    assert bool(got[ids[4], 2].isnan()) and int(got.isnan().sum()) == 1


@pytest.mark.gpu
def test_module_gradients():
    """Against differences of a loss that is linear in the table (exact in fp64)."""
    V, d = 50, 24
    emb = torch.nn.Embedding(V, d, padding_idx=2).to(DEV)
    mod = ScaledEmbedding.from_float(emb, scale=math.sqrt(d))
    assert mod.weight is emb.weight
    ids = torch.tensor([[1, 2, 3], [3, 3, 49]], device=DEV)
    up = randn(2, 3, d, seed=8)
    (mod(ids) * up).sum().backward()
    w = emb.weight.detach().double().cpu()

    def loss(t):
        return float((t[ids.cpu()] * math.sqrt(d) * up.double().cpu()).sum())
    for v, c in [(1, 0), (3, 5), (49, 23), (7, 7)]:
        e = torch.zeros_like(w)
        e[v, c] = 1.0
        num = (loss(w + e) - loss(w - e)) / 2
        assert abs(mod.weight.grad[v, c].item() - num) <= 8 * 2.0 ** -24 * math.sqrt(d) * up.abs().sum().item()
    assert not bool(mod.weight.grad[2].any())  # the padding token


@pytest.mark.gpu
def test_refusals():
    w, ids, g = randn(5, 8), torch.tensor([1, 2], device=DEV), randn(2, 8)
    with pytest.raises(TypeError):
        embedding_lookup(w, ids.float())
    with pytest.raises(TypeError):
        embedding_lookup(w.double(), ids)
    with pytest.raises(ValueError):
        embedding_lookup(w[0], ids)
    with pytest.raises(RuntimeError):
        embedding_lookup(w.cpu(), ids)
    with pytest.raises(ValueError):
        embedding_gradient(g, ids[:1], 5)
    with pytest.raises(ValueError):
        embedding_gradient(g, ids, 5, accumulate=True)
    with pytest.raises(ValueError):
        embedding_gradient(g, ids, 5, padding_idx=5)
    with pytest.raises(ValueError):
        embedding_gradient(g, ids, 5, out=torch.zeros(4, 8, device=DEV))
    with pytest.raises(TypeError):
        embedding_gradient(g, ids, 5, out_dtype=torch.float64)
