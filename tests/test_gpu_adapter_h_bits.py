"""h and its gradient keep their 24 bits on the way through the second product, in every form of it.

Ranks cancel: with three columns of 1 in x, three ranks hold c1 + c2 + c3, -c1 and -c2, where c1 lies in [1, 1.25), c2 in
[2^-9, 2^-8) and c3 in [2^-16, 2^-15), each of 8 bits; their sums are exact in fp32, and one value of the second bank
for the three ranks leaves c3 of y. Of an h of 16 bits up to 2^-17 = 128 u would be missing (u = 2^-24).

Bound: three parts of h lose u of it (fp16's two 2^-22 = 4 u, and what is subnormal), the 9 products of nonzero parts are
added in 9 roundings, twice that allowed for those inside an instruction: 26 u of the sum of magnitudes; then y's own
rounding: half a step, relative to the value, or 2^-25 where an fp16 result is subnormal (below 2^-14 its steps are 2^-24;
c3 alone, of a row whose c1 and c2 are dropped, is one). A mask of p = 1/2 doubles, which is exact."""

import pytest
import torch

from ksdraft_amd.kernels.adapters import adapter_linear, adapter_linear_backward, adapter_linear_train
from tests.philox import mask

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
LEAST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}

# rows, width of the contraction, width of the result, rank, adapters, masked
CASES = [
    (1, 64, 64, 8, 1, False), (5, 40, 129, 3, 2, False), (64, 96, 256, 16, 64, False), (700, 128, 192, 16, 3, False),
    (700, 127, 193, 16, 3, False), (700, 128, 192, 12, 3, False), (700, 128, 192, 16, 3, True), (700, 127, 193, 16, 3, True),
    (700, 128, 192, 12, 3, True), (300, 64, 192, 24, 2, False), (300, 65, 191, 32, 2, True), (300, 64, 192, 40, 2, True),
    (300, 64, 192, 64, 2, False), (300, 65, 193, 64, 2, False), (300, 64, 192, 100, 2, False), (300, 64, 192, 128, 2, True),
    (300, 63, 192, 128, 2, False), (90, 4224, 192, 16, 2, False), (8200, 64, 128, 16, 1, False), (8200, 64, 128, 32, 1, True),
    (8200, 64, 128, 64, 1, False),
    # an adapter for nearly every row: many values of c1, c2 and c3
    (40, 128, 192, 8, 40, False), (40, 128, 192, 12, 40, True), (40, 127, 191, 16, 40, True), (40, 128, 192, 24, 40, True),
    (40, 128, 192, 32, 40, False), (40, 127, 191, 64, 40, False), (40, 128, 192, 100, 40, False), (40, 128, 192, 128, 40, True),
    (40, 4224, 192, 16, 40, False), (8200, 64, 128, 16, 40, False),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N,r,n,masked", CASES)
def test_bits(M, K, N, r, n, masked, dtype):
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(M + r)

    def eighth(lo, shape=()):  # of 8 bits, in [lo, 1.25 lo)
        return lo * (1 + torch.randint(0, 32, shape, generator=g) / 128)
    cols = torch.randperm(K, generator=g)[:3]
    x = torch.zeros(M, K)
    x[:, cols] = 1.0
    first, second = torch.zeros(n, r, K), torch.zeros(n, N, r)
    for i in range(n):
        ranks = torch.randperm(r, generator=g)[:3]
        c1, c2, c3 = eighth(1.0), eighth(2.0 ** -9) * 1.5, eighth(2.0 ** -16)
        first[i, ranks[0], cols] = torch.stack([c1, c2, c3])
        first[i, ranks[1], cols[0]], first[i, ranks[2], cols[1]] = -c1, -c2
        second[i][:, ranks] = (eighth(1.0, (N,)) * (2 * torch.randint(0, 2, (N,), generator=g) - 1))[:, None].expand(N, 3)
    index = torch.randint(0, n, (M,), generator=g)
    keep = mask(M, K, 0.5, 9, 2).double() if masked else torch.ones(M, K, dtype=torch.float64)

    def product(value, z):
        y = torch.zeros(M, N, dtype=torch.float64)
        for i in range(n):
            at = index == i
            y[at] = (value(z[at]) @ value(first[i].double()).t()) @ value(second[i].double()).t()
        return y
    want, size = product(lambda t: t, x.double() * keep), product(torch.abs, x.double() * keep)
    xs, a, b, at = x.to(DEV, dt), first.to(DEV, dt), second.to(DEV, dt), index.to(DEV)
    p = 0.5 if masked else 0.0
    got = adapter_linear_train(xs, a, b, at, dropout=p, seed=9, stream=2)[0] if masked else adapter_linear(xs, a, b, at)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= 26 * U * size + HALF[dt] * want.abs() + LEAST[dt]).all()), float((err / size.clamp(min=1e-9)).max() / U)
    # the gradient goes the other way round: dY = x, banks turned; the mask lies on its result
    z = torch.zeros(M, N, dtype=dt, device=DEV)
    keep = mask(M, N, 0.5, 9, 2).double() if masked else torch.ones(M, N, dtype=torch.float64)
    want, size = product(lambda t: t, x.double()) * keep, product(torch.abs, x.double()) * keep
    saved = adapter_linear_train(z, b.transpose(1, 2).contiguous(), a.transpose(1, 2).contiguous(), at, dropout=p, seed=9, stream=2)[1]
    got = adapter_linear_backward(xs, saved, need_dab=False)[0]
    err = (got.double().cpu() - want).abs()
    assert bool((err <= 26 * U * size + HALF[dt] * want.abs() + LEAST[dt]).all()), float((err / size.clamp(min=1e-9)).max() / U)
