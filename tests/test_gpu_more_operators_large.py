"""Tensors of more than 2^31 elements, and offsets past them, through the adapters, dropout and verification:
rows at the far end against the same rows in a tensor of their own (the same bits: a row's sums do not depend on
where it lies)."""

import pytest
import torch

from ksdraft_amd.kernels.adapters import adapter_linear, adapter_linear_backward, adapter_linear_train
from ksdraft_amd.kernels.dropout import dropout
from ksdraft_amd.kernels.speculate import verify_draft
from tests.philox import mask

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_adapters():
    M, K, N, r, n = 33000, 64, 65600, 16, 2  # 2.16e9 outputs
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(M, K, device=DEV, generator=g).bfloat16()
    a = torch.randn(n, r, K, device=DEV, generator=g).bfloat16()
    b = torch.randn(n, N, r, device=DEV, generator=g).bfloat16()
    index = torch.zeros(M, dtype=torch.int64, device=DEV)
    index[-100:] = 1
    y, saved = adapter_linear_train(x, a, b, index)
    far = slice(M - 40, M)
    want = (x[far].double() @ a[1].double().t()) @ b[1].double().t()
    size = (x[far].double().abs() @ a[1].double().abs().t()) @ b[1].double().abs().t()
    bound = size * (2 * (K + r + 4) * 2.0 ** -24 + 2.0 ** -16)
    assert bool(((y[far].double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())
    assert torch.equal(adapter_linear(x[far], a, b, index[far]), y[far])
    # the gradient's columns: dB of the last columns from the last rows alone
    dy = torch.zeros_like(y)
    dy[-1, -1] = 2.0
    dx, da, db = adapter_linear_backward(dy, saved)
    h = x[-1].double() @ a[1].double().t()
    assert bool(((db[1, -1].double() - 2 * h).abs() <= 1e-5 * (x[-1].double().abs() @ a[1].double().abs().t())).all())
    assert not bool(db[0].any()) and not bool(db[1, :-1].any()) and not bool(dx[:-1].any()) and bool(dx[-1].any())
    assert not bool(da[0].any())


def test_dropout():
    rows, d = 70000, 31000  # 2.17e9
    x = torch.ones(rows, d, dtype=torch.float16, device=DEV)
    y = dropout(x, 0.25, 9, 1, residual=x)
    keep = mask(rows, 8, 0.25, 9, 1)[-3:]
    assert torch.equal(y[-3:, :8].float().cpu(), (keep + 1).half().float())
    part = dropout(torch.zeros(2, d, dtype=torch.float16, device=DEV), 0.25, 9, 1)
    assert part.shape == (2, d) and bool((y[-1] >= 1).all())


def test_verification():
    V = 3000
    g = torch.Generator(device=DEV).manual_seed(0)
    buffer = torch.zeros(2 ** 31 + 4 * V, dtype=torch.bfloat16, device=DEV)
    target = buffer.as_strided((2, 3, V), (2 ** 31, V, 1))
    rows = torch.randn(2, 3, V, device=DEV, generator=g).mul(2).bfloat16()
    target.copy_(rows)
    draft = (rows[:, :2].float() + 0.2 * torch.randn(2, 2, V, device=DEV, generator=g)).bfloat16()
    tokens = draft.float().argmax(2)
    u = torch.rand(2, 3, device=DEV, generator=g)
    got, want = verify_draft(target, tokens, u, draft), verify_draft(rows, tokens, u, draft)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
