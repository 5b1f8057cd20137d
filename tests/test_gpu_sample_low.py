"""Drawing from rows whose largest logit is negative and many temperatures below 0, in one piece of a row and in many: equal to
the definition in 64 bits, as test_gpu_speculate's draws are."""

import pytest
import torch

from ksdraft_amd.kernels.speculate import sample_tokens, verify_draft
from tests.test_gpu_speculate import TYPES, gpu, verify_cpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [3, 100, 2049, 40000, 150144, 260000])  # 1, 1, 2, 20, 74 and 127 pieces
def test_negative_rows(V, dtype):
    g = torch.Generator().manual_seed(V)
    z = torch.randn(7, V, generator=g) * 2
    z[0] -= 1000
    z[1:4] = torch.log_softmax(z[1:4], 1)
    z[4] = torch.finfo(TYPES[dtype]).min
    z[5] = -float("inf")
    z[5, V // 2] = torch.finfo(TYPES[dtype]).min
    z[6] -= 8
    temps = torch.tensor([1.0, 1e-3, 1e-30, 1e-4, 1.0, 1.0, 0.01])
    rows, u = z.to(TYPES[dtype]), torch.rand(7, generator=g)
    want = verify_cpu(rows[:, None], None, u[:, None], None, temps)[0][:, 0]
    assert bool((want >= 0).all())
    got = sample_tokens(gpu(rows), gpu(u), gpu(temps)).cpu()
    assert torch.equal(got, want)
    one = [int(sample_tokens(gpu(rows[i]), gpu(u[i]), float(temps[i]))) for i in range(7)]  # a row alone has more pieces
    assert one == want.tolist()
    none = torch.zeros(7, 0, dtype=torch.int64)
    assert torch.equal(verify_draft(gpu(rows)[:, None], gpu(none), gpu(u)[:, None], temperatures=gpu(temps))[0][:, 0].cpu(), want)
