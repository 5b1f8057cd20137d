"""An adapted int8 model with no adapter selected: the unadapted model's bits by the unadapted model's joint calls."""

import pytest
import torch

from ksdraft_amd.kernels import rosa as R
from ksdraft_amd.model import add_adapters, select_adapters, to_int8
from tests.test_gpu_adapted_model import INDEX, make, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("targets", [("q_proj", "k_proj", "v_proj", "out_proj"), ("v_proj",)])
def test_no_adapter_selected(targets, monkeypatch):
    base = to_int8(make()).eval()
    m = add_adapters(base, 3, 8, targets=targets).eval()
    calls = []
    for name in ("shift_project", "hard_out"):
        monkeypatch.setattr(R, name, lambda *a, f=getattr(R, name), n=name: (calls.append(n), f(*a))[1])
    with torch.no_grad():
        want = base(tokens())[0]
        plain, calls[:] = list(calls), []
        assert torch.equal(m(tokens())[0], want) and calls == plain and "shift_project" in plain
        select_adapters(m, INDEX.cuda())
        m(tokens())
        select_adapters(m, None)
        calls.clear()
        assert torch.equal(m(tokens())[0], want) and calls == plain
