"""Adapted models converted to another type: the adapters stay in fp32, with their bits (CPU)."""

import pytest
import torch

from ksdraft_amd.model.adapters import AdaptedLinear, AdapterSelection


@pytest.mark.parametrize("convert", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16),
                                     lambda m: torch.nn.Sequential(m).bfloat16()[0], lambda m: m.to("cpu", torch.float16)])
def test_adapters_stay_in_fp32(convert):
    lin = AdaptedLinear(torch.nn.Linear(8, 5), 2, 3, AdapterSelection(), alpha=1.0)
    lin.adapter_a.grad = torch.randn(2, 3, 8)
    kept = [t.detach().clone() for t in (lin.adapter_a, lin.adapter_b, lin.adapter_scales, lin.adapter_a.grad)]
    out = convert(lin)
    assert out.weight.dtype != torch.float32
    now = (out.adapter_a, out.adapter_b, out.adapter_scales, out.adapter_a.grad)
    assert all(t.dtype == torch.float32 and torch.equal(t, k) for t, k in zip(now, kept))
    assert isinstance(out.adapter_a, torch.nn.Parameter) and out.adapter_a.requires_grad


def test_other_moves():
    lin = AdaptedLinear(torch.nn.Linear(8, 5), 2, 3, AdapterSelection())
    meta = lin.to("meta")
    assert meta.adapter_a.is_meta and meta.adapter_scales.is_meta and meta.weight.is_meta
    assert lin.to_empty(device="cpu").adapter_a.device.type == "cpu"
