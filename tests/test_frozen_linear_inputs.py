"""The inputs of a float model's frozen bfloat16 products are dense (CPU: stub layers; torch multiplies strided rows by a frozen
weight as a batch of products with a transposed right operand)."""

import pytest
import torch
from torch import nn
from torch.nn import functional as F

from ksdraft_amd.config import KSDraftConfig
from ksdraft_amd.model import AdjacentInjection, KSDraftModel, RosaMixer, add_adapters


@pytest.fixture
def batched(monkeypatch):
    """Calls of F.linear by how torch multiplies them: strided 3-D rows that no view folds, a bfloat16 weight without gradient."""
    seen, linear = [], F.linear

    def watched(x, w, bias=None):
        folds = x.dim() < 3 or x.stride(0) == x.stride(1) * x.shape[1] or x.shape[0] == 1
        if w.dtype == torch.bfloat16 and not w.requires_grad and not (x.is_contiguous() or folds):
            seen.append(tuple(x.shape))
        return linear(x, w, bias)
    monkeypatch.setattr(F, "linear", watched)
    return seen


def strided(B, T, S):
    return torch.randn(B, S, T).permute(0, 2, 1).bfloat16()


@pytest.mark.parametrize("targets", [None, ("q_proj",), ("out_proj",)])
def test_mixer(batched, targets):
    cfg = KSDraftConfig(vocab_size=16, layers=1, d_model=32, rosa_streams=16, ks3_charts=24)
    model = KSDraftModel(cfg).bfloat16().requires_grad_(False)
    if targets:
        model = add_adapters(model, 2, 4, targets=targets)
    mixer = model.blocks[0].rosa
    x = strided(2, 5, 16)
    if targets != ("out_proj",):
        want = F.linear(x.contiguous(), mixer.out_proj.weight, mixer.out_proj.bias)
        assert torch.equal(mixer._out(x, None), want)
        res = torch.randn(2, 5, 32).bfloat16()
        assert torch.equal(mixer._out(x, res), res + want)
    else:
        mixer._out(x, None)  # no adapter is selected: the base layer alone
    assert not batched


def test_trained_mixer_takes_its_input_as_it_is(monkeypatch):
    mixer = RosaMixer(32, 16).bfloat16()
    seen = []
    mixer.out_proj.register_forward_pre_hook(lambda m, a: seen.append(a[0]))
    x = strided(2, 5, 16)
    mixer._out(x, None)
    assert seen[0] is x


def test_injection_and_teacher(batched):
    inject = AdjacentInjection(32).bfloat16().requires_grad_(False)
    z = torch.randn(2, 5, 32).bfloat16()
    inject(z)
    inject(z, torch.randn(2, 5, 32).bfloat16())
    assert not batched
    cfg = KSDraftConfig(vocab_size=16, layers=1, d_model=32, rosa_streams=16, ks3_charts=24)
    model = KSDraftModel(cfg, teacher_dim=24).bfloat16().requires_grad_(False)
    model.blocks = nn.ModuleList()
    model.backbone(torch.zeros(2, 5, dtype=torch.int64), torch.randn(2, 9, 24).bfloat16()[:, 4:])
    assert not batched
