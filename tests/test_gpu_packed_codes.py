"""TokenChannelLinear's stored codes follow the master: every way to change it that torch can see leads to
the output of the unpacked layer, bit for bit."""

import copy

import pytest
import torch

from ksdraft_amd.kernels import ScaledEmbedding, TokenChannelLinear
from ksdraft_amd.train import AdamWRequant

pytestmark = pytest.mark.gpu
DEV = "cuda"


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def fresh(mod, x):
    other = TokenChannelLinear(mod.in_features, mod.out_features, bias=False).to(DEV)
    other.weight = mod.weight
    return other(x)


def write(mod):
    mod.weight.copy_(randn(*mod.weight.shape, seed=5))


def write_part(mod):
    mod.weight[3:5] *= 2


def assign(mod):
    mod.weight = torch.nn.Parameter(randn(*mod.weight.shape, seed=6))


def swap_data(mod):
    mod.weight.data = randn(*mod.weight.shape, seed=7)


def average(mod):
    mod.weight.lerp_(randn(*mod.weight.shape, seed=8), 0.1)


@pytest.mark.parametrize("change", [write, write_part, assign, swap_data, average])
@torch.no_grad()
def test_changed_master(change):
    mod = TokenChannelLinear.from_float(torch.nn.Linear(200, 77, bias=False).to(DEV)).pack()
    x = randn(9, 200, seed=1)
    before = mod(x)
    for _ in range(2):
        change(mod)
        y = mod(x)
        assert torch.equal(y, fresh(mod, x)) and not torch.equal(y, before)
        held = mod._packed
        assert torch.equal(mod(x), y) and mod._packed is held  # stored again, once
    assert torch.equal(copy.deepcopy(mod)(x), y)


@pytest.mark.parametrize("optimizer", [torch.optim.SGD, AdamWRequant])
@pytest.mark.parametrize("rows", [50, 900])
def test_tied_master_stepped_through_the_lookup(optimizer, rows):
    """900 x 96 is large enough for the optimizer's own kernel, 50 x 96 is not."""
    emb = ScaledEmbedding(rows, 96).to(DEV)
    head = TokenChannelLinear(96, rows, bias=False)
    head.weight = emb.weight
    with torch.no_grad():
        emb.weight.copy_(randn(rows, 96))
    head.pack()
    opt, x = optimizer(emb.parameters(), lr=0.1), randn(4, 96, seed=2)
    for _ in range(2):
        with torch.no_grad():
            before = head(x)
        emb(torch.arange(rows, device=DEV)).sum().backward()
        opt.step()
        with torch.no_grad():
            y = head(x)
            assert torch.equal(y, fresh(head, x)) and not torch.equal(y, before)


def test_inference_master():
    with torch.inference_mode():
        mod = TokenChannelLinear(96, 40, bias=False).to(DEV)
        mod.weight.copy_(randn(40, 96))
        x = randn(4, 96, seed=2)
        assert torch.equal(mod.pack()(x), fresh(mod, x))
