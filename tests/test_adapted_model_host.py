"""Adapters on a model: what is wrapped, frozen, selected and refused (CPU: construction only)."""

import copy

import pytest
import torch

from ksdraft_amd.config import KSDraftConfig
from ksdraft_amd.model import (AdaptedLinear, KSDraftModel, adapter_parameters, adapter_state_dict, add_adapters,
                               select_adapters, to_int8, to_token_channel)
from ksdraft_amd.model.adapters import AdapterSelection, adapted_layers
from ksdraft_amd.train.adapter_step import AdapterTrainer


def model(**kwargs):
    return KSDraftModel(KSDraftConfig(vocab_size=64, layers=2, d_model=32, rosa_streams=16, ks3_charts=24, **kwargs))


def test_added():
    base = model()
    m = add_adapters(base, 3, 4, targets=("q_proj", "out_proj", "head", "up"), alpha=8.0, dropout=0.1, seed=5)
    layers = adapted_layers(m)
    assert len(layers) == 2 + 2 + 1 + 2 and not adapted_layers(base)
    assert all(p.requires_grad == ("adapter_" in n) for n, p in m.named_parameters())
    assert all(p.requires_grad for p in base.parameters())
    assert len(adapter_parameters(m)) == 2 * len(layers)
    assert m.head.weight is m.embedding.weight and m.head.out_features == 64
    assert sorted(l.dropout.seed for l in layers) == list(range(5, 5 + len(layers)))
    assert torch.equal(layers[0].adapter_scales, torch.full((3,), 2.0)) and not bool(layers[0].adapter_b.any())
    keys = adapter_state_dict(m)
    assert len(keys) == 3 * len(layers) and all("adapter_" in k for k in keys)
    other = add_adapters(base, 3, 4, targets=("q_proj", "out_proj", "head", "up"))
    missing, unexpected = other.load_state_dict(keys, strict=False)
    assert not unexpected and torch.equal(adapted_layers(other)[0].adapter_a, layers[0].adapter_a)
    index = torch.tensor([0, 1])
    select_adapters(m, index)
    assert all(l.selection.index is index for l in layers)
    assert all(l.selection.index is None for l in adapted_layers(copy.deepcopy(m)))


def test_index_of_an_input():
    lin = AdaptedLinear(torch.nn.Linear(8, 4), 2, 3, AdapterSelection())
    x = torch.zeros(2, 5, 8)
    assert lin._index(x) is None
    for index in (torch.tensor([0, 1]), torch.zeros(2, 5, dtype=torch.int64)):
        lin.selection.index = index
        assert lin._index(x) is index
        assert torch.equal(lin._index(x.reshape(10, 8)), index.reshape(2, -1).expand(2, 5).reshape(-1))
    for bad in (torch.zeros(3, dtype=torch.int64), torch.zeros(0, dtype=torch.int64)):
        lin.selection.index = bad
        with pytest.raises(ValueError):
            lin._index(x)


def test_refusals():
    m = model()
    for kwargs in (dict(count=0, rank=4), dict(count=1, rank=129), dict(count=1, rank=4, targets=("embedding",)),
                   dict(count=1, rank=4, targets=()), dict(count=1, rank=4, targets=("teacher_proj",))):
        with pytest.raises(ValueError):
            add_adapters(m, **kwargs)
    with pytest.raises(ValueError):
        add_adapters(add_adapters(m, 1, 4), 1, 4)
    for convert in (to_int8, to_token_channel):
        with pytest.raises(ValueError):
            convert(add_adapters(m, 1, 4))
    with pytest.raises(TypeError):
        AdaptedLinear(torch.nn.LayerNorm(8), 1, 4, AdapterSelection())
    with pytest.raises(ValueError):
        select_adapters(m, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        select_adapters(add_adapters(m, 1, 4), torch.zeros(2))
    with pytest.raises(ValueError):
        AdapterTrainer(m)


def test_dropout_in_blocks():
    assert all(b.drop_attn is None and b.drop_ffn is None for b in model().blocks)
    m = model(dropout=0.2)
    assert all(b.drop_attn.p == 0.2 and b.drop_ffn.p == 0.2 for b in m.blocks)
    assert set(m.state_dict()) == set(model().state_dict())
    for p in (-0.1, 1.5):
        with pytest.raises(ValueError):
            model(dropout=p)
