"""Which adapters a model's layers see: threads that serve different requests on one model, a training step between two serving
calls, copies and saved models (CPU)."""

import io
import threading
import time

import pytest
import torch

from ksdraft_amd.config import KSDraftConfig
from ksdraft_amd.model import KSDraftModel, add_adapters, select_adapters, selected_adapters
from ksdraft_amd.model.adapters import adapted_layers
from ksdraft_amd.train.adapter_step import AdapterTrainer


def model():
    cfg = KSDraftConfig(vocab_size=16, layers=2, d_model=32, rosa_streams=16, ks3_charts=24)
    return add_adapters(KSDraftModel(cfg), 4, 2)


def seen(m, pause=0.0):
    """The index of each layer in turn, as a call of the model reads it."""
    out = []
    for layer in adapted_layers(m):
        out.append(layer._index(torch.zeros(2, 3, layer.in_features)))
        time.sleep(pause)
    return out


def test_threads():
    m, wrong = model(), []
    ready = threading.Barrier(4)

    def serve(i):
        index = torch.tensor([i, -1])
        ready.wait()
        for _ in range(3):
            with selected_adapters(m, index):
                wrong.extend(x for x in seen(m, 0.001) if x is not index)
    threads = [threading.Thread(target=serve, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and seen(m) == [None] * 8


def test_nested_and_restored():
    m, first, second = model(), torch.tensor([0, 1]), torch.tensor([2, 3])
    select_adapters(m, first)
    with selected_adapters(m, second):
        assert all(x is second for x in seen(m))
        with selected_adapters(m, None):
            assert seen(m) == [None] * 8
        select_adapters(m, torch.tensor([1, 1]))  # for the rest of the block
    assert all(x is first for x in seen(m))
    with pytest.raises(KeyError):
        with selected_adapters(m, second):
            raise KeyError
    assert all(x is first for x in seen(m))
    for bad in (lambda: selected_adapters(m, torch.zeros(2)), lambda: selected_adapters(KSDraftModel(m.config), second)):
        with pytest.raises((TypeError, ValueError)):
            with bad():
                pass


def test_a_training_step_leaves_the_selection(monkeypatch):
    m, serving, batch = model(), torch.tensor([0, 1]), torch.tensor([2, 3])
    t = object.__new__(AdapterTrainer)
    t.model = m

    def loss(tokens, index, states=None):
        select_adapters(m, index)
        return (torch.zeros(()),) * 3
    monkeypatch.setattr(t, "loss", loss)
    monkeypatch.setattr(t, "backward", lambda loss: [x is batch for x in seen(m)] == [True] * 8 or pytest.fail("another batch's"))
    monkeypatch.setattr(t, "optimizer_step", lambda: None)
    select_adapters(m, serving)
    t.step(torch.zeros(2, 4, dtype=torch.int64), batch)
    assert all(x is serving for x in seen(m))


def test_saved_with_its_selection():
    m = model()
    select_adapters(m, torch.tensor([3, 0]))
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    again = torch.load(f, weights_only=False)
    assert all(x.tolist() == [3, 0] for x in seen(again))
    assert len({id(layer.selection) for layer in adapted_layers(again)}) == 1
    with selected_adapters(again, None):
        assert seen(again) == [None] * 8


def test_a_recomputed_pass_in_another_thread_does_not_wait():
    """A backward pass on the GPU runs in a thread of torch's, while its caller holds the block around it."""
    m, index = model(), torch.tensor([1, 2])

    class Recomputes(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, g):
            with selected_adapters(m, index):
                assert all(x is index for x in seen(m))
            return g
    x = torch.ones((), requires_grad=True)
    done = []

    def holder():
        with selected_adapters(m, None):
            t = threading.Thread(target=lambda: (Recomputes.apply(x).backward(), done.append(1)), daemon=True)
            t.start()
            t.join(20)
    holder()
    assert done
