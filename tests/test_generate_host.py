"""Drafting around stub models (CPU: the drawing kernel is replaced): what a block keeps, and what the models are fed."""

import weakref

import pytest
import torch

from ksdraft_amd.model import generate


@pytest.fixture
def drawn(monkeypatch):
    """The tokens that sample_tokens is to give, call after call."""
    queue = []
    monkeypatch.setattr(generate, "sample_tokens", lambda logits, u=None, t=None: queue.pop(0))
    return queue


def test_a_block_keeps_one_row_a_step(drawn):
    """No step's logits of all positions outlive the step."""
    alive, seen = [], []

    def model(tokens):
        assert all(ref() is None for ref in alive)
        logits = torch.randn(*tokens.shape, 11)
        seen.append(logits[:, -1].clone())
        alive.append(weakref.ref(logits.untyped_storage()))
        return logits, []
    drawn += [torch.tensor([t, t + 1]) for t in range(3)]
    tokens, rows = generate.draft_block(model, torch.zeros(2, 5, dtype=torch.int64), 3, temperatures=0.0)
    assert torch.equal(rows, torch.stack(seen, 1)) and tokens.tolist() == [[0, 1, 2], [1, 2, 3]]


def test_models_are_fed_tokens_only(drawn, monkeypatch):
    """A row without a distribution draws -1: the block says so, the models get token 0 in its place."""
    fed = []

    def model(tokens):
        fed.append(tokens.clone())
        return torch.zeros(*tokens.shape, 11), []
    monkeypatch.setattr(generate, "verify_draft", lambda logits, block, *a, **k: (block, logits))
    for dtype in (torch.int64, torch.int32):
        drawn[:] = [torch.tensor([-1, 3]), torch.tensor([5, -1])]
        block, logits = generate.speculative_step(model, model, torch.ones(2, 4, dtype=dtype), 2, temperatures=0.0)
        assert block.tolist() == [[-1, 5], [3, -1]] and logits.shape == (2, 3, 11)
        assert fed[-1].tolist() == [[1, 1, 1, 1, 0, 5], [1, 1, 1, 1, 3, 0]] and fed[-2].tolist() == [[1, 1, 1, 1, 0], [1, 1, 1, 1, 3]]
        assert all(t.dtype == dtype for t in fed[-3:])
