"""The targets of a token/channel training step: what the losses are given (CPU only: no kernel runs)."""

import pytest
import torch

from ksdraft_amd.train import IGNORE_INDEX
from ksdraft_amd.train.token_channel_step import check_targets


@pytest.mark.parametrize("check", [True, False])
def test_tokens_pass_as_they_are(check):
    t = torch.tensor([[0, 9, 4], [3, 3, 9]])
    assert torch.equal(check_targets(t, 10, check), t)


@pytest.mark.parametrize("bad", [-1, IGNORE_INDEX, 10, 1 << 40, -(1 << 40)])
def test_others_are_refused_or_left_out(bad):
    t = torch.tensor([[0, 9, 4], [3, bad, 9]])
    with pytest.raises(IndexError, match=str(bad)):
        check_targets(t, 10, True)
    kept = check_targets(t, 10, False)
    assert torch.equal(kept, torch.where(t == bad, IGNORE_INDEX, t))
    logits = torch.randn(6, 10)
    loss = torch.nn.functional.cross_entropy(logits, kept.reshape(-1), ignore_index=IGNORE_INDEX)
    rows = [0, 1, 2, 3, 5]
    assert torch.equal(loss, torch.nn.functional.cross_entropy(logits[rows], t.reshape(-1)[rows]))
