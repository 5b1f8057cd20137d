"""A training step on targets that are no tokens: refused before the model runs, or, where the model does not
check its ids, left out of the cross entropy."""

import pytest
import torch
import torch.nn.functional as F

from ksdraft_amd.model import to_token_channel
from ksdraft_amd.train import IGNORE_INDEX
from ksdraft_amd.train.token_channel_step import TokenChannelTrainer
from tests.test_gpu_token_channel_step import _batch, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [IGNORE_INDEX, -1, 512])
def test_checked(bad):
    trainer = TokenChannelTrainer(to_token_channel(_model()))
    trainer.model.embedding.register_forward_pre_hook(lambda *a: pytest.fail("the model ran"))
    tokens, states = _batch()
    tokens[1, -1] = bad
    with pytest.raises(IndexError, match=str(bad)):
        trainer.loss(tokens, states)


def test_unchecked():
    trainer = TokenChannelTrainer(to_token_channel(_model(), check_ids=False))
    model = trainer.model
    tokens, states = _batch()
    tokens[0, -1], tokens[1, -1] = IGNORE_INDEX, 512
    loss, ce, ts = trainer.loss(tokens, states)
    with torch.no_grad():
        logits = model(tokens[:, :-1], states)[0][:, :-1]
        want = F.cross_entropy(logits.reshape(-1, 512).double(), tokens[:, 1:-1].reshape(-1))
    # 94 losses of some ten fp32 operations each on values below 16
    assert abs(ce.item() - want.item()) <= 32 * 2.0 ** -24 * 16
    trainer.backward(loss)
    assert all(bool(p.grad.isfinite().all()) for p in model.parameters() if p.grad is not None)
    trainer.optimizer_step()
    assert all(bool(p.isfinite().all()) for p in model.parameters())
