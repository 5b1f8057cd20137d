"""ScaledEmbedding's construction (CPU only: no kernel runs)."""

import pytest
import torch

from ksdraft_amd.kernels import ScaledEmbedding


@pytest.mark.parametrize("option", [dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)])
def test_options_that_it_lacks_are_refused(option):
    with pytest.raises(ValueError, match=next(iter(option))):
        ScaledEmbedding.from_float(torch.nn.Embedding(10, 4, **option))


def test_from_float_keeps_the_master():
    emb = torch.nn.Embedding(10, 4, padding_idx=-2)
    mod = ScaledEmbedding.from_float(emb, 2.0, out_dtype=torch.bfloat16, check_ids=False)
    assert mod.weight is emb.weight and (mod.padding_idx, mod.scale, mod.out_dtype, mod.check_ids) == (8, 2.0, torch.bfloat16, False)


@pytest.mark.parametrize("idx", [10, -11, 1 << 40])
def test_padding_out_of_range(idx):
    """Refused at once, not in the first backward."""
    with pytest.raises(ValueError, match="padding_idx"):
        ScaledEmbedding(10, 4, padding_idx=idx)
    assert ScaledEmbedding(10, 4, padding_idx=-10).padding_idx == -10
