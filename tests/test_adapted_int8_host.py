"""An adapted mixer of int8 projections with no adapter selected takes the unadapted mixer's joint calls (CPU: the choice only)."""

import pytest
import torch
from torch import nn

from ksdraft_amd.kernels.linear import Int8Linear
from ksdraft_amd.model import RosaMixer
from ksdraft_amd.model.adapters import AdaptedLinear, AdapterSelection

NAMES = ("q_proj", "k_proj", "v_proj", "out_proj")


def int8(lin: nn.Linear) -> Int8Linear:
    """An Int8Linear of its sizes without codes, which are made on the GPU."""
    out = Int8Linear.__new__(Int8Linear)
    nn.Module.__init__(out)
    out.in_features, out.out_features = lin.in_features, lin.out_features
    out.weight, out.bias = lin.weight, lin.bias
    return out


@pytest.mark.parametrize("targets", [("q_proj",), NAMES])
def test_choice(targets):
    mixer, selection = RosaMixer(32, 16), AdapterSelection()
    assert not mixer._int8_projections()
    for name in NAMES:
        setattr(mixer, name, int8(getattr(mixer, name)))
    assert mixer._int8_projections()
    for name in targets:
        setattr(mixer, name, AdaptedLinear(getattr(mixer, name), 2, 4, selection))
    assert mixer._int8_projections() and isinstance(mixer._unadapted(mixer.out_proj), Int8Linear)
    selection.index = torch.tensor([0])
    assert not mixer._int8_projections()
    assert isinstance(mixer._unadapted(mixer.out_proj), Int8Linear) == ("out_proj" not in targets)
    selection.index = None
    assert mixer._int8_projections()
