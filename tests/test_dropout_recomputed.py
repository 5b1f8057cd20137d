"""Forward passes that are run again for their backward pass: a module's counted stream would be another mask, so it is named or
the pass refused (CPU: the kernel is replaced by its formula)."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from ksdraft_amd.config import KSDraftConfig
from ksdraft_amd.kernels import adapters
from ksdraft_amd.kernels.dropout import Dropout, name_streams
from ksdraft_amd.model import KSDraftModel, add_adapters
from ksdraft_amd.model.adapters import AdaptedLinear, AdapterSelection
from tests.philox import mask
from tests.test_dropout_forward_mode import kernel  # noqa: F401


@pytest.mark.parametrize("reentrant", [False, True])
def test_named_or_refused(kernel, reentrant):  # noqa: F811
    drop, x = Dropout(0.5, seed=9), torch.randn(6, 16, requires_grad=True)
    lin = torch.nn.Linear(16, 16, bias=False)  # which saves its input, and so has the pass run again
    with torch.no_grad():
        lin.weight.copy_(torch.eye(16))
    net = torch.nn.Sequential(drop, lin)
    with pytest.raises(RuntimeError, match="stream"):
        checkpoint(net, x, use_reentrant=reentrant).sum().backward()
    drop.calls, lin.weight.grad = 0, None
    x.grad = None
    name_streams(net, 4)
    y = checkpoint(net, x, use_reentrant=reentrant)
    y.sum().backward()
    keep = mask(6, 16, 0.5, 9, 4)
    assert torch.equal(y.detach(), x.detach() * keep) and torch.equal(x.grad, keep)
    assert torch.allclose(lin.weight.grad, (x.detach() * keep).sum(0).expand(16, 16), rtol=1e-5, atol=1e-6)
    assert drop.calls == 0
    name_streams(drop, None)
    drop(x), drop(x)
    assert drop.calls == 2
    for bad in (-1, 1 << 32):
        with pytest.raises(ValueError):
            name_streams(drop, bad)


def test_adapted_layer(kernel, monkeypatch):  # noqa: F811
    seen = []
    monkeypatch.setattr(adapters, "adapter_linear_backward",
                        lambda g, s, *a: (torch.zeros_like(s.x), torch.zeros_like(s.a), torch.zeros_like(s.b)))
    train = adapters.adapter_linear_train

    def watched(x, a, b, index, scales, base, p, seed, stream):
        seen.append(stream)
        return train(x, a, b, index, scales, base, p, seed, stream)
    monkeypatch.setattr(adapters, "adapter_linear_train", watched)
    lin = AdaptedLinear(torch.nn.Linear(16, 8), 2, 3, AdapterSelection(), dropout=0.5, seed=9)
    lin.selection.index = torch.tensor([0, 1, -1])
    x = torch.randn(3, 16, requires_grad=True)
    with pytest.raises(RuntimeError, match="stream"):
        checkpoint(lin, x, use_reentrant=False).sum().backward()
    seen.clear()
    name_streams(lin, 12)
    checkpoint(lin, x, use_reentrant=False).sum().backward()
    assert seen == [12, 12]


def test_all_of_a_model():
    cfg = KSDraftConfig(vocab_size=16, layers=2, d_model=32, rosa_streams=16, ks3_charts=24, dropout=0.1)
    m = add_adapters(KSDraftModel(cfg), 2, 4, dropout=0.2)
    name_streams(m, 3)
    drops = [d for d in m.modules() if isinstance(d, Dropout)]
    assert len(drops) == 4 + 8 and all(d.next_stream() == 3 for d in drops)
    name_streams(m, None)
    assert [drops[0].next_stream() for _ in range(3)] == [0, 1, 2]
