"""The token/channel training step at a small shape: a 2-layer draft (d 256, 64 Rosa streams, 384
KS3 charts, vocabulary 512) through to_token_channel and TokenChannelTrainer.

Each TokenChannelLinear's output is checked against 64-bit arithmetic on the codes of its own input
(five fp32 roundings of the values that meet), the clip against the norm of all gradients in fp64
(the norm is one rounding of an fp64 sum and one division; the factor two more operations), the
step's repeatability bit for bit."""

import math

import pytest
import torch

from ksdraft_amd.config import KSDraftConfig
from ksdraft_amd.kernels.embedding import ScaledEmbedding
from ksdraft_amd.kernels.token_channel import TokenChannelLinear
from ksdraft_amd.model import KSDraftModel, int8_surfaces, to_int8, to_token_channel
from ksdraft_amd.train.int8_step import Int8DraftTrainer
from ksdraft_amd.train.token_channel_step import TokenChannelTrainer
from tests.test_gpu_token_channel import close, rows_cpu

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _model():
    torch.manual_seed(0)
    cfg = KSDraftConfig(vocab_size=512, layers=2, d_model=256, rosa_streams=64, ks3_charts=384)
    m = KSDraftModel(cfg, teacher_dim=256).to(DEV)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.endswith(("up.weight", "out_proj.weight", "teacher_proj.weight", "embedding.weight")):
                p.normal_(0, 0.02)
    return m


def _batch(seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 512, (2, 49), generator=g).to(DEV),
            torch.randn(2, 48, 256, generator=g).to(torch.bfloat16).to(DEV))


def test_surfaces():
    model = to_token_channel(_model(), embedding_scale=4.0)
    assert int8_surfaces(model)["scales"] == "token_channel"
    assert isinstance(model.embedding, ScaledEmbedding) and model.embedding.weight is model.head.weight
    tokens, states = _batch()
    seen = []
    for name, mod in model.named_modules():
        if isinstance(mod, TokenChannelLinear):
            mod.register_forward_hook(lambda m, a, k, out, n=name: seen.append((n, m, a[0].detach(), k.get("residual"), out.detach())),
                                      with_kwargs=True)
    logits, _ = model(tokens[:, :-1], states)
    assert logits.shape == (2, 48, 512) and len(seen) == 2 * 4 + 2
    for name, mod, x, res, out in seen:
        xq, xs = rows_cpu(x.reshape(-1, x.shape[-1]))
        wq, ws = rows_cpu(mod.weight.detach())
        main = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
        ref, size = main.clone(), main.abs()
        for extra in (mod.bias, res):
            if extra is not None:
                e = extra.detach().double().cpu().reshape(-1, out.shape[-1])
                ref, size = ref + e, size + e.abs()
        close(out.reshape(-1, out.shape[-1]), ref, size, out.dtype)
    rows = model.embedding(tokens)
    assert torch.equal(rows, (model.embedding.weight.detach() * 4.0)[tokens])


def test_step_clips_and_repeats():
    runs = []
    for _ in range(2):
        trainer = TokenChannelTrainer(to_token_channel(_model()), lr=1e-3, grad_clip=0.05, loss_scale=4096.0)
        loss, ce, ts = trainer.loss(*_batch())
        trainer.backward(loss)
        grads = [p.grad.clone() for p in trainer.model.parameters() if p.grad is not None]
        total = math.sqrt(sum(float(g.double().pow(2).sum()) for g in grads)) / 4096.0
        trainer.optimizer_step()
        assert abs(trainer.grad_norm.item() - total) <= 3 * 2.0 ** -24 * total
        runs.append((loss.detach(), grads, [p.detach().clone() for p in trainer.model.parameters()]))
    assert torch.equal(runs[0][0], runs[1][0])
    for a, b in zip(runs[0][1], runs[1][1]):
        assert torch.equal(a, b)
    for a, b in zip(runs[0][2], runs[1][2]):
        assert torch.equal(a, b)


def test_steps_learn():
    """On one batch the loss falls, about as it does with the group-scaled surfaces."""
    def run(trainer):
        tokens, states = _batch(3)
        return [trainer.step(tokens, states)[1].item() for _ in range(12)]
    ours = run(TokenChannelTrainer(to_token_channel(_model()), lr=2e-3))
    theirs = run(Int8DraftTrainer(to_int8(_model(), trainable=True), lr=2e-3))
    assert ours[-1] < ours[0] - 0.5 * (theirs[0] - theirs[-1]) and ours[-1] < ours[0]


def test_refusals():
    with pytest.raises(ValueError):
        TokenChannelTrainer(to_int8(_model(), trainable=True))
    with pytest.raises(ValueError):
        TokenChannelTrainer(to_token_channel(_model()), loss_scale=3.0)
