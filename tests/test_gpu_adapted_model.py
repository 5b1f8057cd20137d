"""Adapters, dropout and verification on a draft model, together as they are used: a small draft (2 layers,
d 256, 64 Rosa streams, 384 charts, vocabulary 512), as floats and with int8 products. Every adapted layer is
checked against fp64 arithmetic on its own input, base output and, in training, upstream gradient."""

import pytest
import torch

from ksdraft_amd.config import KSDraftConfig
from ksdraft_amd.kernels.dropout import dropout
from ksdraft_amd.kernels.speculate import verify_draft
from ksdraft_amd.model import (KSDraftModel, add_adapters, draft_block, select_adapters, speculative_step, to_int8,
                               to_token_channel)
from ksdraft_amd.model.adapters import AdaptedLinear, AdapterSelection, adapted_layers, adapter_parameters
from ksdraft_amd.train.adapter_step import AdapterTrainer
from tests.philox import mask

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TARGETS = ("q_proj", "k_proj", "v_proj", "out_proj", "head")


def make(**kwargs):
    torch.manual_seed(0)
    m = KSDraftModel(KSDraftConfig(vocab_size=512, layers=2, d_model=256, rosa_streams=64, ks3_charts=384, **kwargs)).to(DEV)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.endswith(("up.weight", "out_proj.weight", "embedding.weight")):
                p.normal_(0, 0.02)
    return m


def adapted(base, count=3, rank=8, **kwargs):
    m = add_adapters(base, count, rank, targets=TARGETS, **kwargs)
    g = torch.Generator().manual_seed(4)
    with torch.no_grad():
        for layer in adapted_layers(m):
            layer.adapter_b.copy_(torch.randn(layer.adapter_b.shape, generator=g) * 0.05)
    return m


def tokens(B=3, T=33, seed=0):
    return torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(seed)).to(DEV)


INDEX = torch.tensor([2, -1, 0])


@pytest.mark.parametrize("kind", ["float", "int8", "token_channel"])
def test_serving(kind):
    """Each sequence gets its adapter; without one, and without a selection, the base's own bits."""
    base = make()
    base = base if kind == "float" else to_int8(base) if kind == "int8" else to_token_channel(base)
    m = adapted(base).eval()
    base.eval()
    t = tokens()
    with torch.no_grad():
        # torch's float products of a strided input (the output projection's) round by whether the weight is frozen
        plain = m(t)[0] if kind == "float" else base(t)[0]
        assert torch.equal(m(t)[0], plain)
        select_adapters(m, INDEX.to(DEV))
        seen = []
        for layer in adapted_layers(m):
            layer.base.register_forward_hook(lambda mod, a, out, l=layer: seen.append((l, a[0].clone(), out.clone())))
            layer.register_forward_hook(lambda mod, a, k, out: seen.append((mod, out.clone(), k.get("residual"))), with_kwargs=True)
        logits = m(t)[0]
        assert len(seen) == 2 * len(adapted_layers(m))
        for (layer, x, y), (same, out, res) in zip(seen[::2], seen[1::2]):
            assert layer is same
            K, N, r = layer.in_features, layer.out_features, 8
            want, size = y.double().reshape(3, -1, N), y.double().abs().reshape(3, -1, N)
            if kind == "float" and res is not None:  # added around the base layer, not by it
                want, size = want + res.double(), size + res.double().abs()
            for s, i in enumerate(INDEX.tolist()):
                if i >= 0:
                    xs, a, b = x.double().reshape(3, -1, K)[s], layer.adapter_a[i].double(), layer.adapter_b[i].double()
                    want[s] += xs @ a.t() @ b.t()
                    size[s] += xs.abs() @ a.abs().t() @ b.abs().t()
            err = (out.double().reshape(want.shape) - want).abs()
            assert bool((err <= 2 * (K + r + 6) * U * size).all())
            if kind != "float" or res is None:
                assert torch.equal(out.reshape(3, -1, N)[1], y.reshape(3, -1, N)[1])
        assert not torch.equal(logits[0], plain[0]) and not torch.equal(logits[2], plain[2])
        assert torch.equal(logits[1], plain[1])  # the other sequences' adapters do not reach it
        select_adapters(m, None)
        assert torch.equal(m(t)[0], plain)


@pytest.mark.parametrize("kind", ["float", "token_channel"])
def test_training(kind):
    base = make()
    base = base if kind == "float" else to_token_channel(base)
    m = adapted(base, dropout=0.2, seed=11)
    trainer = AdapterTrainer(m, lr=1e-3, grad_clip=1.0, loss_scale=1024.0)
    m.train()
    frozen = {n: p.detach().clone() for n, p in m.named_parameters() if "adapter_" not in n}
    seen = {}

    def keep(mod, a, out):
        seen[mod] = [a[0].detach().clone()]
        out.register_hook(lambda g: seen[mod].append(g.clone()))
    for layer in adapted_layers(m):
        layer.register_forward_hook(keep)
    index = INDEX.to(DEV)
    loss, ce, ts = trainer.loss(tokens(), index)
    trainer.backward(loss)
    for layer in adapted_layers(m):
        x, g = seen[layer]
        K, N = layer.in_features, layer.out_features
        x, g = x.double().cpu().reshape(-1, K), g.double().cpu().reshape(-1, N)
        x = x * mask(x.shape[0], K, 0.2, layer.dropout.seed, 0).double()
        which = INDEX.repeat_interleave(32)
        for i in range(3):
            at = which == i
            a, b = layer.adapter_a[i].detach().double().cpu(), layer.adapter_b[i].detach().double().cpu()
            for got, want, size in ((layer.adapter_a.grad[i], (g[at] @ b).t() @ x[at], (g[at].abs() @ b.abs()).t() @ x[at].abs()),
                                    (layer.adapter_b.grad[i], g[at].t() @ (x[at] @ a.t()), g[at].abs().t() @ (x[at].abs() @ a.abs().t()))):
                assert bool(((got.double().cpu() - want).abs() <= 2 * (K + N + 32 + 8) * U * size + 1e-37).all())
    grads = [p.grad.clone() for p in adapter_parameters(m)]
    assert any(bool(g.any()) for g in grads)
    total = sum(float(g.double().pow(2).sum()) for g in grads) ** 0.5 / 1024.0
    trainer.optimizer_step()
    assert abs(trainer.grad_norm.item() - total) <= 3 * U * total
    for n, p in m.named_parameters():
        if "adapter_" not in n:
            assert torch.equal(p, frozen[n]) and p.grad is None
    assert all(l.dropout.calls == 1 for l in adapted_layers(m))
    # an adapter that no sequence has is as it was, but for the optimizer's decay (0)
    assert not bool(adapted_layers(m)[0].adapter_b.grad[1].any())
    for _ in range(2):
        assert all(bool(torch.isfinite(v)) for v in trainer.step(tokens(seed=1), index))


def test_step_repeats():
    runs = []
    for _ in range(2):
        m = adapted(to_token_channel(make()), dropout=0.1, seed=3)
        torch.manual_seed(1)
        trainer = AdapterTrainer(m)
        trainer.step(tokens(), INDEX.to(DEV))
        runs.append([p.detach().clone() for p in adapter_parameters(m)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_block_dropout():
    """config.dropout: the residual adds take dropout's output, in training only."""
    m = make(dropout=0.25)
    plain = make()
    plain.load_state_dict(m.state_dict())
    t = tokens()
    with torch.no_grad():
        m.eval(), plain.eval()
        assert torch.equal(m(t)[0], plain(t)[0])
    m.train()
    b = m.blocks[0]
    seen = {}
    b.rosa.register_forward_hook(lambda mod, a, out: seen.update(y=out.detach().clone()))
    b.injection.register_forward_pre_hook(lambda mod, a: seen.update(h=a[0].detach().clone()))
    b.register_forward_pre_hook(lambda mod, a: seen.update(x=a[0].detach().clone()))
    m(t)[0].sum().backward()
    assert torch.equal(seen["h"], dropout(seen["y"], 0.25, b.drop_attn.seed, 0, seen["x"]))
    assert b.drop_attn.calls == b.drop_ffn.calls == 1 and all(p.grad is not None for p in b.rosa.out_proj.parameters())


def test_drafting():
    """Serve, draft and verify: adapted requests draft blocks that the base verifies."""
    base = to_token_channel(make()).eval()
    m = adapted(base).eval()
    select_adapters(m, INDEX.to(DEV))
    t = tokens(T=9)
    g = torch.Generator().manual_seed(0)
    u = torch.rand(3, 9, generator=g).to(DEV)
    block, rows = draft_block(m, t, 4, u[:, :4], 0.8)
    with torch.no_grad():
        logits = m(torch.cat([t, block], 1))[0]
    out, accepted = speculative_step(m, base, t, 4, u, 0.8)
    with torch.no_grad():
        target = base(torch.cat([t, block], 1))[0][:, 8:]
    want = verify_draft(target, block, u[:, 4:], draft_logits=rows, temperatures=0.8)
    assert torch.equal(out, want[0]) and torch.equal(accepted, want[1])
    # the draft model verifies its own block whole: p = q
    again, all_in = verify_draft(rows_of(logits, rows), block, u[:, 4:], draft_logits=rows, temperatures=0.8)
    assert all_in.tolist() == [4, 4, 4] and torch.equal(again[:, :4], block)
    # a target of another type: both as floats, q still what the block was drawn from
    half = speculative_step(m, lambda s: base(s)[0].bfloat16(), t, 4, u, 0.8)
    want = verify_draft(target.bfloat16().float(), block, u[:, 4:], draft_logits=rows, temperatures=0.8)
    assert torch.equal(half[0], want[0]) and torch.equal(half[1], want[1])
    # greedily the tokens are the target's own, whatever is proposed
    with pytest.raises(ValueError):
        speculative_step(m, base, t[:1], 4, temperatures=0.0)  # three adapters, one sequence
    select_adapters(m, INDEX[:1].to(DEV))
    seen = t
    for _ in range(3):
        out, accepted = speculative_step(m, base, seen[:1], 4, temperatures=0.0)
        n = int(accepted[0])
        new = seen[:1]
        for k in range(n + 1):
            with torch.no_grad():
                best = base(new)[0][:, -1].argmax(-1)
            assert int(best) == int(out[0, k])
            new = torch.cat([new, best[:, None]], 1)
        assert out[0, n + 1:].tolist() == [-1] * (4 - n)
        seen = new
    for bad in (lambda: draft_block(m, t, 0), lambda: draft_block(m, t, 4, u), lambda: speculative_step(m, base, t, 4, u[:, :4])):
        with pytest.raises(ValueError):
            bad()


def rows_of(logits, rows):
    """The target's rows where the draft is its own target: the rows that the block was drawn from, then the next."""
    return torch.cat([rows, logits[:, -1:]], 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_mode_without_gradients(dtype):
    """A layer in training mode drops with and without gradients: the same streams, the same bits."""
    torch.manual_seed(1)
    base = torch.nn.Linear(96, 80, device=DEV, dtype=dtype)
    layers = [AdaptedLinear(base, 2, 8, AdapterSelection(), dropout=0.5, seed=3) for _ in range(2)]
    layers[1].load_state_dict(layers[0].state_dict())
    x = torch.randn(3, 5, 96, device=DEV, dtype=dtype)
    for layer in layers:
        layer.selection.index = torch.tensor([1, -1, 0], device=DEV)
        torch.nn.init.normal_(layer.adapter_b, generator=torch.Generator(DEV).manual_seed(5))
    y = layers[0](x)
    with torch.no_grad():
        z = layers[1](x)
        assert layers[1].dropout.calls == layers[0].dropout.calls == 1
        assert torch.equal(y, z) and not z.requires_grad
        layers[1].eval()
        assert not torch.equal(y, layers[1](x))
        layers[1].train()
        layers[1].dropout.p = 1.0
        assert torch.equal(layers[1](x), base(x))


@pytest.mark.parametrize("kind", ["float", "token_channel"])
def test_an_adapter_for_each_token(kind):
    """Indices (B, T), out of range for none, on layers of (B, T, K) and of flattened inputs."""
    base = make()
    m = adapted(base if kind == "float" else to_token_channel(base)).eval()
    index = torch.randint(-1, 4, (3, 33), generator=torch.Generator().manual_seed(8))
    select_adapters(m, index.to(DEV))
    seen = []
    for layer in adapted_layers(m):
        layer.base.register_forward_hook(lambda mod, a, out, l=layer: seen.append((l, a[0].clone(), out.clone())))
        layer.register_forward_hook(lambda mod, a, k, out: seen.append((mod, out.clone(), k.get("residual"))), with_kwargs=True)
    with torch.no_grad():
        m(tokens())
    assert len(seen) == 2 * len(adapted_layers(m))
    at = index.reshape(-1).to(DEV)
    for (layer, x, y), (same, out, res) in zip(seen[::2], seen[1::2]):
        assert layer is same
        K, N, r = layer.in_features, layer.out_features, 8
        want, size = y.double().reshape(-1, N), y.double().abs().reshape(-1, N)
        if kind == "float" and res is not None:
            want, size = want + res.double().reshape(-1, N), size + res.double().abs().reshape(-1, N)
        xs = x.double().reshape(-1, K)
        for i in range(3):
            a, b, of = layer.adapter_a[i].double(), layer.adapter_b[i].double(), at == i
            want[of] += xs[of] @ a.t() @ b.t()
            size[of] += xs[of].abs() @ a.abs().t() @ b.abs().t()
        err = (out.double().reshape(want.shape) - want).abs()
        assert bool((err <= 2 * (K + r + 6) * U * size).all())
