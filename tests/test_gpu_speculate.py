"""Verification of drafted tokens and drawing against the definition in 64 bits on the CPU.

Tokens are whole numbers and equal. A draw is moved by an error e of a running sum only if its number lies within
e of a border: with sums in 64 bits (e below 1e-12) that has a chance below 1e-6 over all the draws here; a test u q < p
in 32-bit sums (e about 1e-7, a few hundred tests) one of 1e-4. The seeds are fixed, and an input with a number
within 1e-5 of its test's or 1e-9 of its draw's border would be no test of the kernel: `near` says so."""

import math

import pytest
import torch

from ksdraft_amd.kernels.speculate import sample_tokens, verify_draft

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def softmax64(row, T):
    """Probabilities, or None where there is no distribution."""
    x = row.double()
    if bool(torch.isnan(x).any()) or bool((x == math.inf).any()) or not bool(torch.isfinite(x).any()):
        return None
    e = torch.exp((x - x.max()) / T)
    return e / e.sum()


def drawn(w, u, near):
    run = torch.cumsum(w, 0)
    goal = u * run[-1]
    if float(run[-1]) > 0:
        near.append(float(((run - goal).abs() / run[-1]).min()))
    hit = (run > goal) & (w > 0)
    return int(hit.nonzero()[0]) if bool(hit.any()) else int((w > 0).nonzero()[-1])


def verify_cpu(target, tokens, u, draft=None, temps=None, lengths=None):
    B, rows, V = target.shape
    L = rows - 1
    out, acc, near, draws = torch.full((B, L + 1), -1), torch.zeros(B, dtype=torch.int64), [1.0], [1.0]
    for b in range(B):
        T = 1.0 if temps is None else float(temps[b])
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        t, new = 0, None
        while new is None:
            row = target[b, t]
            if not T > 0:
                x = row.float()
                best = -1 if bool(torch.isnan(x).any()) or bool((x == -math.inf).all()) else int((x == x.max()).nonzero()[0])
                if t == n or best != int(tokens[b, t]) or best < 0:
                    new = best
                    break
            else:
                p = softmax64(row, T)
                if t == n:
                    new = -1 if p is None else drawn(p, float(u[b, L]), draws)
                    break
                tok = int(tokens[b, t])
                ok = p is not None and 0 <= tok < V
                q = None
                if draft is not None:
                    d = draft[b, t].double()
                    empty = bool((d == -math.inf).all())
                    q = torch.zeros(V, dtype=torch.float64) if empty else softmax64(d, T)
                    ok = ok and q is not None
                if ok:
                    qt, pt = 1.0 if draft is None else float(q[tok]), float(p[tok])
                    if pt > 0:
                        near.append(abs(float(u[b, t]) * qt / pt - 1))
                    ok = float(u[b, t]) * qt < pt
                if not ok:
                    if p is None:
                        new = -1
                        break
                    if draft is None:
                        w = p.clone()
                        if 0 <= tok < V:
                            w[tok] = 0
                    else:
                        w = p if q is None else (p - q).clamp(min=0)
                    new = drawn(w if float(w.sum()) > 0 else p, float(u[b, L]), draws)
                    break
            out[b, t] = int(tokens[b, t])
            t += 1
        out[b, t], acc[b] = new, t
    assert min(near) > 1e-5 and min(draws) > 1e-9, "an input next to a border"
    return out, acc


def make(B, L, V, dtype, seed, greedy=0, peaks=8):
    """Rows with a broad bulk and a few likely tokens; the draft's a noisy copy, its tokens drawn from it."""
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, L + 1, V, generator=g) * 2
    z.scatter_add_(2, torch.randint(0, V, (B, L + 1, peaks), generator=g), 6 + 2 * torch.randn(B, L + 1, peaks, generator=g))
    target = z.to(TYPES[dtype])
    draft = (z[:, :L] + 0.5 * torch.randn(B, L, V, generator=g)).to(TYPES[dtype])
    temps = 0.5 + torch.rand(B, generator=g)
    temps[:greedy] = 0
    t = temps.clamp(min=1e-3)[:, None, None]
    noise = -torch.log(-torch.log(torch.rand(B, L, V, generator=g).clamp(1e-20, 1 - 1e-7)))
    tokens = (draft.float() / t + noise * (temps > 0)[:, None, None]).argmax(2)
    return target, draft, tokens, torch.rand(B, L + 1, generator=g), temps


def gpu(t):
    return None if t is None else t.to(DEV)


def both(target, tokens, u, draft=None, temps=None, lengths=None):
    out, acc = verify_draft(gpu(target), gpu(tokens), gpu(u), gpu(draft), gpu(temps), gpu(lengths))
    want = verify_cpu(target, tokens, u, draft, temps, lengths)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(acc.cpu(), want[1])
    return want


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("B,L,V", [(1, 1, 2), (3, 4, 7), (5, 3, 1000), (2, 16, 4099), (9, 5, 2048), (17, 2, 2049), (1, 70, 65)])
def test_against_definition(B, L, V, with_draft, dtype):
    target, draft, tokens, u, temps = make(B, L, V, dtype, 7 * V + L, greedy=B // 3)
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, L + 1, (B,), generator=g)
    d = draft if with_draft else None
    both(target, tokens, u, d, temps)
    both(target, tokens, u, d, temps, lengths)
    both(target, tokens, u.double(), d)


@pytest.mark.parametrize("dtype,V", [("bf16", 150144), ("fp16", 32003), ("fp32", 150144), ("bf16", 600001)])
def test_long_rows(dtype, V):
    target, draft, tokens, u, temps = make(2, 3, V, dtype, 5)
    for d in (draft, None):
        both(target, tokens, u, d, temps)
    got = [sample_tokens(gpu(target[:, 0]), gpu(u[:, k]), gpu(temps)) for k in range(4)]
    for k in range(4):
        assert torch.equal(got[k].cpu(), verify_cpu(target[:, :1], None, u[:, k:k + 1], None, temps)[0][:, 0])


@pytest.mark.parametrize("L", [20, 5])
def test_long_batches(L):
    """Batches whose positions go in several launches, and whose sums are 32-bit ones in one: streams refused early,
    late and never, greedy ones, every length; rows shared between the streams (strides of 0), their tokens and
    numbers their own."""
    B, V = 64, 30000
    target, draft, _, _, _ = make(1, L, V, "bf16", 51, peaks=4)
    g = torch.Generator().manual_seed(3)
    temps = torch.full((B,), 0.9)
    temps[::7] = 0
    tokens = torch.multinomial(torch.softmax(draft[0].float() / 0.9, 1), B, replacement=True, generator=g).t().contiguous()
    tokens[::7] = target[0, :L].float().argmax(1)
    tokens[7, 4], tokens[14, 0], tokens[21, L - 1], tokens[28, L // 2] = 1, 2, 3, 4
    u = torch.rand(B, L + 1, generator=g) * (torch.arange(B)[:, None] % 3 / 2).clamp(min=1e-3)  # 0.001, 0.5 and 1 times
    lengths = torch.randint(0, L + 1, (B,), generator=g)
    lengths[::2] = L
    for d in (draft, None):
        want = verify_cpu(target.expand(B, L + 1, V), tokens, u, None if d is None else d.expand(B, L, V), temps, lengths)
        for n in (lengths, None):
            if n is None:
                want = verify_cpu(target.expand(B, L + 1, V), tokens, u, None if d is None else d.expand(B, L, V), temps)
            got = verify_draft(gpu(target).expand(B, L + 1, V), gpu(tokens), gpu(u), None if d is None else gpu(d).expand(B, L, V),
                               gpu(temps), gpu(n))
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
        assert len(set(want[1].tolist())) >= min(L, 6)


def test_masks():
    """-inf and the type's lowest values, rows with one finite logit, with none, with NaN and +inf."""
    inf, nan = math.inf, math.nan
    for dtype in TYPES:
        target, draft, tokens, u, temps = make(12, 3, 301, dtype, 11)
        low = torch.finfo(TYPES[dtype]).min
        target[0, 0, ::2] = -inf
        target[1, :, 1:] = low
        target[2, 1] = -inf
        target[3, 0, 5:] = -inf
        draft[3, 0, :100] = -inf
        tokens[3, 0] = 200
        draft[4, 0] = -inf
        draft[5, 1, 7] = nan
        target[6, 0, 9] = nan
        target[7, 2, 300] = inf
        draft[8, 0, 3] = inf
        target[9, 3] = -inf
        target[10] = low
        draft[11] = target[11, :3]
        for T in (temps, temps * (torch.arange(12) % 2 == 0), None):
            if T is not None and not bool((T > 0).all()):
                tg = target.clone()
                tg[7, 2, 300] = 5.0  # +inf is a largest logit like any other where nothing is drawn
                both(tg, tokens, u, draft, T)
            else:
                both(target, tokens, u, draft, T)
                both(target, tokens, u, None, T)
    x = torch.full((3, 64), -inf)
    x[1, 40] = 2.0
    x[2, 3] = nan
    want = [-1, 40, -1]
    assert sample_tokens(gpu(x), gpu(torch.full((3,), 0.9))).tolist() == want
    assert sample_tokens(gpu(x), temperatures=0.0).tolist() == want
    y = torch.zeros(2, 64)
    y[0, 9] = y[0, 50] = inf
    assert sample_tokens(gpu(y), temperatures=0.0).tolist() == [9, 0]
    assert sample_tokens(gpu(y), gpu(torch.tensor([0.305, 0.305]))).tolist()[0] == -1


def test_numbers_and_tokens_out_of_range():
    target, draft, tokens, u, temps = make(6, 2, 500, "fp32", 3)
    tokens[0, 0], tokens[1, 0], tokens[2, 0] = -1, 500, 1 << 40
    u[3] = 0.0
    both(target, tokens, u, draft, temps)
    both(target, tokens, u, None, temps)
    both(target, tokens, u, draft, torch.zeros(6))
    big = u.clone()
    big[:, 2] = 1.0  # the last token with a weight
    out, acc = verify_draft(gpu(target), gpu(tokens), gpu(big), gpu(draft), gpu(temps))
    for b in range(6):
        assert 0 <= int(out[b, acc[b]]) < 500
    lengths = torch.tensor([-3, 0, 1, 2, 99, 2])
    both(target, tokens, u, draft, temps, lengths)


def test_temperatures():
    target, draft, tokens, u, _ = make(8, 3, 700, "bf16", 23)
    cold = torch.tensor([1e-30, 1e-3, 1e-2, 0.1, 10.0, 1e4, -1.0, math.nan])
    got = verify_draft(gpu(target), gpu(tokens), gpu(u), gpu(draft), gpu(cold))
    want = verify_cpu(target, tokens, u, draft, cold)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert torch.equal(verify_draft(gpu(target), gpu(tokens), gpu(u), gpu(draft), 0.7)[0],
                       verify_draft(gpu(target), gpu(tokens), gpu(u), gpu(draft), torch.full((8,), 0.7, device=DEV))[0])
    assert torch.equal(verify_draft(gpu(target), gpu(tokens), None, temperatures=0.0)[0].cpu(),
                       verify_cpu(target, tokens, u, None, torch.zeros(8))[0])


def test_layouts():
    """Strides, int32 tokens, broadcast rows, a slice of a larger buffer that ends with it."""
    target, draft, tokens, u, temps = make(4, 3, 333, "fp16", 31)
    want = verify_cpu(target, tokens, u, draft, temps)[0]
    wide = torch.zeros(4, 4, 340, dtype=torch.float16)
    wide[:, :, 7:] = target
    turned = target.transpose(0, 1).contiguous().transpose(0, 1)
    last = target.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    for t in (wide[:, :, 7:], turned, last):
        assert torch.equal(verify_draft(gpu(t), gpu(tokens.int()), gpu(u), gpu(draft), gpu(temps))[0].cpu(), want)
    on_gpu = wide.to(DEV)[:, :, 7:]
    assert torch.equal(verify_draft(on_gpu, gpu(tokens), gpu(u), gpu(draft), gpu(temps))[0].cpu(), want)
    same = target[:1].expand(4, 4, 333)
    assert torch.equal(verify_draft(gpu(target[:1]).expand(4, 4, 333), gpu(tokens), gpu(u), gpu(draft), gpu(temps))[0].cpu(),
                       verify_cpu(same, tokens, u, draft, temps)[0])
    shaped = sample_tokens(gpu(target), gpu(u), 0.8)
    assert shaped.shape == (4, 4)
    assert torch.equal(shaped.reshape(-1).cpu(), verify_cpu(target.reshape(16, 1, 333), None, u.reshape(16, 1), None,
                                                            torch.full((16,), 0.8))[0][:, 0])
    empty = verify_draft(gpu(target[:0]), gpu(tokens[:0]), gpu(u[:0]), gpu(draft[:0]))
    assert empty[0].shape == (0, 4) and empty[1].shape == (0,)
    assert sample_tokens(gpu(target[0, 0]), gpu(u[0, 0]), 0.0).shape == ()


def test_frequencies():
    """Verified and drawn tokens are distributed as the target's own: 20000 streams over 6 tokens, each count
    within 5 standard deviations."""
    n = 20000
    p, q = torch.tensor([0.4, 0.3, 0.15, 0.1, 0.05, 0.0]), torch.tensor([0.1, 0.1, 0.3, 0.3, 0.1, 0.1])
    g = torch.Generator().manual_seed(2)
    tokens = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
    u = torch.rand(n, 2, generator=g)
    target = p.log().to(DEV).expand(n, 2, 6)
    out, acc = verify_draft(target, gpu(tokens), gpu(u), q.log().to(DEV).expand(n, 1, 6))
    counts = torch.bincount(out[:, 0].cpu(), minlength=6).double()
    for i in range(6):
        assert abs(float(counts[i]) - n * float(p[i])) <= 5 * math.sqrt(n * float(p[i]) * (1 - float(p[i]))) + 1e-9
    share = float(torch.minimum(p, q).sum())
    assert abs(float(acc.double().mean()) - share) < 5 * math.sqrt(share * (1 - share) / n)


def test_captured_and_on_another_stream():
    target, draft, tokens, u, temps = (gpu(t) for t in make(5, 4, 3001, "bf16", 41, greedy=2))
    want = verify_draft(target, tokens, u, draft, temps)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = verify_draft(target, tokens, u, draft, temps)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = verify_draft(target, tokens, u, draft, temps)
        other = sample_tokens(target[:, 0], u[:, 0], temps)
    g = torch.Generator(device=DEV).manual_seed(0)
    for _ in range(4):
        u.copy_(torch.rand(5, 5, device=DEV, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        eager = verify_draft(target, tokens, u, draft, temps)
        assert torch.equal(kept[0], eager[0]) and torch.equal(kept[1], eager[1])
        assert torch.equal(other, sample_tokens(target[:, 0], u[:, 0], temps))


def test_refusals():
    target, draft, tokens, u, temps = (gpu(t) for t in make(3, 2, 50, "fp32", 1))
    for f in (lambda: verify_draft(target[0], tokens, u), lambda: verify_draft(target, tokens[:, :1], u),
              lambda: verify_draft(target, tokens, u[:, :2]), lambda: verify_draft(target, tokens, u, draft[:, :1]),
              lambda: verify_draft(target, tokens, u, temperatures=temps[:2]), lambda: verify_draft(target, tokens, u, temperatures=-1.0),
              lambda: verify_draft(target, tokens, u, temperatures=temps.double()), lambda: verify_draft(target, tokens, None),
              lambda: verify_draft(target, None, u), lambda: verify_draft(target, tokens, u, lengths=tokens[:, 0][:2]),
              lambda: verify_draft(target[:, :0], tokens, u), lambda: sample_tokens(target, u[:, :2]),
              lambda: sample_tokens(target[..., :0], u), lambda: sample_tokens(target)):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: verify_draft(target.double(), tokens, u), lambda: verify_draft(target, tokens.float(), u),
              lambda: verify_draft(target, tokens, u.half()), lambda: verify_draft(target, tokens, u, draft.half())):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(RuntimeError):
        verify_draft(target.cpu(), tokens, u)
