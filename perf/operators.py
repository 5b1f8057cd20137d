"""The measured calls of the W8A8 product with scales for each token and channel, the scaled
embedding lookup with its gradient, and the clipping of gradients by their global norm.

A case is a dict of plain values; ``kind`` names the call and the rest its sizes:

  linear      the product on a layer's stored codes: quantize the tokens, multiply, scale
  train       a layer's training call on its float masters: y, then dX, dW and db from dY
  lookup      rows of a float table times a scale
  embed_grad  the table's gradient from the rows' gradients
  embed       a lookup and the gradient of its table
  clip        all gradients of a model scaled by min(1, max_norm / (norm + 1e-6))

Widths, stream, chart and vocabulary counts are those of ksdraft_amd/config.py (d 1536 and
1792, 512 and 597 streams, 5888 and 6869 charts, 150144 entries, 4 x 2048 tokens), with odd
sizes between them. The plain forms are written in elementary torch operations in 32 bits.
"""

from __future__ import annotations

import torch

own = False

DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
TINY = 2.0 ** -100  # rows whose largest magnitude is below this count as zero


def listed():
    return [
        # one token through a Rosa projection: the smallest product, all latency
        dict(name="linear_token", kind="linear", M=1, K=1536, N=512, dtype="bf16", bias=True, residual=False),
        # four streams' next tokens through the vocabulary head: one read of the codes
        dict(name="head_tokens", kind="linear", M=4, K=1536, N=150144, dtype="bf16", bias=False, residual=False),
        # a draft batch's projection with the block's residual in its store
        dict(name="linear_batch", kind="linear", M=8192, K=1536, N=1536, dtype="bf16", bias=True, residual=True),
        # a ragged prompt through the output projection of 597 streams
        dict(name="linear_ragged", kind="linear", M=1021, K=597, N=1792, dtype="fp16", bias=True, residual=False),
        # a projection's training call at 4 x 2048 tokens
        dict(name="train_batch", kind="train", M=8192, K=1536, N=1536, dtype="bf16", bias=True),
        # an up projection onto an odd number of charts, an odd number of tokens, all fp32
        dict(name="train_ragged", kind="train", M=2047, K=1792, N=6869, dtype="fp32", bias=True),
        # the vocabulary head's training call: the largest matrices of the step
        dict(name="train_head", kind="train", M=4096, K=1536, N=150144, dtype="bf16", bias=False),
        # a few streams' next tokens
        dict(name="lookup_tokens", kind="lookup", n=4, V=150144, d=1536, dtype="fp32", out="bf16"),
        # the gradient of the whole table from one training batch (4 x 2048 tokens)
        dict(name="embed_grad_batch", kind="embed_grad", n=8192, V=150144, d=1536, dtype="fp32", padding=False),
        # a long ragged packed batch with padding on a smaller half precision table
        dict(name="embed_long", kind="embed", n=65521, V=32003, d=1792, dtype="bf16", padding=True),
        # norms, biases and gates of 24 blocks alone: hundreds of short tensors
        dict(name="clip_vectors", kind="clip", layers=24, d=1536, S=0, charts=0, V=0, dtype="fp32", max_norm=1.0),
        # every gradient of the draft model
        dict(name="clip_model", kind="clip", layers=24, d=1536, S=512, charts=5888, V=150144, dtype="fp32", max_norm=1.0),
    ]


def _log(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi], every third one a multiple of 128."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 1 / 3 and v >= 128:
        v = v // 128 * 128
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["linear", "linear", "train", "train", "lookup", "embed_grad", "embed", "clip"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind in ("linear", "train"):
        K, N = _log(rng, 64, 6869), _log(rng, 64, 150144)
        most = min(8192, 4096 * 1536 * 150144 // (K * N), 4096 * 150144 // N)
        M = _log(rng, 1 if kind == "linear" else 16, max(16, most))
        c = dict(kind=kind, M=M, K=K, N=N, dtype=dtype, bias=rng.random() < 0.5)
        return dict(c, residual=rng.random() < 0.5) if kind == "linear" else c
    if kind == "clip":
        return dict(kind=kind, layers=rng.randint(1, 24), d=_log(rng, 64, 1792), S=rng.choice([0, _log(rng, 16, 597)]),
                    charts=rng.choice([0, _log(rng, 64, 5888)]), V=rng.choice([0, _log(rng, 256, 150144)]),
                    dtype=dtype, max_norm=rng.choice([0.25, 1.0, 1e4]))
    n, V, d = _log(rng, 1, 65536), _log(rng, 256, 150144), _log(rng, 16, 1792)
    if kind == "lookup":
        return dict(kind=kind, n=n, V=V, d=d, dtype=dtype, out=rng.choice([dtype, "bf16"]))
    return dict(kind=kind, n=n, V=V, d=d, dtype=dtype, padding=rng.random() < 0.5)


def _clip_shapes(c):
    """The parameter shapes of a draft model of these sizes (absent parts left out)."""
    d, S, F = c["d"], c["S"], c["charts"]
    block = [(d,)] * 8
    if S:
        block += [(S, d), (S, d), (S, d), (d, S), (S,), (S,), (S,), (S,)]
    if F:
        block += [(F, d), (d, F), (F, 6), (F,), (F,)]
    return ([(c["V"], d)] if c["V"] else []) + block * c["layers"] + [(d,)] * 4


def _codes(w):
    """Per-row int8 codes of w in rows padded with zeros to 16 bytes, and their fp32 scales:
    what a program keeps of a layer's weights."""
    scale = w.abs().amax(1) / 127
    codes = torch.zeros(w.shape[0], -(-w.shape[1] // 16) * 16, dtype=torch.int8, device=w.device)
    codes[:, :w.shape[1]] = torch.round(w / scale[:, None])
    return codes[:, :w.shape[1]], scale


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DT[c["dtype"]]

    def randn(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)

    s = dict(case=c)
    if c["kind"] in ("linear", "train"):
        M, K, N = c["M"], c["K"], c["N"]
        # normalised tokens with a few channels that stand out, as a model's own have
        s["x"] = (randn(M, K) * (1 + 7 * (torch.rand(K, device=DEV, generator=g) < 0.01))).to(dt)
        w = randn(N, K, scale=K ** -0.5)
        s["bias"] = randn(N, scale=0.1) if c["bias"] else None
        if c["kind"] == "linear":
            s["codes"], s["scales"] = _codes(w)
            s["residual"] = randn(M, N, dtype=dt) if c["residual"] else None
        else:
            s["weight"] = w
            # gradients (of a scaled loss) whose size differs from token to token
            s["g"] = (randn(M, N) * 2.0 ** -randn(M, 1).abs()).to(dt)
    elif c["kind"] == "clip":
        s["grads"] = [randn(*shape, scale=1e-2, dtype=dt) for shape in _clip_shapes(c)]
        # the clipped gradients go into one flat buffer, as an optimizer over flat storage keeps it
        s["flat"] = torch.empty(sum(t.numel() for t in s["grads"]), dtype=dt, device=DEV)
        s["out"] = [v.view(t.shape) for v, t in zip(s["flat"].split([t.numel() for t in s["grads"]]), s["grads"])]
    else:
        n, V, d = c["n"], c["V"], c["d"]
        # token frequencies fall with the rank, as a vocabulary's do
        u = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
        s["ids"] = ((V + 1) ** u).long().sub(1).clamp(0, V - 1)
        s["scale"] = float(d) ** 0.5
        if c.get("padding"):
            s["ids"][torch.rand(n, device=DEV, generator=g) < 0.1] = 0
        if c["kind"] != "embed_grad":
            s["weight"] = randn(V, d, scale=0.02, dtype=dt)
        if c["kind"] != "lookup":
            s["g"] = randn(n, d, scale=1e-3, dtype=dt)
    return s


def _rows(x):
    """Codes (as floats) and scales of the rows of an fp32 matrix."""
    a = x.abs().amax(1, keepdim=True)
    some = a >= TINY
    top = torch.full_like(a, 127.0)  # a tensor: by a number torch multiplies with its reciprocal
    inv = torch.where(some, top / torch.where(some, a, 1.0), 0.0)
    return torch.round(x * inv), torch.where(some, a / top, 0.0)


def _plain_linear(x, wq, sw, bias):
    xq, sx = _rows(x.float())
    y = (xq @ wq.t()) * sx * sw
    return y if bias is None else y + bias


def _plain(s):
    c = s["case"]
    dt = DT[c["dtype"]]
    if c["kind"] == "linear":
        y = _plain_linear(s["x"], s["codes"].float(), s["scales"], s["bias"])
        return (y if s["residual"] is None else y + s["residual"].float()).to(dt)
    if c["kind"] == "train":
        wq, sw = _rows(s["weight"])
        xq, sx = _rows(s["x"].float())
        y = (xq @ wq.t()) * sx * sw[:, 0]
        y = (y if s["bias"] is None else y + s["bias"]).to(dt)
        g = s["g"].float()
        gq, e = _rows(g * sw[:, 0])
        dx = ((gq @ wq) * e).to(dt)
        gq, f = _rows((g * sx).t())
        dw = (gq @ xq) * f
        return [y, dx, dw] if s["bias"] is None else [y, dx, dw, g.sum(0)]
    if c["kind"] == "clip":
        norm = torch.stack([t.float().square().sum() for t in s["grads"]]).sum().sqrt()
        coef = torch.clamp(c["max_norm"] / (norm + 1e-6), max=1.0)
        return [norm, torch.cat([(t.float() * coef).to(t.dtype).reshape(-1) for t in s["grads"]])]
    out = []
    if c["kind"] != "embed_grad":
        out.append((s["weight"][s["ids"]].float() * s["scale"]).to(DT[c.get("out", c["dtype"])]))
    if c["kind"] != "lookup":
        dw = torch.zeros(c["V"], c["d"], device=DEV)
        dw.index_add_(0, s["ids"], s["g"].float())
        if c["padding"]:
            dw[0] = 0
        out.append(dw * s["scale"])
    return out


def run(s):
    if not own:
        return _plain(s)
    from ksdraft_amd.kernels.embedding import embedding_gradient, embedding_lookup
    from ksdraft_amd.kernels.token_channel import (token_channel_linear, token_channel_linear_backward,
                                                   token_channel_linear_train)
    from ksdraft_amd.train.clip import clip_gradients
    c = s["case"]
    if c["kind"] == "linear":
        return token_channel_linear(s["x"], s["codes"], s["scales"], bias=s["bias"], residual=s["residual"])
    if c["kind"] == "train":
        y, saved = token_channel_linear_train(s["x"], s["weight"], s["bias"])
        dx, dw, db = token_channel_linear_backward(s["g"], saved)
        return [y, dx, dw] if db is None else [y, dx, dw, db]
    if c["kind"] == "clip":
        norm = clip_gradients(s["grads"], c["max_norm"], out=s["out"])
        return [norm, s["flat"]]
    out = []
    if c["kind"] != "embed_grad":
        out.append(embedding_lookup(s["weight"], s["ids"], s["scale"], out_dtype=DT[c.get("out", c["dtype"])],
                                    check_ids=False))
    if c["kind"] != "lookup":
        out.append(embedding_gradient(s["g"], s["ids"], c["V"], s["scale"],
                                      padding_idx=0 if c["padding"] else None, check_ids=False))
    return out


def work(c):
    e = SIZE[c["dtype"]]
    if c["kind"] in ("linear", "train"):
        M, K, N = c["M"], c["K"], c["N"]
        small = N * 4 if c["bias"] else 0
        if c["kind"] == "linear":
            return dict(bytes=e * (M * K + M * N * (2 if c["residual"] else 1)) + N * K + N * 4 + small,
                        flops=2 * M * N * K)
        # x, W, dY read; y, dX, dW, db written
        return dict(bytes=e * 2 * (M * K + M * N) + 8 * N * K + 2 * small, flops=6 * M * N * K)
    if c["kind"] == "clip":
        n = 0
        for shape in _clip_shapes(c):
            size = 1
            for v in shape:
                size *= v
            n += size
        return dict(bytes=2 * e * n, flops=3 * n)
    n, V, d = c["n"], c["V"], c["d"]
    b = 8 * n
    if c["kind"] != "embed_grad":
        b += n * d * (e + SIZE[c.get("out", c["dtype"])])
    if c["kind"] != "lookup":
        b += n * d * e + V * d * 4
    return dict(bytes=b, flops=n * d)


def _quantized(x):
    """The row quantization of a matrix in 64 bits: codes and scales."""
    top = x.abs().max(dim=1, keepdim=True).values
    zero = top < TINY
    codes = (x / top.masked_fill(zero, 1.0) * 127).round().masked_fill(zero, 0.0)
    return codes, (top / 127).masked_fill(zero, 0.0)


def exact(c, seed):
    s = prepare(c, seed)
    f64 = torch.float64
    if c["kind"] == "linear":
        q, t = _quantized(s["x"].to(f64))
        y = torch.matmul(q, s["codes"].to(f64).t()).mul_(t).mul_(s["scales"].to(f64))
        if s["bias"] is not None:
            y += s["bias"].to(f64)
        if s["residual"] is not None:
            y += s["residual"].to(f64)
        return y
    if c["kind"] == "train":
        wq, ws = _quantized(s["weight"].to(f64))
        xq, xs = _quantized(s["x"].to(f64))
        dy = s["g"].to(f64)
        y = torch.matmul(xq, wq.t()).mul_(xs).mul_(ws.t())
        if s["bias"] is not None:
            y += s["bias"].to(f64)
        q, t = _quantized(dy * ws.t())
        dx = torch.matmul(q, wq).mul_(t)
        q, t = _quantized((dy * xs).t().contiguous())
        dw = torch.matmul(q, xq).mul_(t)
        return [y, dx, dw] if s["bias"] is None else [y, dx, dw, dy.sum(0)]
    if c["kind"] == "clip":
        total = sum(float(t.to(f64).pow(2).sum()) for t in s["grads"]) ** 0.5
        factor = min(1.0, c["max_norm"] / (total + 1e-6))
        return [torch.tensor(total, dtype=f64, device=DEV), torch.cat([t.reshape(-1).to(f64) for t in s["grads"]]) * factor]
    out = []
    if c["kind"] != "embed_grad":
        out.append(torch.index_select(s["weight"], 0, s["ids"]).to(f64) * s["scale"])
    if c["kind"] != "lookup":
        keep = s["ids"] != 0 if c["padding"] else torch.ones_like(s["ids"], dtype=torch.bool)
        # rows in the order of their token, then differences of running sums of equal tokens
        ids, at = torch.sort(s["ids"][keep], stable=True)
        dw = torch.zeros(c["V"], c["d"], dtype=f64, device=DEV)
        if ids.numel():
            run_sum = torch.cumsum(s["g"][keep].to(f64)[at], 0)
            last = torch.cat([ids[1:] != ids[:-1], torch.ones(1, dtype=torch.bool, device=DEV)])
            ends = run_sum[last]
            dw[ids[last]] = torch.cat([ends[:1], ends[1:] - ends[:-1]])
        out.append(dw * s["scale"])
    return out
