"""The measured calls of low-rank adapters beside a shared projection, counter-based dropout and the
verification of drafted tokens.

A case is a dict of plain values; ``kind`` names the call and the rest its sizes:

  adapter   y = base + scale_i (x A_i^T) B_i^T, each token or sequence with an adapter of its own or none
  train     that call with dropout on x, then dX, dA and dB from dY
  dropout   residual + dropout(x), and the gradient's pass under the same mask
  verify    drafted tokens against the target's probabilities, the first refused one drawn anew

Widths, stream, chart and vocabulary counts, block and batch lengths are those of ksdraft_amd/config.py and of
the training step (d 1536 and 1792, 512 and 597 streams, 6869 charts, 150144 entries, blocks of 16, 4 x 2048
tokens), with odd sizes between them. The plain forms are elementary torch operations in 32 bits, in 64
where a running sum is compared with a drawn number.
"""

from __future__ import annotations

import torch

own = False

DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one token through a Rosa projection with its request's adapter: all latency
        dict(name="adapter_token", kind="adapter", B=1, T=1, K=1536, N=512, r=16, n=4, dtype="bf16", per="token"),
        # 64 streams' next tokens, as many adapters: one read of those that are used
        dict(name="adapter_decode", kind="adapter", B=64, T=1, K=1536, N=1536, r=16, n=64, dtype="bf16", per="token"),
        # four prompts, an adapter for each sequence
        dict(name="adapter_prefill", kind="adapter", B=4, T=2048, K=1536, N=1536, r=16, n=4, dtype="bf16", per="sequence"),
        # a packed batch of odd width with adapters of an odd rank, tokens in any order
        dict(name="adapter_ragged", kind="adapter", B=1, T=1021, K=597, N=1792, r=24, n=5, dtype="fp16", per="token"),
        # one adapter trained on the model's fp32 stream with dropout
        dict(name="train_batch", kind="train", B=4, T=2048, K=1536, N=1536, r=16, n=1, dtype="fp32", per="sequence", p=0.1),
        # three adapters of an up projection onto an odd number of charts, an odd number of tokens
        dict(name="train_ragged", kind="train", B=1, T=2047, K=1792, N=6869, r=8, n=3, dtype="bf16", per="token", p=0.05),
        # a verified block's tokens: the launch
        dict(name="dropout_block", kind="dropout", M=17, d=1536, dtype="bf16", residual=False, p=0.1),
        # a training batch's stream with its residual
        dict(name="dropout_batch", kind="dropout", M=8192, d=1536, dtype="bf16", residual=True, p=0.1),
        # one token drawn from a row of logits
        dict(name="verify_sample", kind="verify", B=1, L=0, V=150144, dtype="fp32", draft=False, greedy=0),
        # one stream's block of 16 drafted tokens
        dict(name="verify_block", kind="verify", B=1, L=16, V=150144, dtype="bf16", draft=True, greedy=0),
        # greedy streams on a smaller odd vocabulary
        dict(name="verify_greedy", kind="verify", B=8, L=5, V=32003, dtype="fp16", draft=False, greedy=8),
        # 64 streams' blocks, a quarter of them greedy
        dict(name="verify_batch", kind="verify", B=64, L=16, V=150144, dtype="bf16", draft=True, greedy=16),
    ]


def _log(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi], every third one a multiple of 128."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 1 / 3 and v >= 128:
        v = v // 128 * 128
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["adapter", "adapter", "train", "train", "dropout", "verify", "verify"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind in ("adapter", "train"):
        K, N = _log(rng, 64, 6869), _log(rng, 64, 6869)
        r, n = rng.choice([1, 4, 8, 8, 16, 16, 16, 24, 32, 64]), _log(rng, 1, 64)
        M = _log(rng, 1 if kind == "adapter" else 16, min(8192, 8192 * 2 * 1536 // (K + N) if kind == "train" else 8192))
        n = max(1, min(n, 1024 // r))
        per = rng.choice(["token", "sequence"])
        B = min(M, _log(rng, 1, 64))
        c = dict(kind=kind, B=B, T=max(1, M // B), K=K, N=N, r=r, n=n, dtype=dtype, per=per)
        return dict(c, p=rng.choice([0.0, 0.05, 0.1, 0.5])) if kind == "train" else c
    if kind == "dropout":
        d = _log(rng, 16, 6869)
        return dict(kind=kind, M=_log(rng, 1, max(1, 8192 * 1536 // d)), d=d, dtype=dtype, residual=rng.random() < 0.5,
                    p=rng.choice([0.01, 0.1, 0.25, 0.5]))
    V, L = _log(rng, 1000, 150144), rng.randint(0, 16)
    B = _log(rng, 1, max(1, min(64, 64 * 33 * 150144 * 2 // ((2 * L + 1) * V * SIZE[dtype]))))
    return dict(kind=kind, B=B, L=L, V=V, dtype=dtype, draft=rng.random() < 0.7, greedy=rng.choice([0, 0, B // 2, B]))


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DT[c["dtype"]]

    def randn(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)

    s = dict(case=c, seed=seed * 2654435761 % 2 ** 63)
    if c["kind"] in ("adapter", "train"):
        B, T, K, N, r, n = (c[k] for k in ("B", "T", "K", "N", "r", "n"))
        # normalised tokens with a few channels that stand out, as a model's own have
        s["x"] = (randn(B, T, K) * (1 + 7 * (torch.rand(K, device=DEV, generator=g) < 0.01))).to(dt)
        s["base"] = randn(B, T, N, dtype=dt)
        s["a"] = randn(n, r, K, scale=K ** -0.5, dtype=dt)
        s["b"] = randn(n, N, r, scale=r ** -0.5, dtype=dt)
        s["scales"] = 0.5 + torch.rand(n, device=DEV, generator=g)
        # every ninth request or token on average has no adapter
        shape = (B, T) if c["per"] == "token" else (B,)
        index = torch.randint(0, n, shape, device=DEV, generator=g)
        s["index"] = torch.where(torch.rand(shape, device=DEV, generator=g) < 1 / 9, -1, index)
        if B * T == 1 or n == 1:
            s["index"] = index
        if c["kind"] == "train":
            # gradients (of a scaled loss) whose size differs from token to token
            s["dy"] = (randn(B, T, N) * 2.0 ** -randn(B, T, 1).abs()).to(dt)
            s["dx_base"] = randn(B, T, K, dtype=dt)
    elif c["kind"] == "dropout":
        s["x"], s["dy"] = randn(c["M"], c["d"], dtype=dt), randn(c["M"], c["d"], dtype=dt)
        s["residual"] = randn(c["M"], c["d"], dtype=dt) if c["residual"] else None
    else:
        B, L, V = c["B"], c["L"], c["V"]
        s["target"] = torch.empty(B, L + 1, V, dtype=dt, device=DEV)
        s["draft"] = torch.empty(B, L, V, dtype=dt, device=DEV)
        s["tokens"] = torch.empty(B, L, dtype=torch.int64, device=DEV)
        s["temperatures"] = 0.6 + 0.6 * torch.rand(B, device=DEV, generator=g)
        if c["greedy"]:
            s["temperatures"][:c["greedy"]] = 0.0
        for i in range(B):
            # a language model's rows: a broad bulk and a few likely tokens; the draft's is a noisy copy
            z = randn(L + 1, V, scale=2.0)
            top = torch.randint(0, V, (L + 1, 24), device=DEV, generator=g)
            z.scatter_(1, top, 14 + randn(L + 1, 24, scale=1.5))
            s["target"][i] = z
            s["draft"][i] = z[:L] + randn(L, V, scale=0.5)
            if L:
                t = float(s["temperatures"][i])
                noise = -torch.log(-torch.log(torch.rand(L, V, device=DEV, generator=g).clamp(1e-30, 1 - 1e-7)))
                s["tokens"][i] = (s["draft"][i].float() + (noise * t if t else 0.0)).argmax(1)
        s["uniforms"] = torch.rand(B, L + 1, device=DEV, generator=g)
        s["lengths"] = torch.randint(max(0, L - 2), L + 1, (B,), device=DEV, generator=g)
        if B == 1:
            s["lengths"] = None
        if not c["draft"]:
            s["draft"] = None
    return s


def _mul_hi_lo(a, m):
    """High and low words of 32 x 32 bit products; int64 products wrap, which keeps their 64 bits."""
    p = a * m
    return (p >> 32) & 0xFFFFFFFF, p & 0xFFFFFFFF


def _kept(M, d, p, seed, stream):
    """The mask as factors (0 or 1 / (1 - p)): 16 bits for each value from Philox4x32 of 10 rounds, its
    counter (column / 8, row, 0, stream), its key the seed."""
    row = torch.arange(M, device=DEV)[:, None]
    col = torch.arange(-(-d // 8), device=DEV)[None]
    c0, c1, c2, c3 = (col.expand(M, -1), row.expand(-1, col.shape[1]), torch.zeros_like(row), torch.full_like(row, stream))
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _mul_hi_lo(c0, 0xD2511F53)
        h1, l1 = _mul_hi_lo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c0, c1, c2, c3], 2)
    u = torch.stack([words & 0xFFFF, words >> 16], 3).reshape(M, -1)[:, :d]
    drop = round(p * 65536)
    return (u >= drop).float() * (65536 / (65536 - drop))


def _plain_adapter(s, x, index):
    """(h of every adapter with the others' zeroed (M, n r), y)."""
    c = s["case"]
    M, n, r = x.shape[0], c["n"], c["r"]
    mine = (index[:, None] == torch.arange(n, device=DEV)).float() * s["scales"]
    a = s["a"].float().reshape(n * r, -1)
    h = ((x @ a.t()).view(M, n, r) * mine[:, :, None]).reshape(M, n * r)
    b = s["b"].float().transpose(1, 2).reshape(n * r, -1)
    return h, s["base"].float().reshape(M, -1) + h @ b, a, b, mine


def _plain_verify(s):
    c = s["case"]
    B, L, V = c["B"], c["L"], c["V"]
    temps = s["temperatures"].double()
    greedy = temps == 0
    inv = 1 / torch.where(greedy, 1.0, temps)
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((B,), L, device=DEV)

    def chance(logits, at):
        """The softmax probability of each row's token `at`: 32-bit sums, the token's own power in 64."""
        x = logits.float()
        top = x.amax(2, keepdim=True)
        total = torch.exp((x - top) * inv.float()[:, None, None]).sum(2)
        mine = (x.gather(2, at[:, :, None]) - top)[:, :, 0].double()
        return torch.exp(mine * inv[:, None]) / total.double()

    best = s["target"].argmax(2)
    if L:
        p = chance(s["target"][:, :L], s["tokens"])
        q = chance(s["draft"], s["tokens"]) if s["draft"] is not None else torch.ones_like(p)
        ok = torch.where(greedy[:, None], s["tokens"] == best[:, :L], s["uniforms"][:, :L].double() * q < p)
        ok &= torch.arange(L, device=DEV) < lengths[:, None]
        accepted = ok.long().cumprod(1).sum(1)
    else:
        accepted = torch.zeros(B, dtype=torch.int64, device=DEV)
    rows = torch.arange(B, device=DEV)

    def power(x):
        e = torch.exp((x.double() - x.double().amax(1, keepdim=True)) * inv[:, None])
        return e / e.sum(1, keepdim=True)

    w = power(s["target"][rows, accepted])
    if L:
        last = accepted.clamp(max=L - 1)
        refused = (accepted < lengths)[:, None]
        if s["draft"] is not None:
            less = power(s["draft"][rows, last])
        else:
            less = torch.zeros_like(w).scatter_(1, s["tokens"][rows, last][:, None], 1.0)
        rest = torch.where(refused, (w - less).clamp(min=0), w)
        w = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
    run = w.cumsum(1)
    drawn = (run > s["uniforms"][:, L].double()[:, None] * run[:, -1:]).long().argmax(1)
    drawn = torch.where(greedy, best[rows, accepted], drawn)
    at = torch.arange(L + 1, device=DEV)
    padded = torch.cat([s["tokens"], s["tokens"].new_zeros(B, 1)], 1)
    tokens = torch.where(at < accepted[:, None], padded, torch.where(at == accepted[:, None], drawn[:, None], -1))
    return [tokens, accepted]


def _plain(s):
    c = s["case"]
    if c["kind"] == "verify":
        return _plain_verify(s)
    dt = DT[c["dtype"]]
    if c["kind"] == "dropout":
        keep = _kept(c["M"], c["d"], c["p"], s["seed"], 3)
        y = s["x"].float() * keep
        y = y if s["residual"] is None else y + s["residual"].float()
        return [y.to(dt), (s["dy"].float() * keep).to(dt)]
    B, T, K, N, r, n = (c[k] for k in ("B", "T", "K", "N", "r", "n"))
    index = s["index"].reshape(-1) if c["per"] == "token" else s["index"][:, None].expand(B, T).reshape(-1)
    x = s["x"].float().reshape(B * T, K)
    if c["kind"] == "adapter":
        return _plain_adapter(s, x, index)[1].to(dt).view(B, T, N)
    if c["p"]:
        keep = _kept(B * T, K, c["p"], s["seed"], 3)
        x = x * keep
    h, y, a, b, mine = _plain_adapter(s, x, index)
    dy = s["dy"].float().reshape(B * T, N)
    dh = ((dy @ b.t()).view(B * T, n, r) * mine[:, :, None]).reshape(B * T, n * r)
    dx = dh @ a
    dx = s["dx_base"].float().reshape(B * T, K) + (dx * keep if c["p"] else dx)
    da = (dh.t() @ x).view(n, r, K)
    db = (dy.t() @ h).view(N, n, r).transpose(0, 1).contiguous()
    return [y.to(dt).view(B, T, N), dx.to(dt).view(B, T, K), da, db]


def run(s):
    if not own:
        return _plain(s)
    c = s["case"]
    if c["kind"] in ("adapter", "train"):
        from ksdraft_amd.kernels.adapters import adapter_linear, adapter_linear_backward, adapter_linear_train
        if c["kind"] == "adapter":
            return adapter_linear(s["x"], s["a"], s["b"], s["index"], s["scales"], base=s["base"])
        y, saved = adapter_linear_train(s["x"], s["a"], s["b"], s["index"], s["scales"], base=s["base"],
                                        dropout=c["p"], seed=s["seed"], stream=3)
        dx, da, db = adapter_linear_backward(s["dy"], saved, base=s["dx_base"])
        return [y, dx, da, db]
    if c["kind"] == "dropout":
        from ksdraft_amd.kernels.dropout import dropout
        return [dropout(s["x"], c["p"], s["seed"], stream=3, residual=s["residual"]),
                dropout(s["dy"], c["p"], s["seed"], stream=3)]
    from ksdraft_amd.kernels.speculate import sample_tokens, verify_draft
    if not c["L"]:
        tokens = sample_tokens(s["target"][:, 0], s["uniforms"][:, 0], s["temperatures"])
        return [tokens[:, None], torch.zeros_like(tokens)]
    tokens, accepted = verify_draft(s["target"], s["tokens"], s["uniforms"], draft_logits=s["draft"],
                                    temperatures=s["temperatures"], lengths=s["lengths"])
    return [tokens, accepted]


def work(c):
    e = SIZE[c["dtype"]]
    if c["kind"] in ("adapter", "train"):
        M, K, N, r = c["B"] * c["T"], c["K"], c["N"], c["r"]
        used = min(c["n"], M if c["per"] == "token" else c["B"])
        bank = used * r * (K + N)
        if c["kind"] == "adapter":
            return dict(bytes=e * (M * (K + 2 * N) + bank), flops=2 * M * r * (K + N))
        # x, base, dY, dX's base and the adapters read; y, dX, dA, dB written
        return dict(bytes=e * (M * (3 * K + 3 * N) + bank) + 4 * c["n"] * r * (K + N), flops=6 * M * r * (K + N))
    if c["kind"] == "dropout":
        n = c["M"] * c["d"]
        return dict(bytes=e * n * (5 if c["residual"] else 4), flops=4 * n)
    rows = c["B"] * (c["L"] + 1 + (c["L"] if c["draft"] else 0))
    return dict(bytes=e * rows * c["V"], flops=4 * rows * c["V"])


def _words(block, row, stream, seed):
    """Philox4x32 of 10 rounds on numpy's unsigned 64-bit integers."""
    import numpy as np
    low = np.uint64(0xFFFFFFFF)
    shape = np.broadcast(block, row).shape
    x = [np.broadcast_to(v, shape).astype(np.uint64) for v in (block, row, np.uint64(0), np.uint64(stream))]
    keys = [seed % 2 ** 32, seed // 2 ** 32]
    for i in range(10):
        k = [np.uint64((key + i * step) % 2 ** 32) for key, step in zip(keys, (0x9E3779B9, 0xBB67AE85))]
        left, right = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(right >> np.uint64(32)) ^ x[1] ^ k[0], right & low, (left >> np.uint64(32)) ^ x[3] ^ k[1], left & low]
    return x


def _mask64(M, d, p, seed, stream):
    import numpy as np
    words = _words(np.arange((d + 7) // 8, dtype=np.uint64)[None, :], np.arange(M, dtype=np.uint64)[:, None], stream, seed)
    u = np.empty((M, (d + 7) // 8 * 8), dtype=np.uint32)
    for j in range(8):
        u[:, j::8] = (words[j // 2] >> np.uint64(16 * (j % 2))) & np.uint64(0xFFFF)
    drop = round(p * 65536)
    factor = np.where(u[:, :d] < drop, 0.0, 65536.0 / (65536 - drop))
    return torch.from_numpy(factor).to(DEV)


def _drawn(weights, u):
    """The first place where the running sum passes u times the whole."""
    run = torch.cumsum(weights, 0)
    return int(torch.searchsorted(run, u * float(run[-1]), right=True).clamp(max=weights.numel() - 1))


def exact(c, seed):
    s = prepare(c, seed)
    f64 = torch.float64
    if c["kind"] == "dropout":
        keep = _mask64(c["M"], c["d"], c["p"], s["seed"], 3)
        y = s["x"].to(f64) * keep
        return [y if s["residual"] is None else y + s["residual"].to(f64), s["dy"].to(f64) * keep]
    if c["kind"] in ("adapter", "train"):
        B, T, K, N = (c[k] for k in ("B", "T", "K", "N"))
        x = s["x"].to(f64).view(B * T, K)
        index = s["index"] if c["per"] == "token" else s["index"].repeat_interleave(T)
        index = index.reshape(-1)
        y = s["base"].to(f64).view(B * T, N).clone()
        train = c["kind"] == "train"
        if train:
            keep = _mask64(B * T, K, c["p"], s["seed"], 3) if c["p"] else torch.ones_like(x)
            x = x * keep
            dy = s["dy"].to(f64).view(B * T, N)
            dx = s["dx_base"].to(f64).view(B * T, K).clone()
            da, db = torch.zeros_like(s["a"], dtype=f64), torch.zeros_like(s["b"], dtype=f64)
        for i in range(c["n"]):
            at = (index == i).nonzero()[:, 0]
            a, b = s["a"][i].to(f64), s["b"][i].to(f64)
            h = torch.matmul(x[at], a.t()) * float(s["scales"][i])
            y[at] += torch.matmul(h, b.t())
            if train:
                dh = torch.matmul(dy[at], b) * float(s["scales"][i])
                dx[at] += torch.matmul(dh, a) * keep[at]
                da[i], db[i] = torch.matmul(dh.t(), x[at]), torch.matmul(dy[at].t(), h)
        y = y.view(B, T, N)
        return [y, dx.view(B, T, K), da, db] if train else y
    B, L = c["B"], c["L"]
    tokens = torch.full((B, L + 1), -1, dtype=torch.int64, device=DEV)
    accepted = torch.zeros(B, dtype=torch.int64, device=DEV)
    temps, uniforms, ids = s["temperatures"].tolist(), s["uniforms"].tolist(), s["tokens"].tolist()
    lengths = [L] * B if s["lengths"] is None else s["lengths"].tolist()
    for i in range(B):
        k = 0
        while True:
            x = s["target"][i, k].to(f64)
            if temps[i] == 0:
                new = int(x.argmax())
                if k == lengths[i] or ids[i][k] != new:
                    break
            else:
                p = torch.softmax(x / temps[i], 0)
                if k == lengths[i]:
                    new = _drawn(p, uniforms[i][L])
                    break
                if s["draft"] is None:
                    q = torch.zeros_like(p)
                    q[ids[i][k]] = 1
                else:
                    q = torch.softmax(s["draft"][i, k].to(f64) / temps[i], 0)
                if not uniforms[i][k] * float(q[ids[i][k]]) < float(p[ids[i][k]]):
                    rest = (p - q).clamp(min=0)
                    new = _drawn(rest if float(rest.sum()) > 0 else p, uniforms[i][L])
                    break
            tokens[i, k] = ids[i][k]
            k += 1
        tokens[i, k], accepted[i] = new, k
    return [tokens, accepted]
