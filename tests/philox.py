"""Philox4x32 with 10 rounds (Salmon et al., 2011) on numpy integers, and the dropout mask made of it."""

import numpy as np
import torch

LOW = np.uint64(0xFFFFFFFF)


def philox(counter, key):
    """counter: four arrays of 32-bit words, key: two words -> four arrays."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & LOW, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & LOW]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def halves(rows, d, seed, stream, row0=0):
    """The 16 bits of each value of a (rows, d) matrix whose first row is row0."""
    nb = -(-d // 8)
    row = np.arange(row0, row0 + rows, dtype=np.uint64)[:, None] + np.zeros((1, nb), np.uint64)
    block = np.zeros((rows, 1), np.uint64) + np.arange(nb, dtype=np.uint64)[None]
    w = philox([block, row & LOW, row >> np.uint64(32), np.full_like(row, stream)], [seed % 2 ** 32, seed >> 32])
    u = np.stack([w[0] & np.uint64(0xFFFF), w[0] >> np.uint64(16), w[1] & np.uint64(0xFFFF), w[1] >> np.uint64(16),
                  w[2] & np.uint64(0xFFFF), w[2] >> np.uint64(16), w[3] & np.uint64(0xFFFF), w[3] >> np.uint64(16)], 2)
    return u.reshape(rows, nb * 8)[:, :d]


def mask(rows, d, p, seed, stream=0):
    """Factors of dropout on a (rows, d) matrix, fp32 on the CPU."""
    drop = round(p * 65536)
    scale = np.float32(65536.0 / (65536 - drop)) if drop < 65536 else np.float32(0)
    return torch.from_numpy(np.where(halves(rows, d, seed, stream) >= drop, scale, np.float32(0)))
