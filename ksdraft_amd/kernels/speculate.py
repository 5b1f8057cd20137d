"""Verification of drafted tokens against a target's logits, and drawing tokens from logits, from given
random numbers.

With p = softmax(target / T) and q = softmax(draft / T), position t's token is accepted while
u[t] q(token) < p(token); the first refused position draws from max(p - q, 0), and where none is refused the
target's last row draws from p. The tokens that come out are then distributed as the target's own. The same
logits and numbers give the same tokens on every call. There is no CPU path, and nothing is read back to the
host.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _logits(t: torch.Tensor, shape, name: str) -> torch.Tensor:
    if t.dim() != 3 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError(f"{name} must be {shape or '(streams, positions, tokens)'}, got {tuple(t.shape)}")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name}: unsupported dtype {t.dtype}")
    return t if t.stride(2) == 1 else t.contiguous()


def _integers(t: torch.Tensor, shape, name: str) -> torch.Tensor:
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be integers, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    return t.to(torch.int64).contiguous()


def _verify(target, tokens, uniforms, draft, temperatures, lengths):
    dev = _lib.require_gpu(target, tokens, uniforms, draft, lengths,
                           temperatures if isinstance(temperatures, torch.Tensor) else None)
    target = _logits(target, None, "target_logits")
    B, rows, V = target.shape
    L = rows - 1
    if L < 0 or V == 0:
        raise ValueError(f"target_logits must hold a row more than drafted tokens, got {tuple(target.shape)}")
    if L:
        tokens = _integers(tokens, (B, L), "draft_tokens")
    if draft is not None:
        draft = _logits(draft, (B, L, V), "draft_logits")
        if draft.dtype != target.dtype:
            raise TypeError(f"draft_logits are {draft.dtype}, target_logits {target.dtype}")
    temps, temp = None, 1.0
    if isinstance(temperatures, torch.Tensor):
        if temperatures.dtype != torch.float32 or tuple(temperatures.shape) != (B,):
            raise ValueError(f"temperatures must be {B} float32 values, got {tuple(temperatures.shape)} {temperatures.dtype}")
        temps = temperatures.contiguous()
    elif temperatures is not None:
        temp = float(temperatures)
        if not temp >= 0:
            raise ValueError(f"temperature must not be negative, got {temp}")
    if uniforms is not None:
        if uniforms.dtype not in (torch.float32, torch.float64):
            raise TypeError(f"uniforms must be float32 or float64, got {uniforms.dtype}")
        if tuple(uniforms.shape) != (B, L + 1):
            raise ValueError(f"uniforms must be {(B, L + 1)}, got {tuple(uniforms.shape)}")
        uniforms = uniforms.contiguous()
    elif temps is not None or temp > 0:
        raise ValueError("only temperature 0 draws without uniforms")
    if lengths is not None:
        lengths = _integers(lengths, (B,), "lengths")
    out = torch.empty((B, L + 1), dtype=torch.int64, device=dev)
    accepted = torch.empty(B, dtype=torch.int64, device=dev)
    if B == 0:
        return out, accepted
    need = ctypes.c_int64()
    _lib.call("ksd_verify_draft_workspace", B, L, V, int(draft is not None), ctypes.byref(need))
    work = torch.empty(need.value, dtype=torch.int8, device=dev)
    db, dt = (0, 0) if draft is None else (draft.stride(0), draft.stride(1))
    _lib.call_on(dev, "ksd_verify_draft", target.data_ptr(), _lib.ptr(draft), _lib.dtype_code(target.dtype), B, L, V,
                 target.stride(0), target.stride(1), db, dt, tokens.data_ptr() if L else None, _lib.ptr(uniforms),
                 int(uniforms is not None and uniforms.dtype == torch.float64), _lib.ptr(temps), temp, _lib.ptr(lengths),
                 out.data_ptr(), accepted.data_ptr(), work.data_ptr(), need.value)
    return out, accepted


def verify_draft(target_logits: torch.Tensor, draft_tokens: torch.Tensor, uniforms: torch.Tensor | None,
                 draft_logits: torch.Tensor | None = None, temperatures: torch.Tensor | float | None = None,
                 lengths: torch.Tensor | None = None):
    """(tokens (B, L + 1), accepted (B,)), int64: per stream the accepted drafted tokens, one token drawn by the
    target, then -1; and how many were accepted.

    target_logits (B, L + 1, V) float: row t is the target's at drafted token t, the last the one behind them.
    draft_tokens (B, L) integers, drawn from softmax(draft_logits / T); draft_logits (B, L, V) of the target's
    type, or None for tokens chosen without chance (q = 1). uniforms (B, L + 1) float32 or float64 in [0, 1): one for
    each test, the last for the draw. temperatures: (B,) float32, a number, or None (1); 0 verifies greedily against
    the largest logit (the lowest index of equal ones), and then needs no uniforms where it is a number. lengths
    (B,): drafted tokens of each stream (None: L); stream b's row lengths[b] is then the one behind the last.

    Logits of -inf have probability 0. A drafted token outside the vocabulary is refused. A target row
    without a finite logit, or with NaN or +inf, refuses its token and draws -1."""
    if draft_tokens is None:
        raise ValueError("draft_tokens are needed; sample_tokens draws without a draft")
    return _verify(target_logits, draft_tokens, uniforms, draft_logits, temperatures, lengths)


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor | None = None,
                  temperatures: torch.Tensor | float | None = None) -> torch.Tensor:
    """A token for each row of logits (..., V): the first whose running sum of softmax(logits / T) passes its
    number of uniforms (...), or the largest logit at T = 0 (uniforms may then be None for a T given as a
    number); -1 for a row without a distribution. temperatures: (...) float32, a number or None (1). int64 (...)."""
    if logits.dim() == 0:
        raise ValueError("logits must have a last dimension of tokens")
    lead = logits.shape[:-1]

    def flat(t, name):
        if t is not None and isinstance(t, torch.Tensor) and t.shape != lead:
            raise ValueError(f"{name} must be {tuple(lead)}, got {tuple(t.shape)}")
        return t
    uniforms = flat(uniforms, "uniforms")
    temperatures = flat(temperatures, "temperatures")
    if isinstance(temperatures, torch.Tensor):
        temperatures = temperatures.reshape(-1)
    rows = logits.reshape(-1, 1, logits.shape[-1]) if logits.shape[-1] else logits.new_empty((0, 1, 0))
    out, _ = _verify(rows, None, None if uniforms is None else uniforms.reshape(-1, 1), None, temperatures, None)
    return out.reshape(lead)
