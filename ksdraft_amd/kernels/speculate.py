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
import functools

import torch

from .. import _lib

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _integers(t: torch.Tensor, shape, name: str) -> torch.Tensor:
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be integers, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    return t if t.dtype == torch.int64 and t.is_contiguous() else t.to(torch.int64).contiguous()


def _numbers(uniforms, temperatures, shape, lead):
    """(uniforms, whether they are fp64, temperatures on the device or None, else one for all)."""
    temps, temp = None, 1.0
    if isinstance(temperatures, torch.Tensor):
        if temperatures.dtype != torch.float32 or temperatures.shape != lead:
            raise ValueError(f"temperatures must be {tuple(lead)} float32 values, got {tuple(temperatures.shape)} {temperatures.dtype}")
        temps = temperatures if temperatures.is_contiguous() else temperatures.contiguous()
    elif temperatures is not None:
        temp = float(temperatures)
        if not temp >= 0:
            raise ValueError(f"temperature must not be negative, got {temp}")
    wide = False
    if uniforms is not None:
        if uniforms.dtype not in (torch.float32, torch.float64):
            raise TypeError(f"uniforms must be float32 or float64, got {uniforms.dtype}")
        if uniforms.shape != shape:
            raise ValueError(f"uniforms must be {tuple(shape)}, got {tuple(uniforms.shape)}")
        wide = uniforms.dtype == torch.float64
        uniforms = uniforms if uniforms.is_contiguous() else uniforms.contiguous()
    elif temps is not None or temp > 0:
        raise ValueError("only temperature 0 draws without uniforms")
    return uniforms, wide, temps, temp


@functools.lru_cache(maxsize=4096)
def _workspace(B: int, L: int, V: int, draft: bool) -> int:
    need = ctypes.c_int64()
    _lib.call("ksd_verify_draft_workspace", B, L, V, draft, ctypes.byref(need))
    return need.value


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
    without a finite logit, or with NaN or +inf, refuses its token and draws -1 (greedily +inf is a largest logit like any
    other). A draft row with NaN or +inf refuses its token, and the draw is from p; one of nothing but -inf is q = 0."""
    if draft_tokens is None:
        raise ValueError("draft_tokens are needed; sample_tokens draws without a draft")
    dev = _lib.require_gpu(target_logits, draft_tokens, uniforms, draft_logits, lengths,
                           temperatures if isinstance(temperatures, torch.Tensor) else None)
    target, draft, dtype = target_logits, draft_logits, target_logits.dtype
    if target.dim() != 3 or target.shape[1] == 0 or target.shape[2] == 0:
        raise ValueError(f"target_logits must be (streams, a row more than drafted tokens, tokens), got {tuple(target.shape)}")
    if dtype not in _TYPES:
        raise TypeError(f"target_logits: unsupported dtype {dtype}")
    B, rows, V = target.shape
    L = rows - 1
    target = target if target.stride(2) == 1 else target.contiguous()
    tokens = _integers(draft_tokens, (B, L), "draft_tokens")
    db = dt = 0
    if draft is not None:
        if draft.shape != (B, L, V):
            raise ValueError(f"draft_logits must be {(B, L, V)}, got {tuple(draft.shape)}")
        if draft.dtype != dtype:
            raise TypeError(f"draft_logits are {draft.dtype}, target_logits {dtype}")
        draft = draft if draft.stride(2) == 1 else draft.contiguous()
        db, dt, _ = draft.stride()
    uniforms, wide, temps, temp = _numbers(uniforms, temperatures, (B, rows), (B,))
    if lengths is not None:
        lengths = _integers(lengths, (B,), "lengths")
    out = torch.empty((B, rows), dtype=torch.int64, device=dev)
    accepted = torch.empty(B, dtype=torch.int64, device=dev)
    if B:
        size = _workspace(B, L, V, draft is not None)
        work = torch.empty(size, dtype=torch.int8, device=dev)
        tb, tt, _ = target.stride()
        _lib.call_on(dev, "ksd_verify_draft", target.data_ptr(), _lib.ptr(draft), _lib.dtype_code(dtype), B, L, V, tb, tt, db, dt,
                     tokens.data_ptr(), _lib.ptr(uniforms), wide, _lib.ptr(temps), temp, _lib.ptr(lengths), out.data_ptr(),
                     accepted.data_ptr(), work.data_ptr(), size)
    return out, accepted


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor | None = None,
                  temperatures: torch.Tensor | float | None = None) -> torch.Tensor:
    """A token for each row of logits (..., V): the first whose running sum of softmax(logits / T) passes its
    number of uniforms (...), or the largest logit at T = 0 (uniforms may then be None for a T given as a
    number); -1 for a row without a distribution. temperatures: (...) float32, a number or None (1). int64 (...)."""
    dev = _lib.require_gpu(logits, uniforms, temperatures if isinstance(temperatures, torch.Tensor) else None)
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"logits must have a last dimension of tokens, got {tuple(logits.shape)}")
    if logits.dtype not in _TYPES:
        raise TypeError(f"logits: unsupported dtype {logits.dtype}")
    lead, V = logits.shape[:-1], logits.shape[-1]
    uniforms, wide, temps, temp = _numbers(uniforms, temperatures, lead, lead)
    rows = logits if logits.dim() == 2 else logits.reshape(-1, V)
    rows = rows if rows.stride(1) == 1 else rows.contiguous()
    B = rows.shape[0]
    out = torch.empty(lead, dtype=torch.int64, device=dev)
    if B:
        size = _workspace(B, 0, V, False)
        work = torch.empty(size, dtype=torch.int8, device=dev)
        _lib.call_on(dev, "ksd_verify_draft", rows.data_ptr(), None, _lib.dtype_code(rows.dtype), B, 0, V, rows.stride(0), 0, 0, 0,
                     None, _lib.ptr(uniforms), wide, _lib.ptr(temps), temp, None, out.data_ptr(), None, work.data_ptr(), size)
    return out
