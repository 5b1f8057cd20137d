"""Low-rank adapters of many requests beside a shared projection.

    h[m] = s_i x~[m] A_i^T,   y[m] = base[m] + h[m] B_i^T,   i = index[m],   x~ = dropout(x) in training

One base projection serves all requests (whatever layer gave ``base``); each token, sequence or request
names its adapter, or none. A bank holds n adapters: a (n, r, K) and b (n, N, r). The backward pass gives

    g[m] = s_i dY[m] B_i,   dX[m] = mask(g[m] A_i),   dA_i = sum g[m]^T x~[m],   dB_i = sum dY[m]^T h[m]

Sums are fp32 and run in an order that sizes and indices fix: repeated calls give the same bits. There is no
CPU path.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .dropout import mask_arguments

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    t = t if t.dim() == 2 else t.reshape(-1, width)
    return t if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= width) else t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _shared(p: torch.Tensor, q: torch.Tensor) -> bool:
    """Whether the spans of memory of two tensors meet."""
    def span(t):
        at = t.data_ptr()
        return at, at + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
    if not p.numel() or not q.numel():
        return False
    (a, b), (c, d) = span(p), span(q)
    return a < d and c < b


def _bank(x, a, b, index, scales, base):
    """Checks a call: (x as rows, a, b, index, rows of one index, scales, base as rows)."""
    if x.dim() < 2:
        raise ValueError(f"x must be (..., K) with one dimension or more of rows, got {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {x.dtype}")
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or a.shape[2] != x.shape[-1]:
        raise ValueError(f"a must be (n, r, {x.shape[-1]}) and b (n, N, r), got {tuple(a.shape)} and {tuple(b.shape)}")
    if a.dtype != x.dtype or b.dtype != x.dtype:
        raise TypeError(f"adapters must be of x's {x.dtype}, got {a.dtype} and {b.dtype}")
    n, r, K = a.shape
    N = b.shape[1]
    if not (n and r and K and N) or r > 128 or n > 65535:
        raise ValueError(f"a bank holds 1 to 65535 adapters of rank 1 to 128, got {tuple(a.shape)} and {tuple(b.shape)}")
    if index.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"index must be integers, got {index.dtype}")
    if index.dim() == 0 or index.dim() >= x.dim() or index.shape != x.shape[:index.dim()]:
        raise ValueError(f"index must be of x's leading dimensions {tuple(x.shape[:-1])}, got {tuple(index.shape)}")
    if scales is not None and (scales.dtype != torch.float32 or tuple(scales.shape) != (n,)):
        raise ValueError(f"scales must be {n} float32 values, got {tuple(scales.shape)} {scales.dtype}")
    if base is not None and (base.shape != (*x.shape[:-1], N) or base.dtype != x.dtype):
        raise ValueError(f"base must be {(*x.shape[:-1], N)} {x.dtype}, got {tuple(base.shape)} {base.dtype}")
    x2 = _rows(x, K)
    per = x2.shape[0] // max(1, index.numel())
    return (x2, a.contiguous(), b.contiguous(), index.contiguous(), max(1, per),
            None if scales is None else scales.contiguous(), None if base is None else _rows(base, N))


def _forward(x, a, b, index, scales, base, out, mask, train):
    dev = _lib.require_gpu(x, a, b, index, scales, base, out)
    x2, a, b, index, per, scales, base2 = _bank(x, a, b, index, scales, base)
    (M, K), (n, N, r) = x2.shape, b.shape
    y = out
    if out is None:
        y = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=dev)
    else:
        if out.shape != (*x.shape[:-1], N) or out.dtype != x.dtype or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {(*x.shape[:-1], N)} {x.dtype} tensor")
        for name, t in (("x", x2), ("a", a), ("b", b), ("index", index)):
            if _shared(out, t):
                raise ValueError(f"out shares memory with {name}")
        if base2 is not None and _shared(out, base2) and (base2.data_ptr() != out.data_ptr() or _pitch(base2) != N):
            raise ValueError("out shares memory with base and is not base itself")
    h = torch.empty((M, r), dtype=torch.float32, device=dev) if train else None
    groups, size = None, _groups_bytes(M, K, N, r, n, per, _lib.dtype_code(x.dtype), train)
    if size:
        groups = torch.empty(size, dtype=torch.int8, device=dev)
    if M or train:
        _lib.call_on(dev, "ksd_adapter_linear", x2.data_ptr(), _lib.dtype_code(x.dtype), M, K, _pitch(x2), a.data_ptr(),
                     b.data_ptr(), n, r, N, index.data_ptr(), int(index.dtype == torch.int64), per, _lib.ptr(scales),
                     _lib.ptr(base2), 0 if base2 is None else _pitch(base2), *mask, y.data_ptr(), _lib.ptr(h),
                     _lib.ptr(groups), size)
    if out is not None:
        _lib.wrote((out,))
    return y, (x2, a, b, index, per, scales, h, groups)


@functools.lru_cache(maxsize=4096)
def _groups_bytes(M: int, K: int, N: int, r: int, n: int, per: int, dtype: int, train: bool) -> int:
    need = ctypes.c_int64()
    _lib.call("ksd_adapter_linear_groups", M, K, N, r, n, per, dtype, int(train), ctypes.byref(need))
    return need.value


_NO_MASK = (0, 0, None, 0)


def adapter_linear(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor,
                   scales: torch.Tensor | None = None, base: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """base + s_i (x A_i^T) B_i^T: x (..., K), a (n, r, K) and b (n, N, r) of one float type -> (..., N) of it.

    index (int32 or int64) has x's leading dimensions, or the first of them: index (B,) for x (B, T, K) gives each
    sequence its adapter. An index outside [0, n) (-1, say) takes none: such rows are base (0 without one).
    scales (n,) float32, None: 1. out, contiguous, may be base itself. Sums are fp32, rounded once."""
    return _forward(x, a, b, index, scales, base, out, _NO_MASK, False)[0]


class Saved:
    """What adapter_linear_backward needs of a training forward: its inputs, h (r floats a token) and the tokens
    listed by adapter."""

    __slots__ = ("x", "a", "b", "index", "per", "scales", "hidden", "groups", "lead", "mask", "seed")


def adapter_linear_train(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor,
                         scales: torch.Tensor | None = None, base: torch.Tensor | None = None, dropout: float = 0.0,
                         seed: int | torch.Tensor = 0, stream: int = 0):
    """The training forward: (y, saved), y as adapter_linear gives it on dropout(x) (``kernels.dropout`` with
    this probability, seed and stream; base is not touched by it)."""
    dev = _lib.require_gpu(x)
    if isinstance(seed, torch.Tensor) and dropout:
        seed = seed.clone()  # the caller may count it on before the backward pass
    mask = mask_arguments(dropout, seed, stream, dev)
    s = Saved()
    s.mask, s.seed, s.lead = mask, seed, x.shape[:-1]
    y, (s.x, s.a, s.b, s.index, s.per, s.scales, s.hidden, s.groups) = _forward(x, a, b, index, scales, base, None, mask, True)
    return y, s


def adapter_linear_backward(grad: torch.Tensor, saved: Saved, base: torch.Tensor | None = None, need_dx: bool = True,
                            need_dab: bool = True):
    """(dx (..., K) of x's type, da (n, r, K) fp32, db (n, N, r) fp32) for the upstream gradient of y. base, shaped
    like x, is another branch's gradient of x (the shared projection's), added in the store. What is not needed is
    None; an adapter that no token has gets zeros."""
    dev = _lib.require_gpu(grad, saved.x, base)
    x, a, b = saved.x, saved.a, saved.b
    (M, K), (n, N, r) = x.shape, b.shape
    if grad.shape != (*saved.lead, N) or grad.dtype != x.dtype:
        raise ValueError(f"grad must be {(*saved.lead, N)} {x.dtype}, got {tuple(grad.shape)} {grad.dtype}")
    if base is not None and (base.shape != (*saved.lead, K) or base.dtype != x.dtype):
        raise ValueError(f"base must be {(*saved.lead, K)} {x.dtype}, got {tuple(base.shape)} {base.dtype}")
    if not need_dx and not need_dab:
        return None, None, None
    g = _rows(grad, N)
    base = None if base is None or not need_dx else _rows(base, K)
    dx = torch.empty((*saved.lead, K), dtype=x.dtype, device=dev) if need_dx else None
    da = torch.empty((n, r, K), dtype=torch.float32, device=dev) if need_dab else None
    db = torch.empty((n, N, r), dtype=torch.float32, device=dev) if need_dab else None
    need = ctypes.c_int64()
    dt = _lib.dtype_code(x.dtype)
    _lib.call("ksd_adapter_linear_backward_workspace", M, K, N, r, n, dt, ctypes.byref(need))
    work = torch.empty(need.value, dtype=torch.int8, device=dev)
    _lib.call_on(dev, "ksd_adapter_linear_backward", g.data_ptr(), dt, M, N, _pitch(g), x.data_ptr(), K, _pitch(x),
                 saved.hidden.data_ptr(), saved.groups.data_ptr(), saved.groups.numel(), a.data_ptr(), b.data_ptr(), n, r, saved.index.data_ptr(),
                 int(saved.index.dtype == torch.int64), saved.per, _lib.ptr(saved.scales), _lib.ptr(base),
                 0 if base is None else _pitch(base), *saved.mask, _lib.ptr(dx) if M else None, _lib.ptr(da), _lib.ptr(db),
                 work.data_ptr(), need.value)
    return dx, da, db


class _AdapterFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, index, scales, base, p, seed, stream):
        ctx.guard = _lib.capture_guard(_lib.require_gpu(x), x, a, b, base)
        y, s = adapter_linear_train(x, a, b, index, scales, base, p, seed, stream)
        # through save_for_backward, so that they are freed with the graph and writes into them are noticed
        device_seed = s.seed if isinstance(s.seed, torch.Tensor) else None
        ctx.save_for_backward(x, a, b, s.index, s.scales, s.hidden, s.groups, device_seed)
        ctx.args = (s.per, s.lead, s.mask)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, a, b, index, scales, hidden, groups, seed = ctx.saved_tensors
        s = Saved()
        s.per, s.lead, s.mask = ctx.args
        s.x, s.a, s.b = _rows(x, x.shape[-1]), a.contiguous(), b.contiguous()
        s.index, s.scales, s.hidden, s.groups, s.seed = index, scales, hidden, groups, seed
        need = ctx.needs_input_grad
        dx = da = db = None
        if need[0] or need[1] or need[2]:
            dx, da, db = adapter_linear_backward(grad, s, None, need[0], need[1] or need[2])
        return (dx, da.to(a.dtype) if need[1] else None, db.to(b.dtype) if need[2] else None, None, None,
                grad if need[5] else None, None, None, None)


def adapt(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor, scales: torch.Tensor | None = None,
          base: torch.Tensor | None = None, dropout: float = 0.0, seed: int | torch.Tensor = 0,
          stream: int = 0) -> torch.Tensor:
    """adapter_linear_train's y with gradients for x, a, b and base. A backward pass is captured only while no
    eager graph of the same leaves is alive (RuntimeError, where that graph is of this function)."""
    return _AdapterFunction.apply(x, a, b, index, scales, base, dropout, seed, stream)
