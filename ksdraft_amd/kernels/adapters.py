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
from .dropout import _rows, mask_arguments

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_INDEX = (torch.int64, torch.int32)


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _shared(p: torch.Tensor, q: torch.Tensor) -> bool:
    """Whether the spans of memory of two tensors meet."""
    def span(t):
        at = t.data_ptr()
        return at, at + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
    if not p.numel() or not q.numel():
        return False
    (a, b), (c, d) = span(p), span(q)
    return a < d and c < b


def _check(x, a, b, index, scales, base):
    """(M's leading dimensions, K, n, r, N), with the calls that are refused."""
    xs, shape_a, shape_b, at, dtype = x.shape, a.shape, b.shape, index.shape, x.dtype
    if len(xs) < 2:
        raise ValueError(f"x must be (..., K) with one dimension or more of rows, got {tuple(xs)}")
    if dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {dtype}")
    if (len(shape_a) != 3 or len(shape_b) != 3 or shape_a[0] != shape_b[0] or shape_a[1] != shape_b[2]
            or shape_a[2] != xs[-1]):
        raise ValueError(f"a must be (n, r, {xs[-1]}) and b (n, N, r), got {tuple(shape_a)} and {tuple(shape_b)}")
    if a.dtype != dtype or b.dtype != dtype:
        raise TypeError(f"adapters must be of x's {dtype}, got {a.dtype} and {b.dtype}")
    n, r, K = shape_a
    N = shape_b[1]
    if not (n and r and K and N) or r > 128 or n > 65535:
        raise ValueError(f"a bank holds 1 to 65535 adapters of rank 1 to 128, got {tuple(shape_a)} and {tuple(shape_b)}")
    if index.dtype not in _INDEX:
        raise TypeError(f"index must be integers, got {index.dtype}")
    lead = xs[:-1]
    if at != lead and (not at or at != lead[:len(at)]):
        raise ValueError(f"index must be of x's leading dimensions {tuple(lead)}, got {tuple(at)}")
    if scales is not None and (scales.dtype != torch.float32 or scales.shape != (n,)):
        raise ValueError(f"scales must be {n} float32 values, got {tuple(scales.shape)} {scales.dtype}")
    if base is not None and (base.dtype != dtype or base.shape != (*lead, N)):
        raise ValueError(f"base must be {(*lead, N)} {dtype}, got {tuple(base.shape)} {base.dtype}")
    return lead, K, n, r, N


def _forward(x, a, b, index, scales, base, out, mask, train):
    dev = _lib.require_gpu(x, a, b, index, scales, base, out)
    lead, K, n, r, N = _check(x, a, b, index, scales, base)
    x, M, pitch = _rows(x, K)
    a, b, index = _dense(a), _dense(b), _dense(index)
    per = M // (index.numel() or 1) or 1
    if scales is not None:
        scales = _dense(scales)
    base_at, base_pitch = None, 0
    if base is not None:
        base, _, base_pitch = _rows(base, N)
        base_at = base.data_ptr()
    y = out
    if out is None:
        y = torch.empty((*lead, N), dtype=x.dtype, device=dev)
    else:
        if out.shape != (*lead, N) or out.dtype != x.dtype or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {(*lead, N)} {x.dtype} tensor")
        for name, t in (("x", x), ("a", a), ("b", b), ("index", index), ("scales", scales)):
            if t is not None and _shared(out, t):
                raise ValueError(f"out shares memory with {name}")
        if base is not None and _shared(out, base) and (base_at != out.data_ptr() or base_pitch != N):
            raise ValueError("out shares memory with base and is not base itself")
    dt = _lib.dtype_code(x.dtype)
    h = torch.empty((M, r), dtype=torch.float32, device=dev) if train else None
    size = _workspace("ksd_adapter_linear_workspace", M, K, N, r, n, per, dt)
    work = torch.empty(size, dtype=torch.int8, device=dev) if size else None
    if M:
        _lib.call_on(dev, "ksd_adapter_linear", x.data_ptr(), dt, M, K, pitch, a.data_ptr(), b.data_ptr(), n, r, N,
                     index.data_ptr(), index.dtype == torch.int64, per, None if scales is None else scales.data_ptr(), base_at,
                     base_pitch, *mask, y.data_ptr(), None if h is None else h.data_ptr(),
                     None if work is None else work.data_ptr(), size)
    if out is not None:
        _lib.wrote((out,))
    return y, (x, pitch, a, b, index, per, scales, h, work)


@functools.lru_cache(maxsize=4096)
def _workspace(name: str, *sizes: int) -> int:
    need = ctypes.c_int64()
    _lib.call(name, *sizes, ctypes.byref(need))
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
    """What adapter_linear_backward needs of a training forward: its inputs, h (r floats a token) and its
    workspace, where tokens of many adapters are listed by adapter."""

    __slots__ = ("x", "pitch", "a", "b", "index", "per", "scales", "hidden", "work", "lead", "mask", "seed")


def adapter_linear_train(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor,
                         scales: torch.Tensor | None = None, base: torch.Tensor | None = None, dropout: float = 0.0,
                         seed: int | torch.Tensor = 0, stream: int = 0):
    """The training forward: (y, saved), y as adapter_linear gives it on dropout(x) (``kernels.dropout`` with
    this probability, seed and stream; base is not touched by it)."""
    dev = _lib.require_gpu(x)
    mask = mask_arguments(dropout, seed, stream, dev)
    if isinstance(seed, torch.Tensor):
        if mask[0]:
            seed = seed.clone()  # the caller may count it on before the backward pass
            mask = mask_arguments(dropout, seed, stream, dev)
        else:
            seed, mask = 0, _NO_MASK  # nothing is dropped: the seed is not read
    s = Saved()
    s.mask, s.seed, s.lead = mask, seed, x.shape[:-1]
    y, (s.x, s.pitch, s.a, s.b, s.index, s.per, s.scales, s.hidden, s.work) = _forward(x, a, b, index, scales, base, None, mask, True)
    return y, s


def adapter_linear_backward(grad: torch.Tensor, saved: Saved, base: torch.Tensor | None = None, need_dx: bool = True,
                            need_dab: bool = True):
    """(dx (..., K) of x's type, da (n, r, K) fp32, db (n, N, r) fp32) for the upstream gradient of y. base, shaped
    like x, is another branch's gradient of x (the shared projection's), added in the store. What is not needed is
    None; an adapter that no token has gets zeros."""
    dev = _lib.require_gpu(grad, saved.x, base)
    x, a, b = saved.x, saved.a, saved.b
    (n, N, r), K = b.shape, a.shape[2]
    M = saved.hidden.shape[0]
    if grad.shape != (*saved.lead, N) or grad.dtype != x.dtype:
        raise ValueError(f"grad must be {(*saved.lead, N)} {x.dtype}, got {tuple(grad.shape)} {grad.dtype}")
    if base is not None and (base.shape != (*saved.lead, K) or base.dtype != x.dtype):
        raise ValueError(f"base must be {(*saved.lead, K)} {x.dtype}, got {tuple(base.shape)} {base.dtype}")
    if not need_dx and not need_dab:
        return None, None, None
    g, _, pitch = _rows(grad, N)
    base_at, base_pitch = None, 0
    if base is not None and need_dx:
        base, _, base_pitch = _rows(base, K)
        base_at = base.data_ptr()
    dx = torch.empty((*saved.lead, K), dtype=x.dtype, device=dev) if need_dx else None
    da = torch.empty((n, r, K), dtype=torch.float32, device=dev) if need_dab else None
    db = torch.empty((n, N, r), dtype=torch.float32, device=dev) if need_dab else None
    dt = _lib.dtype_code(x.dtype)
    size = _workspace("ksd_adapter_linear_backward_workspace", M, K, N, r, n, saved.per, dt)
    work = torch.empty(size, dtype=torch.int8, device=dev)
    _lib.call_on(dev, "ksd_adapter_linear_backward", g.data_ptr(), dt, M, N, pitch, x.data_ptr(), K, saved.pitch,
                 saved.hidden.data_ptr(), _lib.ptr(saved.work), 0 if saved.work is None else saved.work.numel(), a.data_ptr(),
                 b.data_ptr(), n, r, saved.index.data_ptr(), saved.index.dtype == torch.int64, saved.per,
                 _lib.ptr(saved.scales), base_at, base_pitch, *saved.mask, _lib.ptr(dx) if M else None, _lib.ptr(da),
                 _lib.ptr(db), work.data_ptr(), size)
    return dx, da, db


class _AdapterFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, index, scales, base, p, seed, stream):
        ctx.guard = _lib.capture_guard(_lib.require_gpu(x), x, a, b, base)
        ctx.types = a.dtype, b.dtype
        a, b = (t.to(x.dtype) if t.dtype == torch.float32 else t for t in (a, b))  # masters; their gradients stay fp32
        y, s = adapter_linear_train(x, a, b, index, scales, base, p, seed, stream)
        # through save_for_backward, so that they are freed with the graph and writes into them are noticed
        device_seed = s.seed if isinstance(s.seed, torch.Tensor) else None
        ctx.save_for_backward(x, a, b, s.index, s.scales, s.hidden, s.work, device_seed)
        ctx.args = (s.per, s.lead, (p, None if device_seed is not None else s.seed, stream))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, a, b, index, scales, hidden, work, seed = ctx.saved_tensors
        s = Saved()
        s.per, s.lead, (p, number, stream) = ctx.args
        (s.x, _, s.pitch), s.a, s.b = _rows(x, x.shape[-1]), _dense(a), _dense(b)
        s.index, s.scales, s.hidden, s.work = index, scales, hidden, work
        # what was saved may come back elsewhere (hooks on saved tensors): the address of the seed as it is now
        s.seed = number if seed is None else seed
        s.mask = mask_arguments(p, s.seed, stream, x.device)
        need = ctx.needs_input_grad
        dx = da = db = None
        if need[0] or need[1] or need[2]:
            dx, da, db = adapter_linear_backward(grad, s, None, need[0], need[1] or need[2])
        type_a, type_b = ctx.types
        return (dx, da.to(type_a) if need[1] else None, db.to(type_b) if need[2] else None, None, None,
                grad if need[5] else None, None, None, None)


def adapt(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor, scales: torch.Tensor | None = None,
          base: torch.Tensor | None = None, dropout: float = 0.0, seed: int | torch.Tensor = 0,
          stream: int = 0) -> torch.Tensor:
    """adapter_linear_train's y with gradients for x, a, b and base. a and b may also be fp32 where x is not: they are used
    in x's type, and their gradients are the fp32 sums. A backward pass is captured only while no
    eager graph of the same leaves is alive (RuntimeError, where that graph is of this function)."""
    return _AdapterFunction.apply(x, a, b, index, scales, base, dropout, seed, stream)
