"""Dropout from a counter-based generator, its mask stored nowhere.

    y = residual + x * keep / (1 - p),   keep = (16 random bits of the value) >= round(65536 p)

The bits are Philox4x32's (10 rounds) at a counter made of the value's row and column, under the key
``seed``: the backward pass is the same call on the gradient, and any kernel that reads x can make the mask
again (``kernels.adapters`` does). Masks depend on the shape (rows, last dimension), seed and stream only,
not on the type, the strides or the device. There is no CPU path.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _lib

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def mask_arguments(p: float, seed, stream: int, dev: torch.device):
    """(65536 p, seed, address of a device seed or None, stream) as the C ABI takes a mask."""
    if not 0 <= p <= 1:
        raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
    if not 0 <= stream < 1 << 32:
        raise ValueError(f"stream must lie in [0, 2**32), got {stream}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != dev:
            raise ValueError(f"a seed on the device is one int64 on {dev}, got {tuple(seed.shape)} {seed.dtype} on {seed.device}")
        return round(p * 65536), 0, seed.data_ptr(), stream
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"seed must lie in [0, 2**64), got {seed}")
    return round(p * 65536), seed, None, stream


def _rows(t: torch.Tensor, d: int):
    """(t or a copy, its rows, their pitch) of a tensor (..., d) as the kernels read it (``kernels.adapters``' too)."""
    if t.is_contiguous():
        return t, t.numel() // d, d
    t = t if t.dim() == 2 else t.reshape(-1, d)
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t, t.shape[0], t.stride(0) if t.shape[0] > 1 else d


def _dropout(x, p, seed, stream, residual):
    dev = _lib.require_gpu(x, residual)
    if x.dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {x.dtype}")
    if x.dim() == 0:
        raise ValueError("dropout takes tensors of one dimension or more")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must be {tuple(x.shape)} {x.dtype}, got {tuple(residual.shape)} {residual.dtype}")
    mask = mask_arguments(p, seed, stream, dev)
    out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    d = x.shape[-1]
    if out.numel() == 0:
        return out
    x, rows, pitch = _rows(x, d)
    at, residual_pitch = None, 0
    if residual is not None:
        residual, _, residual_pitch = _rows(residual, d)
        at = residual.data_ptr()
    _lib.call_on(dev, "ksd_dropout", x.data_ptr(), _lib.dtype_code(x.dtype), rows, d, pitch, *mask, at, residual_pitch,
                 out.data_ptr())
    return out


class _DropoutFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, stream, residual):
        ctx.guard = _lib.capture_guard(_lib.require_gpu(x), x, residual)
        if isinstance(seed, torch.Tensor):  # the caller may count it on before the backward pass
            seed = seed.clone()
            ctx.save_for_backward(seed)
            ctx.save_for_forward(seed)
            ctx.args = (p, None, stream)
        else:
            ctx.args = (p, seed, stream)
        return _dropout(x, p, seed, stream, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        p, seed, stream = ctx.args
        seed = ctx.saved_tensors[0] if seed is None else seed
        need = ctx.needs_input_grad
        return _dropout(grad, p, seed, stream, None) if need[0] else None, None, None, None, grad if need[4] else None

    @staticmethod
    def jvp(ctx, x, _p, _seed, _stream, residual):
        if x is None:
            return residual.clone()
        p, seed, stream = ctx.args
        return dropout(x, p, ctx.saved_tensors[0] if seed is None else seed, stream, residual)


def _differentiated(*tensors) -> bool:
    """Whether a derivative of a tensor is asked for, backwards or forwards."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return forward_ad._current_level >= 0 and any(  # below 0 no tensor has a tangent
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def dropout(x: torch.Tensor, p: float, seed: int | torch.Tensor, stream: int = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """residual + dropout(x): x (..., d) float, each value dropped with probability p (met to 2**-17), the
    others times 1 / (1 - p), in fp32, rounded once to x's dtype; a dropped value counts as 0 whatever it
    held. residual has x's shape and dtype.

    seed (64 bits) and stream (32 bits, a layer's number for instance) name the mask: the same ones on the
    same shape give the same mask. A seed on the device (one int64) is read by the kernel, so a graph replayed
    after a change of it drops other values. The gradient, and a forward-mode tangent, go through the same mask."""
    if _differentiated(x, residual):
        return _DropoutFunction.apply(x, p, seed, stream, residual)
    return _dropout(x, p, seed, stream, residual)


class Dropout(nn.Module):
    """nn.Dropout on ``dropout``: the n-th training call of a module takes stream n of its seed (drawn from
    torch's CPU generator unless given), so a run is repeated by its seeds. Under graph capture the captured
    stream is part of the graph: a captured step passes a device seed to ``dropout`` itself. A forward pass that is run
    again for its backward (recomputed activations) would take the next stream's mask, and raises RuntimeError, unless the
    stream is named (``name_streams``). ``calls`` counts the streams and may be set, to go on where a run ended."""

    stream = None  # the named one

    def __init__(self, p: float = 0.1, seed: int | None = None):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
        self.p = p
        self.seed = int(torch.randint(0, 1 << 62, ())) if seed is None else seed
        self.calls = 0

    def extra_repr(self) -> str:
        return f"p={self.p}"

    def next_stream(self) -> int:
        if self.stream is not None:
            return self.stream
        if torch._C._current_graph_task_id() != -1:  # inside a backward pass
            raise RuntimeError("a forward pass that is run again for its backward takes a named stream (name_streams)")
        n, self.calls = self.calls, (self.calls + 1) % (1 << 32)
        return n

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        if not self.training or self.p == 0:
            return x if residual is None else residual + x
        return dropout(x, self.p, self.seed, self.next_stream(), residual)


def name_streams(module: nn.Module, stream: int | None) -> None:
    """Every training call of module's ``Dropout`` layers (and those of its adapted layers) takes this stream of the layer's
    seed, until another is named: a step's number for the step whose activations are recomputed. Layers have seeds of their
    own, so one number names different masks; a layer called twice in a step drops the same places. None: streams are
    counted again."""
    if stream is not None and not 0 <= stream < 1 << 32:
        raise ValueError(f"stream must lie in [0, 2**32), got {stream}")
    for m in module.modules():
        if isinstance(m, Dropout):
            m.stream = stream
