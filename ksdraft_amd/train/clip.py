"""The global norm of a model's gradients and their clipping (torch.nn.utils.clip_grad_norm_,
reference ksdraft/train/__init__.py:165) over any number of tensors in a few launches.

    norm   = sqrt(sum of all g^2) / loss_scale          (norm_type inf: max |g| / loss_scale)
    factor = min(1, max_norm / (norm + 1e-6)) / loss_scale,   g' = g * factor

Squares are summed in fp64 in a fixed order: no overflow for any fp32 gradient, and the same bits
on every call. Nothing is read back to the host.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from .. import _lib

# KsdClipTensor of the C ABI
_TENSOR = np.dtype([("grad", "<u8"), ("out", "<u8"), ("n", "<i8"), ("dtype", "<i4"), ("reserved", "<i4")])
_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _check(grads, out, norm_type, loss_scale):
    if norm_type not in (2, math.inf):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    if not loss_scale > 0:
        raise ValueError(f"loss_scale must be positive, got {loss_scale}")
    if out is not None and len(out) != len(grads):
        raise ValueError(f"{len(grads)} gradients, {len(out)} outputs")


def _table(grads, out):
    """The tensors' descriptors (a host array) and their device."""
    dev = _lib.require_gpu(*grads, *(out or ()))
    rows = []
    for i, g in enumerate(grads):
        if g.is_sparse or not g.is_contiguous():
            raise ValueError(f"gradient {i} is not dense and contiguous")
        code = _CODE.get(g.dtype)
        if code is None:
            raise TypeError(f"gradient {i}: unsupported dtype {g.dtype}")
        p = g.data_ptr()
        if out is None:
            rows.append((p, p, g.numel(), code, 0))
            continue
        o = out[i]
        if o.shape != g.shape or o.dtype != g.dtype or not o.is_contiguous():
            raise ValueError(f"output {i} must be contiguous {tuple(g.shape)} {g.dtype}")
        rows.append((p, o.data_ptr(), g.numel(), code, 0))
    return np.array(rows, dtype=_TENSOR), dev


def _norm(table, dev, norm_type, max_norm, loss_scale):
    need = ctypes.c_int64()
    _lib.call("ksd_grad_norm_workspace", table.ctypes.data, len(table), ctypes.byref(need))
    work = torch.empty(need.value, dtype=torch.int8, device=dev)
    res = torch.empty(2, dtype=torch.float32, device=dev)
    _lib.call("ksd_grad_norm", table.ctypes.data, len(table), int(norm_type == math.inf), max_norm, loss_scale,
              res.data_ptr(), res.data_ptr() + 4, work.data_ptr(), need.value, _lib.stream_ptr(dev))
    return res


def gradient_norm(grads, max_norm: float = math.inf, norm_type: float = 2.0, loss_scale: float = 1.0):
    """(norm, factor) as 0-d and 1-element device tensors; factor is what AdamWRequant.step takes as
    ``clip_coef`` to clip the gradients as it loads them. grads: tensors on one GPU."""
    grads = list(grads)
    _check(grads, None, norm_type, loss_scale)
    if not grads:
        raise ValueError("no gradients")
    table, dev = _table(grads, None)
    res = _norm(table, dev, norm_type, max_norm, loss_scale)
    return res[0], res[1:]


def clip_gradients(grads, max_norm: float, norm_type: float = 2.0, out=None, loss_scale: float = 1.0) -> torch.Tensor:
    """Multiplies every gradient by the factor above, in place or into ``out`` (tensors of the same
    shapes and dtypes), and returns the norm (0-d, on the device)."""
    grads = list(grads)
    out = None if out is None else list(out)
    _check(grads, out, norm_type, loss_scale)
    if not grads:
        raise ValueError("no gradients")
    table, dev = _table(grads, out)
    res = _norm(table, dev, norm_type, max_norm, loss_scale)
    _lib.call("ksd_grad_scale", table.ctypes.data, len(table), res.data_ptr() + 4, _lib.stream_ptr(dev))
    return res[0]


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, loss_scale: float = 1.0) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ on the parameters' gradients, in place."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    return clip_gradients(grads, max_norm, norm_type, loss_scale=loss_scale)
