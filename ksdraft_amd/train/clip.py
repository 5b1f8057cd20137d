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
from array import array
from operator import attrgetter

import torch

from .. import _lib

_T = torch.Tensor
_dtype_of = attrgetter("dtype")
_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _check(grads, out, norm_type, loss_scale):
    if norm_type not in (2, math.inf):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    if not loss_scale > 0:
        raise ValueError(f"loss_scale must be positive, got {loss_scale}")
    if out is not None and len(out) != len(grads):
        raise ValueError(f"{len(grads)} gradients, {len(out)} outputs")


class _Table:
    """The tensors as the C ABI takes them: host arrays of addresses, sizes and types. Built by a few
    passes in C over the list (a model has hundreds of gradients, and the call's own cost is this)."""

    def __init__(self, grads, out):
        devices = set(map(_T.get_device, grads))
        if out is not None:
            devices |= set(map(_T.get_device, out))
        if len(devices) > 1 or -1 in devices:
            _lib.require_gpu(*grads, *(out or ()))
        if not all(map(_T.is_contiguous, grads)):  # False for sparse tensors too
            raise ValueError("a gradient is not dense and contiguous")
        dtypes = set(map(_dtype_of, grads))
        for d in dtypes:
            if d not in _CODE:
                raise TypeError(f"unsupported gradient dtype {d}")
        sizes = list(map(_T.numel, grads))
        if len(dtypes) == 1:
            codes = [_CODE[d] for d in dtypes] * len(grads)
        else:
            codes = [_CODE[g.dtype] for g in grads]
        if out is not None and (set(map(_dtype_of, out)) != dtypes or list(map(_T.numel, out)) != sizes
                                or not all(map(_T.is_contiguous, out))
                                or (len(dtypes) > 1 and [_CODE[o.dtype] for o in out] != codes)):
            raise ValueError("outputs must be contiguous and of their gradients' sizes and dtypes")
        self.n = len(grads)
        self.dev = grads[0].device
        self.grads = array("Q", map(_T.data_ptr, grads))
        self.outs = self.grads if out is None else array("Q", map(_T.data_ptr, out))
        self.sizes = array("q", sizes)
        self.types = array("i", codes)


def _at(a: array) -> int:
    return a.buffer_info()[0]


def _norm(t: _Table, norm_type, max_norm, loss_scale):
    need = ctypes.c_int64()
    _lib.call("ksd_grad_norm_workspace", _at(t.sizes), t.n, ctypes.byref(need))
    work = torch.empty(need.value, dtype=torch.int8, device=t.dev)
    res = torch.empty(2, dtype=torch.float32, device=t.dev)
    _lib.call("ksd_grad_norm", _at(t.grads), _at(t.sizes), _at(t.types), t.n, int(norm_type == math.inf), max_norm,
              loss_scale, res.data_ptr(), res.data_ptr() + 4, work.data_ptr(), need.value, _lib.stream_ptr(t.dev))
    return res


def gradient_norm(grads, max_norm: float = math.inf, norm_type: float = 2.0, loss_scale: float = 1.0):
    """(norm, factor) as 0-d and 1-element device tensors; factor is what AdamWRequant.step takes as
    ``clip_coef`` to clip the gradients as it loads them. grads: tensors on one GPU."""
    grads = list(grads)
    _check(grads, None, norm_type, loss_scale)
    if not grads:
        raise ValueError("no gradients")
    res = _norm(_Table(grads, None), norm_type, max_norm, loss_scale)
    return res[0], res[1:]


def clip_gradients(grads, max_norm: float, norm_type: float = 2.0, out=None, loss_scale: float = 1.0) -> torch.Tensor:
    """Multiplies every gradient by the factor above, in place or into ``out`` (contiguous tensors of the
    same sizes and dtypes), and returns the norm (0-d, on the device). A tensor that is written may share no
    memory with another of either list (ValueError): the tensors are scaled side by side."""
    grads = list(grads)
    out = None if out is None else list(out)
    _check(grads, out, norm_type, loss_scale)
    if not grads:
        raise ValueError("no gradients")
    t = _Table(grads, out)
    res = _norm(t, norm_type, max_norm, loss_scale)
    _lib.call("ksd_grad_scale", _at(t.grads), _at(t.outs), _at(t.sizes), _at(t.types), t.n, res.data_ptr() + 4,
              _lib.stream_ptr(t.dev))
    _lib.wrote(grads if out is None else out)
    return res[0]


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, loss_scale: float = 1.0) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ on the parameters' gradients, in place (one that is not
    contiguous through a copy). A parameter that is listed more than once (a tied weight gathered
    module by module) counts and is scaled once."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in {id(p): p for p in parameters}.values() if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    copies = [(g, g.contiguous()) for g in grads if not g.is_sparse and not g.is_contiguous()]
    if copies:
        by_id = {id(g): c for g, c in copies}
        grads = [by_id.get(id(g), g) for g in grads]
    norm = clip_gradients(grads, max_norm, norm_type, loss_scale=loss_scale)
    for g, c in copies:
        g.copy_(c)
    return norm
