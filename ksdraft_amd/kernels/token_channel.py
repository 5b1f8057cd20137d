"""W8A8 products with one fp32 scale per token and one per output channel.

The group-128 product (``kernels.gemm``) rescales its int32 sums every 128 columns; here the
scales stand outside the whole reduction:

    y[m, n] = (sum_k xq[m, k] wq[n, k]) * sx[m] * sw[n] + bias[n]

``quantize_rows`` gives the codes of either operand (symmetric, max |row| / 127). Both gradients
use the forward's codes as they are: a scale along the contracted dimension moves into dY before
dY is quantized,

    dX = e[m] sum_n q[m, n] wq[n, k],   (q, e) = quantize_rows(dY * sw)
    dW = f[n] sum_m c[m, n] xq[m, k],   (c, f) = the same per column of dY * sx

What of a row of dY * sw (dX) or a column of dY * sx (dW) lies below 1/254 of the largest value there
is lost. That is a small part of a projection's gradient and nearly all of a vocabulary head's: a cross
entropy's dY is about -1 at the target and a probability elsewhere, and at 20000 classes the target's
code is the only one left of a row. Such a layer takes its gradients from dY in groups of 128
(``group_gradient``).

``TokenChannelLinear`` is an nn.Linear drop-in on them. There is no CPU path.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .. import _lib
from .linear import w8a8_linear_backward
from .quant import quantize_dual

_OUT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _pitch(n: int) -> int:
    return -(-n // 16) * 16


def _matrix(x: torch.Tensor, name: str) -> torch.Tensor:
    """A 2-D float tensor with dense rows, as the kernels read it."""
    if x.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got {tuple(x.shape)}")
    if x.dtype not in _OUT:
        raise TypeError(f"{name}: unsupported dtype {x.dtype}")
    if x.shape[1] == 0:
        raise ValueError(f"{name} has no columns")
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _rows(x: torch.Tensor, dev: torch.device):
    """Codes in a (M, pitch) buffer with zeros past K, and scales."""
    M, K = x.shape
    codes = torch.empty((M, _pitch(K)), dtype=torch.int8, device=dev)
    scales = torch.empty(M, dtype=torch.float32, device=dev)
    _lib.call("ksd_tc_quantize_rows", x.data_ptr(), _OUT[x.dtype], M, K, x.stride(0) if M > 1 else K,
              codes.data_ptr(), codes.shape[1], scales.data_ptr(), _lib.stream_ptr(dev))
    return codes, scales


def quantize_rows(x: torch.Tensor):
    """x (M, K) float -> (codes (M, K) int8, scales (M,) fp32) with x ~ codes * scales[:, None].

    Per row: a = max |x|; scale = a / 127 and code = rint(x * (127 / a)), each operation rounded to
    fp32; a < 2**-100 gives scale 0 and codes 0, a row with NaN or inf scale NaN and codes 0. The
    codes are a view of rows padded with zeros to a multiple of 16 bytes, the layout the products
    read without a copy."""
    dev = _lib.require_gpu(x)
    x = _matrix(x, "x")
    codes, scales = _rows(x, dev)
    return codes[:, :x.shape[1]], scales


def _codes_operand(q: torch.Tensor, name: str, zeros: bool = False):
    """An int8 matrix as the products read it: (tensor that owns the memory, row pitch). Rows whose
    pitch is no multiple of 16, or that end before their last 16-byte chunk does, are copied; with
    ``zeros`` (one operand of a product needs zeros up to its rows' next multiple of 16) also rows
    of another length, since what follows a caller's rows is not known."""
    if q.dim() != 2 or q.dtype != torch.int8:
        raise ValueError(f"{name} must be a 2-D int8 tensor")
    M, K = q.shape
    if K == 0:
        raise ValueError(f"{name} has no columns")
    ld = q.stride(0) if M > 1 else _pitch(K)
    if q.stride(1) == 1 and ld % 16 == 0 and ld >= _pitch(K) and q.data_ptr() % 16 == 0:
        if K % 16 == 0:
            return q, ld
        end = q.storage_offset() + max(M - 1, 0) * ld + _pitch(K)
        if not zeros and end <= q.untyped_storage().nbytes():
            return q, ld
    out = torch.zeros((M, _pitch(K)), dtype=torch.int8, device=q.device)
    out[:, :K] = q
    return out, _pitch(K)


def _vector(t: torch.Tensor | None, n: int, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != n:
        raise ValueError(f"{name} must hold {n} float32 values, got {tuple(t.shape)} {t.dtype}")
    return t.contiguous()


def _gemm(a, lda, a_t, sa, w, ldw, w_t, sw, M, N, K, bias, residual, out_dtype, dev):
    y = torch.empty((M, N), dtype=out_dtype, device=dev)
    need = ctypes.c_int64()
    _lib.call("ksd_tc_gemm_workspace", M, N, K, ctypes.byref(need))
    work = torch.empty(need.value, dtype=torch.int8, device=dev) if need.value else None
    _lib.call("ksd_tc_gemm", a.data_ptr(), lda, a_t, _lib.ptr(sa), w.data_ptr(), ldw, w_t, _lib.ptr(sw), M, N, K,
              _lib.ptr(bias), _lib.ptr(residual), y.data_ptr(), _OUT[out_dtype], _lib.ptr(work), need.value,
              _lib.stream_ptr(dev))
    return y


def _epilogue(lead, N: int, bias, residual, out_dtype):
    """Checks what is added to an output (*lead, N)."""
    if out_dtype not in _OUT:
        raise TypeError(f"unsupported output dtype {out_dtype}")
    bias = _vector(bias, N, "bias")
    if residual is not None:
        if residual.shape != (*lead, N) or residual.dtype != out_dtype:
            raise ValueError(f"residual must be {(*lead, N)} {out_dtype}, got {tuple(residual.shape)} {residual.dtype}")
        residual = residual.contiguous()
    return bias, residual


def token_channel_gemm(a_codes: torch.Tensor, a_scales: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor,
                       bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                       out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y = (a_codes . w_codes^T) * a_scales[:, None] * w_scales (+ bias) (+ residual), in fp32,
    rounded once to out_dtype. a_codes (M, K), w_codes (N, K) int8 with |code| <= 127; scales and
    bias fp32. K must be the same; the int32 sums are exact for any K."""
    dev = _lib.require_gpu(a_codes, a_scales, w_codes, w_scales, bias, residual)
    a, lda = _codes_operand(a_codes, "a_codes", zeros=True)
    w, ldw = _codes_operand(w_codes, "w_codes")
    (M, K), (N, Kw) = a_codes.shape, w_codes.shape
    if K != Kw:
        raise ValueError(f"a_codes has {K} columns, w_codes {Kw}")
    bias, residual = _epilogue((M,), N, bias, residual, out_dtype)
    return _gemm(a, lda, 0, _vector(a_scales, M, "a_scales"), w, ldw, 0, _vector(w_scales, N, "w_scales"), M, N, K,
                 bias, residual, out_dtype, dev)


def token_channel_linear(x: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor,
                         bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                         out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y = W8A8(x, W) + bias (+ residual): x (..., K) float is quantized per token and multiplied
    with the stored codes (N, K) of quantize_rows(weight). The output has x's dtype unless
    out_dtype is given; residual is (..., N) of the output's."""
    dev = _lib.require_gpu(x, w_codes, w_scales, bias, residual)
    w, ldw = _codes_operand(w_codes, "w_codes")
    N, K = w_codes.shape
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x has shape {tuple(x.shape)}, w_codes {tuple(w_codes.shape)}")
    flat = x.dim() == 2  # a decode call's cost is this function's: no views that change nothing
    x2 = _matrix(x if flat else x.reshape(-1, K), "x")
    M = x2.shape[0]
    out_dtype = out_dtype or x.dtype
    bias, residual = _epilogue(x.shape[:-1], N, bias, residual, out_dtype)
    w_scales = _vector(w_scales, N, "w_scales")
    y = torch.empty((M, N) if flat else (*x.shape[:-1], N), dtype=out_dtype, device=dev)
    need = ctypes.c_int64()
    _lib.call("ksd_tc_linear_workspace", M, N, K, ctypes.byref(need))
    work = torch.empty(need.value, dtype=torch.int8, device=dev) if need.value else None
    _lib.call("ksd_tc_linear", x2.data_ptr(), _OUT[x2.dtype], M, K, x2.stride(0) if M > 1 else K, w.data_ptr(), ldw,
              w_scales.data_ptr(), N, _lib.ptr(bias), _lib.ptr(residual), y.data_ptr(), _OUT[out_dtype],
              _lib.ptr(work), need.value, _lib.stream_ptr(dev))
    return y


class Saved:
    """What token_channel_linear_backward needs of a training forward: both operands' codes and
    scales (a byte per element of x and W instead of x itself)."""

    __slots__ = ("xq", "xs", "wq", "ws", "M", "N", "K", "dtype", "lead", "has_bias")


def token_channel_linear_train(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                               residual: torch.Tensor | None = None):
    """The training forward on a float master ``weight`` (N, K): quantizes both operands and returns
    (y, saved), y as token_channel_linear gives it in x's dtype."""
    dev = _lib.require_gpu(x, weight, bias, residual)
    w2 = _matrix(weight, "weight")
    N, K = w2.shape
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x has shape {tuple(x.shape)}, weight {tuple(weight.shape)}")
    x2 = _matrix(x.reshape(-1, K), "x")
    s = Saved()
    s.M, s.N, s.K, s.dtype, s.lead, s.has_bias = x2.shape[0], N, K, x.dtype, x.shape[:-1], bias is not None
    bias, residual = _epilogue(s.lead, N, bias, residual, x.dtype)
    M, ld = s.M, _pitch(K)
    codes = torch.empty((M + N, ld), dtype=torch.int8, device=dev)
    scales = torch.empty(M + N, dtype=torch.float32, device=dev)
    s.xq, s.wq, s.xs, s.ws = codes[:M], codes[M:], scales[:M], scales[M:]
    y = torch.empty((*s.lead, N), dtype=x.dtype, device=dev)
    need = ctypes.c_int64()
    _lib.call("ksd_tc_gemm_workspace", M, N, K, ctypes.byref(need))
    work = torch.empty(need.value, dtype=torch.int8, device=dev) if need.value else None
    _lib.call("ksd_tc_linear_train", x2.data_ptr(), _OUT[x2.dtype], M, K, x2.stride(0) if M > 1 else K, w2.data_ptr(),
              _OUT[w2.dtype], N, w2.stride(0) if N > 1 else K, _lib.ptr(bias), _lib.ptr(residual), s.xq.data_ptr(),
              s.xs.data_ptr(), s.wq.data_ptr(), s.ws.data_ptr(), y.data_ptr(), _OUT[x.dtype], _lib.ptr(work),
              need.value, _lib.stream_ptr(dev))
    return y, s


def token_channel_linear_backward(grad: torch.Tensor, saved: Saved, need_dx: bool = True, need_dw: bool = True,
                                  need_db: bool | None = None):
    """(dx in x's dtype, dw (N, K) fp32, db (N,) fp32) for the upstream gradient of y; what is not
    needed is None (db by default when the layer has a bias)."""
    dev = _lib.require_gpu(grad, saved.xq)
    M, N, K = saved.M, saved.N, saved.K
    if grad.shape != (*saved.lead, N):
        raise ValueError(f"grad has shape {tuple(grad.shape)}, the output {(*saved.lead, N)}")
    g = _matrix(grad.reshape(-1, N), "grad")
    need_db = saved.has_bias if need_db is None else need_db
    if M == 0:
        return (torch.empty((*saved.lead, K), dtype=saved.dtype, device=dev) if need_dx else None,
                torch.zeros((N, K), device=dev) if need_dw else None,
                torch.zeros(N, device=dev) if need_db else None)
    dx = torch.empty((*saved.lead, K), dtype=saved.dtype, device=dev) if need_dx else None
    dw = torch.empty((N, K), dtype=torch.float32, device=dev) if need_dw else None
    db = torch.empty(N, dtype=torch.float32, device=dev) if need_db else None
    need = ctypes.c_int64()
    _lib.call("ksd_tc_linear_backward_workspace", M, N, K, need_dx, need_dw, ctypes.byref(need))
    work = torch.empty(need.value, dtype=torch.int8, device=dev)
    _lib.call("ksd_tc_linear_backward", g.data_ptr(), _OUT[g.dtype], M, N, g.stride(0) if M > 1 else N, K,
              saved.xq.data_ptr(), saved.xs.data_ptr(), saved.wq.data_ptr(), saved.ws.data_ptr(), _lib.ptr(dx),
              _OUT[saved.dtype], _lib.ptr(dw), _lib.ptr(db), work.data_ptr(), need.value, _lib.stream_ptr(dev))
    return dx, dw, db


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual):
        y, saved = token_channel_linear_train(x, weight, bias, residual)
        # through save_for_backward, so that they are freed with the graph
        ctx.save_for_backward(saved.xq, saved.xs, saved.wq, saved.ws)
        ctx.shape = (saved.M, saved.N, saved.K, saved.dtype, saved.lead, saved.has_bias)
        ctx.weight_dtype = weight.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        s = Saved()
        s.xq, s.xs, s.wq, s.ws = ctx.saved_tensors
        s.M, s.N, s.K, s.dtype, s.lead, s.has_bias = ctx.shape
        need = ctx.needs_input_grad
        if grad.dtype not in _OUT:
            grad = grad.float()
        dx, dw, db = token_channel_linear_backward(grad, s, need[0], need[1], need[2])
        return dx, None if dw is None else dw.to(ctx.weight_dtype), db, grad if need[3] else None


def _lift(g: torch.Tensor):
    """(g * s, 1 / s) for the power of two s that brings max |g| to [2^20, 2^21), without a host read.
    The groups' fp16 scales keep all their bits from 2^-14 on, so 28 binades below the largest value do
    (a mean loss over 8192 tokens has probabilities near 1e-9 in its gradient). For a g with NaN or inf
    the second is NaN: a group's code of inf is finite."""
    from ..train.clip import gradient_norm
    if g.dtype == torch.float16:
        g = g.float()  # 2^20 is past its range
    top = gradient_norm([g], norm_type=math.inf)[0].view(torch.int32) >> 23  # biased exponent
    shift = torch.where(top == 255, 0, 127 + 20 - top).clamp(max=126)
    s = ((127 + shift) << 23).view(torch.float32)
    back = torch.where(top == 255, 0x7fc00000, (127 - shift) << 23).view(torch.float32)
    return g * s.to(g.dtype), back


class _GroupGradientFunction(torch.autograd.Function):
    """_LinearFunction's forward with Int8Linear's backward: dY, X and W in groups of 128 along what
    each product contracts."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual):
        y, saved = token_channel_linear_train(x, weight, bias, residual)
        ctx.shape = (saved.M, saved.N, saved.K, x.dtype, saved.lead)
        xt = (None, None)
        if ctx.needs_input_grad[1] and saved.M:  # dW's operand instead of x itself
            xt = quantize_dual(x.reshape(-1, saved.K), t_from_codes=True)[2:]
        ctx.save_for_backward(weight, *xt)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        weight, *xt = ctx.saved_tensors
        M, N, K, dtype, lead = ctx.shape
        need_dx, need_dw, need_db, need_res = ctx.needs_input_grad
        g = grad if grad.dtype in _OUT else grad.float()
        dres = g if need_res else None
        if M == 0 or not (need_dx or need_dw):
            return (torch.empty((*lead, K), dtype=dtype, device=g.device) if need_dx else None,
                    torch.zeros_like(weight) if need_dw else None, g.reshape(-1, N).float().sum(0) if need_db else None, dres)
        g, back = _lift(g.reshape(-1, N).contiguous())
        wt = quantize_dual(weight.float(), t_from_codes=True)[2:] if need_dx else None
        dx, dw, *db = w8a8_linear_backward(g, None, None, None, None, need_dx=need_dx, need_dw=need_dw,
                                           xt=xt if need_dw else None, wt=wt, want_db=need_db)
        return ((dx * back).to(dtype).reshape(*lead, K) if need_dx else None,
                dw.mul_(back).to(weight.dtype) if need_dw else None, db[0] * back if need_db else None, dres)


class TokenChannelLinear(nn.Module):
    """nn.Linear with int8 products in both directions, scales per token and per output channel.
    With ``group_gradient`` the backward's operands have a scale per 128 values of what is contracted,
    as Int8Linear's: for a layer whose upstream gradient holds values of very different size in one
    row, as a vocabulary head's.

    The float master ``weight`` stays authoritative: its codes are rebuilt in every call, unless
    ``pack()`` has stored them (serving). Stored codes belong to the master's tensor, storage and
    version at that time: a call that finds another rebuilds and stores them again (a write that
    torch does not version, through ``weight.data`` or a raw pointer, needs another ``pack()``).
    ``unpack()``, training calls, moves and state-dict loads drop them."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, group_gradient: bool = False):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.group_gradient = group_gradient
        self.weight = nn.Parameter(torch.zeros(out_features, in_features))
        self.bias = nn.Parameter(torch.zeros(out_features)) if bias else None
        self._packed = self._packed_of = None  # codes and scales, and the master that they are of

    @classmethod
    def from_float(cls, module: nn.Linear, group_gradient: bool = False) -> "TokenChannelLinear":
        lin = cls(module.in_features, module.out_features, module.bias is not None, group_gradient)
        lin = lin.to(module.weight.device)
        with torch.no_grad():
            lin.weight.copy_(module.weight)
            if module.bias is not None:
                lin.bias.copy_(module.bias)
        return lin

    def pack(self) -> "TokenChannelLinear":
        """Stores the codes of the master as it is now for calls without gradients."""
        self._packed = quantize_rows(self.weight.detach())
        self._packed_of = self._master()
        return self

    def _master(self):
        w = self.weight
        return w, w.data_ptr(), 0 if w.is_inference() else w._version

    def _stored(self):
        if self._packed is not None:
            (was, at, version), (w, now_at, now) = self._packed_of, self._master()
            if was is not w or at != now_at or version != now:
                self.pack()
        return self._packed

    def unpack(self) -> "TokenChannelLinear":
        self._packed = self._packed_of = None
        return self

    def _apply(self, fn, *args, **kwargs):
        self.unpack()
        return super()._apply(fn, *args, **kwargs)

    def _load_from_state_dict(self, *args, **kwargs):
        self.unpack()
        return super()._load_from_state_dict(*args, **kwargs)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        """linear(x), or with ``residual`` (shaped like it) their sum, added in the product's store
        where it has x's dtype."""
        if residual is not None and residual.dtype != x.dtype:
            return residual + self.forward(x)
        bias = self.bias if self.bias is None or self.bias.dtype == torch.float32 else self.bias.float()
        if torch.is_grad_enabled() and (self.weight.requires_grad or x.requires_grad
                                        or (bias is not None and bias.requires_grad)
                                        or (residual is not None and residual.requires_grad)):
            self.unpack()
            function = _GroupGradientFunction if self.group_gradient else _LinearFunction
            return function.apply(x, self.weight, bias, residual)
        codes, scales = self._stored() or quantize_rows(self.weight.detach())
        return token_channel_linear(x, codes, scales, None if bias is None else bias.detach(), residual)
