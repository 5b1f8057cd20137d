"""Int8 embedding gather (the staged int8-embedding surface of the reference's INT8 tier:
ksdraft/model/int8_convert.py:9-12 keeps the embedding float and names the per-row-scale
int8 embedding as a separate surface).

The table is quantized per row in GS groups along d exactly as the tied head's weight is
(quantize_last_dim, reference ksdraft/kernels/quant.py:30-52), so one set of codes serves
both the head GEMM and the lookup. ``embedding_gather_int8`` returns the looked-up rows
dequantized (code * scale, exact in fp32). ``Int8Embedding`` is an nn.Embedding drop-in
(fp32 master ``weight``) whose backward is the float embedding's: the scatter-add of the
upstream gradient into the master (straight through the quantization).

``embedding_lookup`` / ``embedding_gradient`` / ``ScaledEmbedding`` are the float table's lookup
times a scale (nn.Embedding and a multiplication) and its gradient by sorted tokens.
"""

from __future__ import annotations

import ctypes

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .. import _lib
from .quant import GROUP_SIZE, SCALE_DTYPE, quantize_last_dim

_OUT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def embedding_gather_int8(codes: torch.Tensor, scales: torch.Tensor, ids: torch.Tensor,
                          group: int = GROUP_SIZE, out_dtype: torch.dtype = torch.float32,
                          check_ids: bool = True) -> torch.Tensor:
    """codes (V, d) int8, scales (V, ceil(d/group)) fp16, ids (...) int -> (..., d)."""
    dev = _lib.require_gpu(codes, scales, ids)
    if codes.dim() != 2 or codes.dtype != torch.int8:
        raise ValueError("codes must be a 2-D int8 table (V, d)")
    V, d = codes.shape
    if scales.dtype != SCALE_DTYPE or scales.shape != (V, -(-d // group)):
        raise ValueError(f"scales must be ({V}, {-(-d // group)}) float16")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError("ids must be integer token indices")
    code = _OUT.get(out_dtype)
    if code is None:
        raise TypeError(f"unsupported output dtype {out_dtype}")
    flat = ids.reshape(-1).to(torch.int64).contiguous()
    if check_ids and flat.numel():  # as nn.Embedding does on the CPU (a host read)
        bad = (flat < 0) | (flat >= V)
        if bool(bad.any()):
            raise IndexError(f"index {int(flat[bad][0])} is out of range for {V} rows")
    out = torch.empty((flat.numel(), d), dtype=out_dtype, device=dev)
    codes, scales = codes.contiguous(), scales.contiguous()  # outlive the enqueued kernel
    _lib.call("ksd_embedding_gather_int8", codes.data_ptr(),
              scales.data_ptr(), flat.data_ptr(), flat.numel(), V, d, group,
              out.data_ptr(), code, _lib.stream_ptr(dev))
    return out.reshape(*ids.shape, d)


class _RowGather(torch.autograd.Function):
    """weight[ids] (F.embedding) whose backward returns a sparse (COO) gradient: the
    upstream rows summed per distinct id, one entry per distinct row.

    A tied weight (embedding lookups beside the LM head) receives a dense gradient from the
    head; autograd adds the sparse row sums into it (one pass over the dense tensor) instead
    of zero-filling and adding a dense (V, d) gradient per lookup. The values are the dense
    embedding backward's: the upstream rows are summed per distinct id by torch's embedding
    backward over a compact table of the distinct ids (sorted, in position order), found
    without a host sync. Slots past the distinct count carry id 0 and zero sums, so adding
    them leaves row 0 unchanged. When the sparse gradient is the weight's only one, its
    .grad is sparse; the caller that uses this lookup (Int8DraftTrainer) always has the
    head's dense gradient on the same weight."""

    @staticmethod
    def forward(ctx, weight, ids):
        ctx.save_for_backward(ids)
        ctx.shape = weight.shape
        return torch.nn.functional.embedding(ids, weight)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        V, d = ctx.shape
        flat = ids.reshape(-1)
        n = flat.numel()
        sid, order = torch.sort(flat, stable=True)
        head = torch.ones(n, dtype=torch.bool, device=flat.device)
        head[1:] = sid[1:] != sid[:-1]
        slot = torch.cumsum(head, 0) - 1
        inv = torch.empty_like(slot)
        inv[order] = slot
        uids = torch.zeros(n, dtype=torch.int64, device=flat.device)
        uids[slot] = sid
        sums = torch.ops.aten.embedding_dense_backward(grad.reshape(-1, d), inv, n, -1, False)
        return torch.sparse_coo_tensor(uids[None], sums, (V, d), check_invariants=False), None


def gather_rows_sparse_grad(weight: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
    """F.embedding(ids, weight) with a sparse row-sum gradient for ``weight``."""
    return _RowGather.apply(weight, ids)


class _Int8EmbeddingFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, codes, scales, group):
        ctx.save_for_backward(ids)
        ctx.num_weights = weight.shape[0]
        return embedding_gather_int8(codes, scales, ids, group, torch.float32)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        dw = torch.ops.aten.embedding_dense_backward(grad.contiguous(), ids, ctx.num_weights,
                                                     -1, False)
        return None, dw, None, None, None


class Int8Embedding(nn.Module):
    """nn.Embedding(V, d) with an int8 GS128 lookup. The fp32 master ``weight`` stays
    authoritative: the codes are rebuilt every call unless ``codes_from`` (an Int8Linear
    tied to the same weight, e.g. the LM head) holds codes of the master as it is now."""

    def __init__(self, num_embeddings: int, embedding_dim: int, group: int = GROUP_SIZE):
        super().__init__()
        self.num_embeddings = num_embeddings
        self.embedding_dim = embedding_dim
        self.group = group
        self.weight = nn.Parameter(torch.zeros(num_embeddings, embedding_dim))
        self.codes_from = None

    @classmethod
    def from_float(cls, module: nn.Embedding, group: int = GROUP_SIZE) -> "Int8Embedding":
        emb = cls(module.num_embeddings, module.embedding_dim, group)
        emb.weight = module.weight  # the same master (a tied head keeps its tie)
        return emb

    def _codes(self):
        src = self.codes_from
        if (src is not None and src.weight is self.weight and src._codes_current()
                and self.group == GROUP_SIZE):
            return src.weight_codes, src.weight_scales
        return quantize_last_dim(self.weight.detach().float(), self.group)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        codes, scales = self._codes()
        return _Int8EmbeddingFunction.apply(ids, self.weight, codes, scales, self.group)


def _check_ids(ids: torch.Tensor, V: int, check: bool) -> torch.Tensor:
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError("ids must be integer token indices")
    flat = ids if ids.dim() == 1 and ids.is_contiguous() else ids.reshape(-1).contiguous()
    if check and flat.numel():  # as nn.Embedding does on the CPU (a host read)
        bad = (flat < 0) | (flat >= V)
        if bool(bad.any()):
            raise IndexError(f"index {int(flat[bad][0])} is out of range for {V} rows")
    return flat


def _dense_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def embedding_lookup(weight: torch.Tensor, ids: torch.Tensor, scale: float = 1.0,
                     out_dtype: torch.dtype | None = None, check_ids: bool = True) -> torch.Tensor:
    """round(scale * weight[ids]) in out_dtype (weight's by default): weight (V, d) float, ids (...)
    int32 or int64 -> (..., d). The product is fp32, rounded once. With check_ids=False (no host
    sync) an id out of range gives a row of zeros."""
    dev = _lib.require_gpu(weight, ids)
    if weight.dim() != 2:
        raise ValueError("weight must be a 2-D table (V, d)")
    out_dtype = out_dtype or weight.dtype
    if weight.dtype not in _OUT or out_dtype not in _OUT:
        raise TypeError(f"unsupported dtypes {weight.dtype} -> {out_dtype}")
    V, d = weight.shape
    flat = _check_ids(ids, V, check_ids)
    if not weight.is_contiguous():
        weight = _dense_rows(weight)
    out = torch.empty((*ids.shape, d), dtype=out_dtype, device=dev)
    _lib.call("ksd_embedding_lookup", weight.data_ptr(), _OUT[weight.dtype], V, d, weight.stride(0) if V > 1 else d,
              flat.data_ptr(), int(flat.dtype == torch.int64), flat.numel(), scale, out.data_ptr(), _OUT[out_dtype],
              _lib.stream_ptr(dev))
    return out


def embedding_gradient(grad: torch.Tensor, ids: torch.Tensor, num_embeddings: int, scale: float = 1.0,
                       padding_idx: int | None = None, out_dtype: torch.dtype = torch.float32,
                       out: torch.Tensor | None = None, accumulate: bool = False,
                       check_ids: bool = True) -> torch.Tensor:
    """The gradient of embedding_lookup's table: dW[v] = scale * sum of grad[i] over ids[i] == v, in
    fp32, rounded once to out_dtype; the row of padding_idx is 0.

    grad (..., d) float, ids of its leading shape -> (num_embeddings, d). ``out`` (dense) takes the
    result; with accumulate=True the sums are added to what it holds and only the rows of ids that
    occur are touched (a tied head's dense gradient). Without atomics, in an order that the ids and
    sizes fix: repeated calls give the same bits. With check_ids=False (no host sync) ids out of range are left out."""
    dev = _lib.require_gpu(grad, ids, out)
    if grad.shape[:-1] != ids.shape:
        raise ValueError(f"grad {tuple(grad.shape)} does not match ids {tuple(ids.shape)}")
    V, d = int(num_embeddings), grad.shape[-1]
    if out is not None:
        if out.shape != (V, d) or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError(f"out must be a contiguous ({V}, {d}) tensor on a 16-byte boundary")
        out_dtype = out.dtype
    elif accumulate:
        raise ValueError("accumulate=True adds to out, and none is given")
    if grad.dtype not in _OUT or out_dtype not in _OUT:
        raise TypeError(f"unsupported dtypes {grad.dtype} -> {out_dtype}")
    if padding_idx is not None and not -V <= padding_idx < V:
        raise ValueError(f"padding_idx {padding_idx} is out of range for {V} rows")
    pad = -1 if padding_idx is None else padding_idx % V
    flat = _check_ids(ids, V, check_ids)
    g = _dense_rows(grad if grad.dim() == 2 else grad.reshape(flat.numel(), d))
    n = flat.numel()
    given = out is not None
    if out is None:
        out = torch.empty((V, d), dtype=out_dtype, device=dev)
    need = ctypes.c_int64()
    _lib.call("ksd_embedding_gradient_workspace", n, d, ctypes.byref(need))
    work = torch.empty(need.value, dtype=torch.int8, device=dev)
    _lib.call("ksd_embedding_gradient", g.data_ptr(), _OUT[g.dtype], n, d, g.stride(0) if n > 1 else d, flat.data_ptr(),
              int(flat.dtype == torch.int64), V, pad, scale, int(accumulate), out.data_ptr(), _OUT[out_dtype],
              work.data_ptr(), need.value, _lib.stream_ptr(dev))
    if given:
        _lib.wrote((out,))
    return out


class _ScaledLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx, out_dtype, check_ids):
        ctx.save_for_backward(ids)
        ctx.args = (weight.shape[0], scale, padding_idx, weight.dtype)
        return embedding_lookup(weight, ids, scale, out_dtype, check_ids)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        V, scale, pad, dtype = ctx.args
        dw = embedding_gradient(grad, ids, V, scale, pad, dtype, check_ids=False)  # checked in the forward
        return dw, None, None, None, None, None


def scaled_rows(weight: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None,
                out_dtype: torch.dtype | None = None, check_ids: bool = True) -> torch.Tensor:
    """embedding_lookup with embedding_gradient as its backward (a dense gradient of weight)."""
    return _ScaledLookup.apply(weight, ids, scale, padding_idx, out_dtype, check_ids)


class ScaledEmbedding(nn.Module):
    """nn.Embedding(V, d) whose rows come out times ``scale`` (a model's sqrt(d), for instance), in
    ``out_dtype``, with the gradient of embedding_gradient."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0, padding_idx: int | None = None,
                 out_dtype: torch.dtype | None = None, check_ids: bool = True):
        super().__init__()
        if padding_idx is not None and not -num_embeddings <= padding_idx < num_embeddings:
            raise ValueError(f"padding_idx {padding_idx} is out of range for {num_embeddings} rows")
        self.num_embeddings = num_embeddings
        self.embedding_dim = embedding_dim
        self.scale = float(scale)
        self.padding_idx = padding_idx
        self.out_dtype = out_dtype
        self.check_ids = check_ids
        self.weight = nn.Parameter(torch.zeros(num_embeddings, embedding_dim))

    @classmethod
    def from_float(cls, module: nn.Embedding, scale: float = 1.0, **kwargs) -> "ScaledEmbedding":
        for name in ("max_norm", "scale_grad_by_freq", "sparse"):
            if getattr(module, name) not in (None, False):
                raise ValueError(f"ScaledEmbedding has no {name}, and the embedding's is {getattr(module, name)}")
        emb = cls(module.num_embeddings, module.embedding_dim, scale, module.padding_idx, **kwargs)
        emb.weight = module.weight  # the same master (a tied head keeps its tie)
        return emb

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return scaled_rows(self.weight, ids, self.scale, self.padding_idx, self.out_dtype, self.check_ids)
