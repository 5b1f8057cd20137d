"""Low-rank adapters on a draft model's projections: one frozen base serves many requests or tenants, each
with its own adapter, or none.

    model = add_adapters(to_token_channel(draft), count=8, rank=16)
    select_adapters(model, index)        # (B,): the adapter of each sequence, -1 for none
    logits, features = model(tokens)

``add_adapters`` returns a copy whose chosen projections are ``AdaptedLinear`` and whose other parameters are
frozen; ``train.adapter_step.AdapterTrainer`` trains the adapters.
"""

from __future__ import annotations

import contextlib
import copy
import threading

import torch
from torch import nn

from ..kernels.adapters import adapt, adapter_linear
from ..kernels.dropout import Dropout
from ..kernels.linear import Int8Linear
from ..kernels.token_channel import TokenChannelLinear

ROSA = ("q_proj", "k_proj", "v_proj", "out_proj")
_ADAPTABLE = (nn.Linear, Int8Linear, TokenChannelLinear)


class AdapterSelection:
    """The index that a model's AdaptedLinear layers share; None: no adapter anywhere. ``lock`` is held where the index
    belongs to one caller (``selected_adapters``)."""

    def __init__(self):
        self.index = None
        self.lock = threading.RLock()

    def __getstate__(self):
        return {"index": self.index}

    def __setstate__(self, state):
        self.__init__()
        self.index = state["index"]

    def __deepcopy__(self, memo):
        return AdapterSelection()  # a copied model selects for itself


class AdaptedLinear(nn.Module):
    """base(x) + scales_i (dropout(x) A_i^T) B_i^T with the adapters that ``selection`` names. The base layer
    (nn.Linear, Int8Linear, TokenChannelLinear) is called as it is; A starts like an nn.Linear's weight, B at
    zero. The adapters are kept in fp32 and used in x's type; their gradients are fp32."""

    def __init__(self, base: nn.Module, count: int, rank: int, selection: AdapterSelection, alpha: float | None = None,
                 dropout: float = 0.0, seed: int | None = None):
        super().__init__()
        if not isinstance(base, _ADAPTABLE):
            raise TypeError(f"adapters go on nn.Linear, Int8Linear and TokenChannelLinear, not on {type(base).__name__}")
        if count < 1 or not 1 <= rank <= 128:
            raise ValueError(f"one adapter or more of rank 1 to 128, got {count} of {rank}")
        self.base = base
        self.selection = selection
        device = base.weight.device
        self.adapter_a = nn.Parameter(torch.empty(count, rank, base.in_features, device=device))
        self.adapter_b = nn.Parameter(torch.zeros(count, base.out_features, rank, device=device))
        bound = base.in_features ** -0.5
        nn.init.uniform_(self.adapter_a, -bound, bound)
        scale = 1.0 if alpha is None else alpha / rank
        self.register_buffer("adapter_scales", torch.full((count,), float(scale), device=device))
        self.dropout = Dropout(dropout, seed)

    def _apply(self, fn, *args, **kwargs):
        adapters = {id(t) for p in (self.adapter_a, self.adapter_b, self.adapter_scales) for t in (p, p.grad)}

        def move(t):  # a model's .bfloat16() and the like: the adapters move, and keep their type
            out = fn(t)
            return t.to(out.device) if id(t) in adapters and out.dtype != t.dtype else out
        return super()._apply(move, *args, **kwargs)

    @property
    def in_features(self) -> int:
        return self.base.in_features

    @property
    def out_features(self) -> int:
        return self.base.out_features

    @property
    def weight(self) -> torch.Tensor:
        return self.base.weight

    @property
    def bias(self):
        return self.base.bias

    def _index(self, x: torch.Tensor):
        """The selection as one entry for each row of x, or for each of its first dimension's."""
        index = self.selection.index
        if index is None or index.shape == x.shape[:index.dim()]:
            return index
        rows = x.numel() // x.shape[-1]
        if index.numel() and rows % index.numel() == 0 and x.dim() == 2:  # a flattened (B, T, .)
            return index.reshape(-1, 1).expand(-1, rows // index.numel()).reshape(-1)
        raise ValueError(f"the selected adapters {tuple(index.shape)} do not match an input {tuple(x.shape)}")

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        x = x.contiguous()  # dense rows for both products (kernels.linear.dense_rows, once)
        if residual is None:
            y = self.base(x)
        elif isinstance(self.base, nn.Linear):
            y = residual + self.base(x)
        else:
            y = self.base(x, residual=residual)
        index = self._index(x)
        if index is None:
            return y
        a, b = self.adapter_a, self.adapter_b
        if y.dtype != x.dtype:  # a residual of another type
            return y + self._delta(x, a, b, index).to(y.dtype)
        if (self.training and self.dropout.p) or (torch.is_grad_enabled() and (
                y.requires_grad or x.requires_grad or a.requires_grad or b.requires_grad)):
            return self._delta(x, a, b, index, y)
        a, b = a.to(x.dtype), b.to(x.dtype)
        return adapter_linear(x, a, b, index, self.adapter_scales, base=y)  # not into y: a hook of the base may hold it

    def _delta(self, x, a, b, index, base=None):
        p = self.dropout.p if self.training else 0.0
        stream = self.dropout.next_stream() if p else 0
        return adapt(x, a, b, index, self.adapter_scales, base, p, self.dropout.seed, stream)


def adapted_layers(model: nn.Module) -> list:
    return [m for m in model.modules() if isinstance(m, AdaptedLinear)]


def adapter_parameters(model: nn.Module) -> list:
    return [p for m in adapted_layers(model) for p in (m.adapter_a, m.adapter_b)]


def adapter_state_dict(model: nn.Module) -> dict:
    """The adapters' part of the state dict: load it with ``strict=False`` into a model of the same adapters."""
    return {k: v for k, v in model.state_dict().items() if k.rsplit(".", 1)[-1].startswith("adapter_")}


def select_adapters(model: nn.Module, index: torch.Tensor | None) -> None:
    """The adapters of the next calls: integers (B,) for each sequence, (B, T) for each token, values outside
    [0, count) for none; None: no adapter anywhere. The tensor is read when a layer runs. A model has one selection:
    threads that call it for different requests use ``selected_adapters``."""
    for s in _selections(model, index):
        s.index = index


@contextlib.contextmanager
def selected_adapters(model: nn.Module, index: torch.Tensor | None):
    """``select_adapters`` for the calls of a with block, the selection before it again behind it. Blocks of other threads on
    the same model wait (for the calls' launches, not for the GPU), so each sees its own adapters in every layer."""
    with contextlib.ExitStack() as held:
        selections = _selections(model, index)
        if torch._C._current_graph_task_id() == -1:  # a backward pass runs again what its caller's block covers, in another thread
            for s in selections:
                held.enter_context(s.lock)
        before = [s.index for s in selections]
        try:
            for s in selections:
                s.index = index
            yield
        finally:
            for s, i in zip(selections, before):
                s.index = i


def _selections(model: nn.Module, index: torch.Tensor | None) -> list:
    """The model's selections (one, unless adapters were added twice) in the order in which they are locked."""
    layers = adapted_layers(model)
    if not layers:
        raise ValueError("the model has no adapters (add_adapters)")
    if index is not None and index.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"index must be integers, got {index.dtype}")
    return sorted({id(m.selection): m.selection for m in layers}.values(), key=id)


def add_adapters(model: nn.Module, count: int, rank: int, *, targets=ROSA, alpha: float | None = None, dropout: float = 0.0,
                 seed: int | None = None) -> nn.Module:
    """A copy of a draft model (float, ``to_int8`` or ``to_token_channel``) with ``count`` adapters of ``rank`` on each
    of ``targets`` (Rosa's q/k/v/out projections, "head", "teacher_proj", and "down" and "up" of a float KS3), every
    other parameter frozen. Their sum counts alpha / rank times (None: once). dropout is that of the adapters' input in
    training; with a seed, layer i draws its masks from seed + i."""
    conv = copy.deepcopy(model)
    selection = AdapterSelection()
    for p in conv.parameters():
        p.requires_grad_(False)
    unknown = set(targets) - set(ROSA) - {"head", "teacher_proj", "down", "up"}
    if unknown or not targets:
        raise ValueError(f"adapters go on {', '.join(ROSA)}, head, teacher_proj, down and up, not on {sorted(unknown)}")
    made = 0
    for name in targets:
        if name in ROSA:
            owners = [b.rosa for b in conv.blocks]
        elif name in ("down", "up"):
            owners = [b.ffn for b in conv.blocks]
        else:
            owners = [conv]
        for owner in owners:
            base = getattr(owner, name, None)
            if not isinstance(base, _ADAPTABLE):
                raise ValueError(f"the model's {name} takes no adapter ({type(base).__name__})")
            setattr(owner, name, AdaptedLinear(base, count, rank, selection, alpha, dropout,
                                               None if seed is None else seed + made))
            made += 1
    return conv
