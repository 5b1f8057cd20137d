"""A training step of the draft model with int8 products scaled per token and output channel:

    lookup     ScaledEmbedding (its gradient by sorted tokens, without atomics)
    linears    TokenChannelLinear: y, dX and dW as int8 products on the same codes (the head's dX
               and dW in groups of 128)
    loss       cross entropy of the head's logits + transfer_weight * the transfer term
    clip       train.clip.gradient_norm over every gradient; the factor goes to the optimizer
    optimizer  AdamWRequant (the factor applied as the gradients are loaded)

``to_token_channel(model)`` converts a float model. The host reads back two checks a step, that the
inputs and that the targets are tokens; a model converted with ``check_ids=False`` reads back nothing.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from ..kernels.embedding import ScaledEmbedding, scaled_rows
from ..kernels.ks3_int8 import KS3Int8Cell
from ..kernels.token_channel import TokenChannelLinear
from . import IGNORE_INDEX, AdamWRequant
from .clip import gradient_norm
from .int8_step import Int8DraftTrainer, _check_loss_scale, transfer_space_loss


def check_targets(tgt: torch.Tensor, V: int, check: bool) -> torch.Tensor:
    """The targets as the losses take them. All must be tokens (a masked target has no row for the
    transfer term): IndexError, before anything runs on them (a host read). Unchecked, those out of
    range become IGNORE_INDEX, on which torch's cross entropy does not abort."""
    bad = (tgt < 0) | (tgt >= V)
    if not check:
        return tgt.masked_fill(bad, IGNORE_INDEX)
    if bool(bad.any()):
        raise IndexError(f"target {int(tgt[bad][0])} is out of range for {V} rows")
    return tgt


class TokenChannelTrainer(Int8DraftTrainer):
    """Int8DraftTrainer's interface (``loss``, ``backward``, ``optimizer_step``, ``step``) on a
    ``to_token_channel`` model. ``grad_norm`` holds the last step's gradient norm (0-d, on the
    device). Every target must be a token. Where the model does not check its ids, an input out of
    range is a row of zeros, a target out of range is left out of the cross entropy and counts as a
    cosine of 0 in the transfer term."""

    def __init__(self, model, lr: float = 3e-4, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, grad_clip: float = 1.0, transfer_weight: float = 0.5,
                 loss_scale: float = 1.0):
        if not isinstance(getattr(model, "head", None), TokenChannelLinear) \
                or not isinstance(model.embedding, ScaledEmbedding):
            raise ValueError("TokenChannelTrainer needs to_token_channel(model)")
        self.model = model
        self.grad_clip = grad_clip
        self.transfer_weight = transfer_weight
        self.loss_scale = _check_loss_scale(loss_scale)
        self.grad_norm = None
        self.opt = AdamWRequant(model.parameters(), lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        for mod in model.modules():
            if isinstance(mod, KS3Int8Cell) and mod.trainable:
                self.opt.register_int8(mod)

    def loss(self, tokens: torch.Tensor, teacher_states: torch.Tensor | None = None):
        """(loss, ce, transfer) as device tensors, with the graph for backward."""
        model, emb = self.model, self.model.embedding
        inp, tgt = tokens[:, :-1], check_targets(tokens[:, 1:], emb.num_embeddings, emb.check_ids)
        h, features = model.backbone(inp, teacher_states)
        rows = scaled_rows(emb.weight, tgt, check_ids=False)
        ts = transfer_space_loss(features, emb.weight, tgt, rows=rows)
        logits = model.head(h.reshape(-1, h.shape[-1]))
        ce = F.cross_entropy(logits.float(), tgt.reshape(-1), ignore_index=IGNORE_INDEX)
        return ce + self.transfer_weight * ts, ce, ts

    def optimizer_step(self):
        grads = [p.grad if p.grad.is_contiguous() else p.grad.contiguous()
                 for p in self.model.parameters() if p.grad is not None]
        self.grad_norm, factor = gradient_norm(grads, self.grad_clip, loss_scale=self.loss_scale)
        self.opt.step(clip_coef=factor)
