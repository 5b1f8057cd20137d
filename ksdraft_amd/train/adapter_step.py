"""A training step of a draft model's adapters on its frozen base (``model.add_adapters`` of a float or a
``to_token_channel`` model):

    loss       cross entropy of the head's logits + transfer_weight * the transfer term
    adapters   dropout on their input, gradients by tokens listed by adapter (kernels.adapters)
    clip       train.clip.gradient_norm over the adapters' gradients; the factor goes to the optimizer
    optimizer  AdamWRequant on the adapters alone
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from ..kernels.ks3_int8 import KS3Int8Cell
from ..model.adapters import adapter_parameters, select_adapters, selected_adapters
from . import IGNORE_INDEX, AdamWRequant
from .clip import gradient_norm
from .int8_step import Int8DraftTrainer, _check_loss_scale, transfer_space_loss
from .token_channel_step import check_targets


class AdapterTrainer(Int8DraftTrainer):
    """Int8DraftTrainer's interface (``loss``, ``backward``, ``optimizer_step``, ``step``) for the adapters of a
    model; ``index`` (B,) names each sequence's adapter. Every target must be a token. ``loss`` leaves its batch's adapters
    selected, which a backward pass with recomputed activations needs; ``step`` gives the selection before it back."""

    def __init__(self, model, lr: float = 3e-4, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                 grad_clip: float = 1.0, transfer_weight: float = 0.5, loss_scale: float = 1.0):
        params = adapter_parameters(model)
        if not params:
            raise ValueError("AdapterTrainer needs add_adapters(model, ...)")
        for m in model.modules():
            if isinstance(m, KS3Int8Cell) and not m.trainable:
                raise ValueError("a KS3Int8Cell without masters passes no gradient: convert with to_token_channel")
        self.model = model
        self.grad_clip = grad_clip
        self.transfer_weight = transfer_weight
        self.loss_scale = _check_loss_scale(loss_scale)
        self.grad_norm = None
        self.opt = AdamWRequant(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)

    def loss(self, tokens: torch.Tensor, index: torch.Tensor, teacher_states: torch.Tensor | None = None):
        """(loss, ce, transfer) as device tensors, with the graph for backward."""
        model = self.model
        inp = tokens[:, :-1]
        tgt = check_targets(tokens[:, 1:], model.config.vocab_size, True)
        select_adapters(model, index)
        h, features = model.backbone(inp, teacher_states)
        rows = F.embedding(tgt, model.head.weight.detach())
        ts = transfer_space_loss(features, model.head.weight, tgt, rows=rows)
        logits = model.head(h)
        ce = F.cross_entropy(logits.reshape(-1, logits.shape[-1]).float(), tgt.reshape(-1), ignore_index=IGNORE_INDEX)
        return ce + self.transfer_weight * ts, ce, ts

    def optimizer_step(self):
        grads = [p.grad for g in self.opt.param_groups for p in g["params"] if p.grad is not None]
        self.grad_norm, factor = gradient_norm(grads, self.grad_clip, loss_scale=self.loss_scale)
        self.opt.step(clip_coef=factor)

    def step(self, tokens: torch.Tensor, index: torch.Tensor, teacher_states: torch.Tensor | None = None):
        self.model.train()
        with selected_adapters(self.model, index):
            loss, ce, ts = self.loss(tokens, index, teacher_states)
            self.backward(loss)
        self.optimizer_step()
        return loss.detach(), ce.detach(), ts.detach()
