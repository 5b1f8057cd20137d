"""Model-wide INT8 conversion (mirror of reference ksdraft/model/int8_convert.py:31-52).

``to_int8(model)`` returns a converted copy: Rosa q/k/v/out and ``teacher_proj`` become
``Int8Linear``, each block's KS3 becomes ``KS3Int8Cell``; LayerNorms, the Rosa payload and
time-mix vectors, the DSpine injection and the embedding stay float (the reference's
conversion doctrine). The reference builds the cells without trainable masters
(int8_convert.py:40); ``trainable=True`` builds them with masters and also turns the tied
head into an ``Int8Linear`` sharing the embedding's weight, so every linear of the step
runs INT8 forward and backward (the config-5 training step). ``int8_embedding=True``
also swaps the embedding lookup for the int8 gather over the head's codes, and
``int8_injection=True`` the DSpine injection's low-rank maps for Int8Linear (their rank-32/64
reductions pad to one 128-wide group, quant.py:9-10): the staged surfaces the reference's
doctrine keeps float until gated.

``to_token_channel(model)`` is the training conversion with one scale per token and output channel
instead of one per 128 columns: the same linears become ``TokenChannelLinear``, the embedding a
``ScaledEmbedding`` tied to the head (``train.token_channel_step.TokenChannelTrainer`` steps it).
"""

from __future__ import annotations

import copy

from ..kernels.embedding import Int8Embedding, ScaledEmbedding
from ..kernels.ks3_int8 import KS3Int8Cell
from ..kernels.linear import Int8Linear
from ..kernels.token_channel import TokenChannelLinear
from .draft import KSDraftModel


def _without_adapters(model: KSDraftModel) -> KSDraftModel:
    from .adapters import adapted_layers
    if adapted_layers(model):
        raise ValueError("the model has adapters, which a conversion would drop: convert first, then add_adapters")
    return model


def to_int8(model: KSDraftModel, group: int = 128, nonlinear: str = "int8", *,
            trainable: bool = False, int8_embedding: bool = False,
            int8_injection: bool = False) -> KSDraftModel:
    conv = copy.deepcopy(_without_adapters(model))
    swapped = 0
    for block in conv.blocks:
        rosa = block.rosa
        for name in ("q_proj", "k_proj", "v_proj", "out_proj"):
            setattr(rosa, name, Int8Linear.from_float(getattr(rosa, name)))
            swapped += 1
        block.ffn = KS3Int8Cell(cell=block.ffn, group=group, nonlinear=nonlinear,
                                trainable=trainable)
        swapped += 1
        if int8_injection:  # DSpine's low-rank maps: reduction 32/64 pads to one group
            inj = block.injection
            for name in ("feature_down", "feature_up"):
                setattr(inj, name, Int8Linear.from_float(getattr(inj, name)))
                swapped += 1
            for lr in (inj.gate_q, inj.gate_p, inj.inject):
                lr.down = Int8Linear.from_float(lr.down)
                lr.up = Int8Linear.from_float(lr.up)
                swapped += 2
    if conv.teacher_proj is not None:
        conv.teacher_proj = Int8Linear.from_float(conv.teacher_proj)
        swapped += 1
    if trainable:
        head = Int8Linear(conv.head.in_features, conv.head.out_features, bias=False)
        head.weight = conv.embedding.weight   # tied, as KSDraftModel ties its head
        head.weight_codes = head.weight_scales = None
        conv.head = head
        swapped += 1
    if int8_embedding:  # the staged int8-embedding surface: lookups from the head's codes
        emb = Int8Embedding.from_float(conv.embedding, group)
        if isinstance(conv.head, Int8Linear):
            emb.codes_from = conv.head
        conv.embedding = emb
        swapped += 1
    conv._int8_tier = {"group": group, "nonlinear": nonlinear, "swapped_surfaces": swapped,
                       "trainable": trainable, "int8_embedding": int8_embedding,
                       "int8_injection": int8_injection}
    return conv


def to_token_channel(model: KSDraftModel, group: int = 128, nonlinear: str = "int8", *,
                     embedding_scale: float = 1.0, check_ids: bool = True) -> KSDraftModel:
    """A copy of the model for training with int8 products scaled per token and channel: Rosa
    q/k/v/out, ``teacher_proj`` and the tied head become TokenChannelLinear (the head's gradients in
    groups of 128), the embedding a ScaledEmbedding on the head's weight (rows times
    embedding_scale), the FFNs trainable KS3Int8Cells as in ``to_int8``; norms, vectors and the
    injection stay float."""
    conv = copy.deepcopy(_without_adapters(model))
    swapped = 0
    for block in conv.blocks:
        for name in ("q_proj", "k_proj", "v_proj", "out_proj"):
            setattr(block.rosa, name, TokenChannelLinear.from_float(getattr(block.rosa, name)))
            swapped += 1
        block.ffn = KS3Int8Cell(cell=block.ffn, group=group, nonlinear=nonlinear, trainable=True)
        swapped += 1
    if conv.teacher_proj is not None:
        conv.teacher_proj = TokenChannelLinear.from_float(conv.teacher_proj)
        swapped += 1
    # a cross entropy's gradient over a vocabulary needs more than a scale per token
    head = TokenChannelLinear(conv.head.in_features, conv.head.out_features, bias=False, group_gradient=True)
    head.weight = conv.embedding.weight  # tied, as KSDraftModel ties its head
    conv.head = head
    conv.embedding = ScaledEmbedding.from_float(conv.embedding, embedding_scale, check_ids=check_ids)
    swapped += 2
    conv._int8_tier = {"group": group, "nonlinear": nonlinear, "swapped_surfaces": swapped,
                       "trainable": True, "scales": "token_channel"}
    return conv


def int8_surfaces(converted: KSDraftModel) -> dict:
    info = getattr(converted, "_int8_tier", None)
    return dict(info) if info else {}
