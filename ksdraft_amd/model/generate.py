"""Drafting and verification: a draft model proposes a block of tokens, the target model's logits verify it.

    draft_tokens, draft_logits = draft_block(draft, tokens, 16, uniforms)
    out, accepted = verify_draft(target(tokens + draft_tokens), draft_tokens, ...)

``speculative_step`` does both. All random numbers are inputs; the tokens that come out are distributed as the
target's own (greedily: are the target's own), whatever the draft model proposes.
"""

from __future__ import annotations

import torch

from ..kernels.speculate import sample_tokens, verify_draft


def _fed(drawn: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Drawn tokens as a model takes them: -1, of a row without a distribution, is no row of an embedding."""
    return drawn.clamp(min=0).to(dtype)


@torch.no_grad()
def draft_block(model, tokens: torch.Tensor, length: int, uniforms: torch.Tensor | None = None, temperatures=None,
                teacher_states: torch.Tensor | None = None):
    """(draft_tokens (B, length) int64, draft_logits (B, length, V)) behind tokens (B, T): token by token, each drawn
    from softmax(logits / T) by its number of uniforms (B, length). temperatures: (B,) float32, a number, or None
    (1); at the number 0 the largest logit is taken and uniforms may be None. teacher_states (B, T, teacher_dim):
    positions behind T get the last one's. A row without a distribution (NaN, or no finite logit) drafts -1, which
    verification refuses; the model goes on from token 0 there."""
    if length < 1:
        raise ValueError(f"a block has one token or more, got {length}")
    if uniforms is not None and uniforms.shape != (tokens.shape[0], length):
        raise ValueError(f"uniforms must be {(tokens.shape[0], length)}, got {tuple(uniforms.shape)}")
    seen, drafted, rows = tokens, [], None
    for t in range(length):
        states = teacher_states
        if states is not None and t:
            states = torch.cat([states, states[:, -1:].expand(-1, t, -1)], 1)
        logits = model(seen, states)[0][:, -1] if states is not None else model(seen)[0][:, -1]
        token = sample_tokens(logits, None if uniforms is None else uniforms[:, t], temperatures)
        drafted.append(token)
        if rows is None:
            rows = logits.new_empty(logits.shape[0], length, logits.shape[1])
        rows[:, t] = logits  # a copy: a view would keep the logits of all positions
        del logits
        seen = torch.cat([seen, _fed(token[:, None], seen.dtype)], 1)
    return torch.stack(drafted, 1), rows


@torch.no_grad()
def speculative_step(draft, target, tokens: torch.Tensor, length: int, uniforms: torch.Tensor | None = None, temperatures=None,
                     teacher_states: torch.Tensor | None = None):
    """One round behind tokens (B, T): the draft model's block, the target's one pass over it, the verification.

    target(tokens (B, T + length)) -> logits (B, T + length, V) (or a tuple that begins with them). uniforms
    (B, 2 length + 1) float32: the block's draws, its tests, and the last draw; None with temperatures 0. Returns
    (tokens (B, length + 1): the accepted ones, one of the target's, -1 behind it; accepted (B,))."""
    B, T = tokens.shape
    if uniforms is not None and uniforms.shape != (B, 2 * length + 1):
        raise ValueError(f"uniforms must be {(B, 2 * length + 1)}, got {tuple(uniforms.shape)}")
    first = None if uniforms is None else uniforms[:, :length]
    block, block_logits = draft_block(draft, tokens, length, first, temperatures, teacher_states)
    logits = target(torch.cat([tokens, _fed(block, tokens.dtype)], 1))
    logits = logits[0] if isinstance(logits, tuple) else logits
    logits = logits[:, T - 1:]
    if logits.dtype != block_logits.dtype:  # not one in the other's type: the block was drawn from its logits as they are
        logits, block_logits = logits.float(), block_logits.float()
    return verify_draft(logits, block, None if uniforms is None else uniforms[:, length:], draft_logits=block_logits,
                        temperatures=temperatures)
