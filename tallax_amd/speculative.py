"""Verification of drafted tokens: how many of a draft the target model agrees
with, and the next token.

No counterpart in the reference, whose sampler draws one token a row
(`sampling.sample`).  One call runs hand-written gfx950 kernels
(include/tallax_hip.h: tallax_verify).
"""
from __future__ import annotations

from typing import Any

import torch

from . import _lib


def verify(draft_tokens: torch.Tensor, target_logits: torch.Tensor, uniforms: torch.Tensor, noise: torch.Tensor, *,
           draft_probs: torch.Tensor | None = None, temperature: Any = 1.0, counts: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Accepts drafted tokens so that every token is distributed as the target's.

    draft_tokens [batch, drafted] int32 (drafted up to 63); target_logits
    [batch, drafted + 1, vocab] float32 or bfloat16, row i after i drafted
    tokens; uniforms [batch, drafted] float32 in [0, 1); noise [batch, vocab]
    float32 > 0, standard exponential; draft_probs [batch, drafted, vocab]
    float32 or bfloat16, the distributions the drafts were drawn from (None:
    each draft was certain); temperature a scalar or [batch]; counts [batch]
    int32, how many drafts each sequence has (default: all).

    With p_i = softmax(target_logits_i / temperature), draft x_i is accepted
    while uniforms_i * q_i(x_i) < p_i(x_i).  The next token is argmax_v of
    max(p - q, 0)(v) / noise(v) in the row of the first refused draft, or of
    p(v) / noise(v) after the last accepted one, ties to the lowest id
    (temperature < 1e-5: the drafts are compared with the largest logit, and
    the next token is that one).  -inf logits (a mask's) are never drawn.  The
    sums of p are of 32-bit weights, off by some 1e-7 of themselves; a draft as
    near as that to its border may fall on either side.

    Returns (tokens [batch, drafted + 1] int32: the accepted drafts, the next
    token, then -1; accepted [batch] int32).  workspace: a uint8 device tensor
    that begins on a multiple of 16 bytes, used instead of the shared
    per-device buffer.
    """
    return _lib.SERVING.verify(draft_tokens, target_logits, uniforms, noise, draft_probs, temperature, counts, workspace)


__all__ = ["verify"]
