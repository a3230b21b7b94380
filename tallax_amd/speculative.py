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
from .sampling import _per_row


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
    the next token is that one).  -inf logits (a mask's) are never drawn.

    Returns (tokens [batch, drafted + 1] int32: the accepted drafts, the next
    token, then -1; accepted [batch] int32).
    """
    _lib.require_cuda(target_logits, draft_tokens, uniforms, noise)
    if target_logits.ndim != 3 or target_logits.shape[1] < 1 or target_logits.shape[2] < 1:
        raise ValueError(f"target_logits must be [batch, drafted + 1, vocab], got {tuple(target_logits.shape)}")
    batch, rows, vocab = target_logits.shape
    drafted = rows - 1
    for name, t, shape, dtype in (("draft_tokens", draft_tokens, (batch, drafted), torch.int32),
                                  ("uniforms", uniforms, (batch, drafted), torch.float32),
                                  ("noise", noise, (batch, vocab), torch.float32)):
        if t.shape != shape or t.dtype is not dtype:
            raise ValueError(f"{name} must be a {dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    dt = _lib.dtype_code(target_logits)
    if dt == _lib.I32:
        raise NotImplementedError("verify needs float logits")
    qdt = _lib.F32
    if draft_probs is not None:
        _lib.require_cuda(target_logits, draft_probs)
        if draft_probs.shape != (batch, drafted, vocab):
            raise ValueError(f"draft_probs must be of shape {(batch, drafted, vocab)}, got {tuple(draft_probs.shape)}")
        qdt = _lib.dtype_code(draft_probs)
        if qdt == _lib.I32:
            raise NotImplementedError("verify needs float draft probabilities")
        draft_probs = draft_probs.contiguous()
    dev = target_logits.device
    if counts is not None:
        _lib.require_cuda(target_logits, counts)
        if counts.shape != (batch,) or counts.dtype is not torch.int32:
            raise ValueError(f"counts must be an int32 tensor of shape ({batch},)")
        counts = counts.contiguous()
    temp = _per_row(temperature, batch, torch.float32, dev)
    logits, draft = target_logits.contiguous(), draft_tokens.contiguous()
    uniforms, noise = uniforms.contiguous(), noise.contiguous()
    tokens = torch.empty((batch, rows), dtype=torch.int32, device=dev)
    accepted = torch.empty(batch, dtype=torch.int32, device=dev)
    need = _lib.LIB.tallax_verify_workspace_size(batch, drafted, vocab, dt)
    ws = _lib.workspace_arg(workspace, dev, max(need, 1))
    _lib.check(_lib.LIB.tallax_verify(
        draft.data_ptr(), logits.data_ptr(), dt, batch, drafted, vocab, _lib.ptr(counts), temp.data_ptr(),
        _lib.ptr(draft_probs), qdt, uniforms.data_ptr(), noise.data_ptr(), tokens.data_ptr(), accepted.data_ptr(),
        ws.data_ptr(), ws.numel(), _lib.stream_of(logits)), "speculative.verify")
    return tokens, accepted


__all__ = ["verify"]
