"""Routing tokens to experts: scores of a router's logits, the choice of the
largest, and their weights.

No counterpart in the reference, whose top-k (`tax.top_k`) picks from values as
they are.  One call runs a hand-written gfx950 kernel (include/tallax_hip.h:
tallax_route).
"""
from __future__ import annotations

import torch

from . import _lib


def route(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
          top_groups: int | None = None, group_score: str = "max", renormalise: bool = True,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Chooses k experts for each token: (weights [tokens, k] float32, ids [tokens, k] int32).

    logits [tokens, experts] float32 or bfloat16 (rows at any stride), up to
    1024 experts; k up to 64.  A token's scores are the softmax of its logits
    or, with score="sigmoid", 1 / (1 + exp(-logit)).  bias [experts] float32 is
    added to the scores for the choice, not to the weights.

    With groups > 1 (up to 64, a divisor of experts; an expert's group is id //
    (experts // groups)) only the experts of the top_groups groups that rank
    first are open (default: all): by the largest score + bias in the group,
    or with group_score="top2" by the sum of the two largest.

    The k largest of score + bias are chosen, in descending order, all ties to
    the lowest id (without a bias by the logits themselves, which no rounding
    of the scores ties).  Comparisons are of 64-bit values.  Their weights are
    the scores, divided by their sum if renormalise (0 where it is 0), times
    scale, in 64 bits until they are rounded; a token's are the same whatever
    tokens are beside it.

    Experts whose logit is -inf or NaN, or whose bias is NaN, are not there:
    they score 0, add nothing to their group, and are chosen after all others
    of the open groups, lowest id first, with weight 0.  +inf logits and
    infinite biases count as the largest finite ones.
    """
    return _lib.SERVING.route(logits, k, score, bias, groups, top_groups, group_score, renormalise, scale)


__all__ = ["route"]
