"""Paged key-value cache: appending tokens, the attention of the newest ones, and
eviction by accumulated attention weight.

No counterpart in the reference, which begins at the logits; these are the steps
of a serving loop before them.  Every call runs hand-written gfx950 kernels
(include/tallax_hip.h: tallax_kv_append, tallax_kv_decode, tallax_kv_evict).

A cache is two pools of pages k_pages, v_pages [pages, kv_heads, page_size, dim]
(bfloat16 or float32; dim a multiple of 8 up to 256, contiguous; any strides of
the first three axes that are multiples of 16 bytes, so a pool laid out [pages,
page_size, kv_heads, dim] is passed as its transpose(1, 2)), a block_table
[batch, table_width] int32 that names the page of every page_size slots of a
sequence, and lens [batch] int32, the slots in use.  An entry that is no page
of the pool (-1) holds nothing: its slots are neither written nor seen.

scores and positions [batch, kv_heads, table_width * page_size] (float32, int32)
go with a cache that evicts: the attention weight each slot has gathered, and
the place in the text of the token it holds.
"""
from __future__ import annotations

import torch

from . import _lib


def append(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
           k_new: torch.Tensor, v_new: torch.Tensor, *, counts: torch.Tensor | None = None,
           scores: torch.Tensor | None = None, positions: torch.Tensor | None = None,
           seen: torch.Tensor | None = None) -> torch.Tensor:
    """Writes new keys and values behind each sequence, in place, and returns the new lens.

    k_new, v_new [batch, tokens, kv_heads, dim] in the cache's dtype; counts
    [batch] int32: how many of `tokens` each sequence has (default: all).  New
    keys and values that are not contiguous are copied first.  Tokens past the
    table's capacity, or whose page the table does not name, are dropped.  With
    scores, positions and seen ([batch] int32: tokens of the text so far) the
    written slots get score 0 and position seen + t.
    """
    return _lib.SERVING.append(k_pages, v_pages, block_table, lens, k_new, v_new, counts, scores, positions, seen)


def decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
           lens: torch.Tensor, *, scale: float | None = None, counts: torch.Tensor | None = None,
           scores: torch.Tensor | None = None, out_scores: torch.Tensor | None = None, max_len: int | None = None,
           workspace: torch.Tensor | None = None):
    """Attention of each sequence's newest tokens over its cache.

    q [batch, queries, heads, dim] in the cache's dtype, heads a multiple of
    kv_heads (head h reads kv head h // (heads // kv_heads)); queries is 1 for
    ordinary decoding, more for the tokens of a draft.  The tokens' own keys
    and values are in the cache already (append): query t of counts[b] (int32,
    default: queries) sees slots below lens[b] - counts[b] + t + 1, queries
    from counts[b] on see none.  Returns (out [batch, queries, heads, dim], lse
    [batch, queries, heads] float32 = log of the sum of exp(scale q.k)); a
    query that sees nothing gives 0 and -inf.

    With scores, returns (out, lse, new_scores): scores plus the weights that
    each slot got, summed over the queries and the heads of its kv head.
    out_scores: a buffer for them (may be scores itself); a new one by default.

    scale: default dim ** -0.5.  max_len: a bound on lens known to the caller
    (default: what the table can hold); the length is split by it, the
    workspace grows with it where there are scores, and lens above it are taken
    as max_len.  A table much wider than its sequences needs it: 4 sequences of
    4096 slots in one of 131072 take 54 us without it and 16 with it.  workspace: a uint8 device tensor that
    begins on a multiple of 16 bytes, used instead of the shared per-device
    buffer.
    """
    return _lib.SERVING.decode(q, k_pages, v_pages, block_table, lens, scale, counts, scores, out_scores, max_len,
                               workspace)


def evict(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
          scores: torch.Tensor, positions: torch.Tensor, seen: torch.Tensor, *, budget: int, recent: int = 0,
          sinks: int = 0, workspace: torch.Tensor | None = None):
    """Cuts every sequence to at most `budget` slots per kv head.

    Each head keeps the tokens of the first `sinks` and the last `recent`
    positions of the text (seen [batch] int32: its length so far), then those of
    the largest scores (NaN last), ties to the lowest slot.  Kept slots below
    the new length stay where they are; the others move into the places that
    became free, both in ascending order.  Keys and values are moved in place
    and only as many as that takes; returns (new_lens, new_scores,
    new_positions), new tensors, with 0 and -1 in the slots from the new length
    on.  Sequences of at most `budget` slots are left alone.  recent + sinks
    must not exceed budget.  workspace: as decode's.
    """
    return _lib.SERVING.evict(k_pages, v_pages, block_table, lens, scores, positions, seen, budget, recent, sinks,
                              workspace)


__all__ = ["append", "decode", "evict"]
