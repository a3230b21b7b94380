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

import ctypes

import torch

from . import _lib


def _cache(k_pages, v_pages, block_table, lens):
    """The library's view of a cache, and lens checked against it."""
    _lib.require_cuda(k_pages, v_pages, block_table, lens)
    if k_pages.ndim != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages must be 4D [pages, kv_heads, page_size, dim] of one shape, got "
                         f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if v_pages.dtype is not k_pages.dtype:
        raise ValueError(f"k_pages {k_pages.dtype} and v_pages {v_pages.dtype} must have one dtype")
    dt = _lib.dtype_code(k_pages)
    if dt == _lib.I32:
        raise NotImplementedError("a cache holds bfloat16 or float32")
    if block_table.ndim != 2 or block_table.dtype is not torch.int32 or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous int32 [batch, table_width] tensor")
    batch, width = block_table.shape
    _int_rows("lens", lens, batch)
    pages, heads, page_size, dim = k_pages.shape
    kp, kh, ks, kd = k_pages.stride()
    vp, vh, vs, vd = v_pages.stride()
    if dim > 1 and (kd != 1 or vd != 1):
        raise ValueError("the dim elements of a slot must be contiguous")
    return _lib.KvCache(k_pages.data_ptr(), v_pages.data_ptr(), dt, dim, pages, heads, page_size, kp, kh, ks, vp, vh, vs,
                        block_table.data_ptr(), batch, width)


def _int_rows(name, t, batch):
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.shape != (batch,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape ({batch},)")


def _per_slot(name, t, c, dtype):
    shape = (c.batch, c.kv_heads, c.table_width * c.page_size)
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape}")


def append(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
           k_new: torch.Tensor, v_new: torch.Tensor, *, counts: torch.Tensor | None = None,
           scores: torch.Tensor | None = None, positions: torch.Tensor | None = None,
           seen: torch.Tensor | None = None) -> torch.Tensor:
    """Writes new keys and values behind each sequence, in place, and returns the new lens.

    k_new, v_new [batch, tokens, kv_heads, dim] in the cache's dtype; counts
    [batch] int32: how many of `tokens` each sequence has (default: all).
    Tokens past the table's capacity, or whose page the table does not name,
    are dropped.  With scores, positions and seen ([batch] int32: tokens of the
    text so far) the written slots get score 0 and position seen + t.
    """
    c = _cache(k_pages, v_pages, block_table, lens)
    _lib.require_cuda(k_pages, k_new, v_new)
    if k_new.ndim != 4 or k_new.shape != v_new.shape or k_new.shape[0] != c.batch or k_new.shape[2] != c.kv_heads \
            or k_new.shape[3] != c.dim:
        raise ValueError(f"k_new and v_new must be [{c.batch}, tokens, {c.kv_heads}, {c.dim}], got "
                         f"{tuple(k_new.shape)} and {tuple(v_new.shape)}")
    if k_new.dtype is not k_pages.dtype or v_new.dtype is not k_pages.dtype:
        raise ValueError(f"k_new and v_new must be {k_pages.dtype}, as the cache")
    if (scores is None) != (positions is None) or (scores is not None and seen is None):
        raise ValueError("scores, positions and seen go together")
    if scores is not None:
        _lib.require_cuda(k_pages, scores, positions, seen)
        _per_slot("scores", scores, c, torch.float32)
        _per_slot("positions", positions, c, torch.int32)
        _int_rows("seen", seen, c.batch)
    if counts is not None:
        _lib.require_cuda(k_pages, counts)
        _int_rows("counts", counts, c.batch)
    k_new, v_new = _aligned(k_new), _aligned(v_new)
    out = torch.empty_like(lens)
    _lib.check(_lib.LIB.tallax_kv_append(
        ctypes.byref(c), lens.data_ptr(), _lib.ptr(counts), k_new.data_ptr(), v_new.data_ptr(), k_new.shape[1],
        _lib.ptr(scores), _lib.ptr(positions), _lib.ptr(seen) if scores is not None else None, out.data_ptr(),
        _lib.stream_of(lens)), "kvcache.append")
    return out


def _aligned(x):
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


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
    (default: what the table can hold); the length is split by it, and lens
    above it are taken as max_len.  workspace: a uint8 device tensor used
    instead of the shared per-device buffer.
    """
    c = _cache(k_pages, v_pages, block_table, lens)
    _lib.require_cuda(k_pages, q)
    if q.ndim != 4 or q.shape[0] != c.batch or q.shape[3] != c.dim:
        raise ValueError(f"q must be [{c.batch}, queries, heads, {c.dim}], got {tuple(q.shape)}")
    if q.dtype is not k_pages.dtype:
        raise ValueError(f"q must be {k_pages.dtype}, as the cache, got {q.dtype}")
    _, queries, heads, dim = q.shape
    if counts is not None:
        _lib.require_cuda(k_pages, counts)
        _int_rows("counts", counts, c.batch)
    if scores is None:
        if out_scores is not None:
            raise ValueError("out_scores without scores")
    else:
        _lib.require_cuda(k_pages, scores)
        _per_slot("scores", scores, c, torch.float32)
        if out_scores is None:
            out_scores = torch.empty_like(scores)
        else:
            _lib.require_cuda(k_pages, out_scores)
            _per_slot("out_scores", out_scores, c, torch.float32)
    capacity = c.table_width * c.page_size
    max_len = capacity if max_len is None else int(max_len)
    es = q.element_size()
    if q.stride(3) != 1 or q.data_ptr() % 16 or any(s < 0 or s * es % 16 for s in q.stride()[:3]):
        q = q.clone(memory_format=torch.contiguous_format)
    qb, qt, qh, _ = q.stride()
    out = torch.empty((c.batch, queries, heads, dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((c.batch, queries, heads), dtype=torch.float32, device=q.device)
    need = _lib.LIB.tallax_kv_decode_workspace_size(ctypes.byref(c), queries, heads, max_len, scores is not None)
    ws = _lib.workspace_arg(workspace, q.device, need) if need else None
    _lib.check(_lib.LIB.tallax_kv_decode(
        ctypes.byref(c), q.data_ptr(), qb, qt, qh, queries, heads, dim ** -0.5 if scale is None else float(scale),
        lens.data_ptr(), _lib.ptr(counts), max_len, _lib.ptr(scores), out.data_ptr(), lse.data_ptr(),
        _lib.ptr(out_scores), _lib.ptr(ws), ws.numel() if need else 0, _lib.stream_of(q)), "kvcache.decode")
    return (out, lse) if scores is None else (out, lse, out_scores)


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
    must not exceed budget.
    """
    c = _cache(k_pages, v_pages, block_table, lens)
    _lib.require_cuda(k_pages, scores, positions, seen)
    _per_slot("scores", scores, c, torch.float32)
    _per_slot("positions", positions, c, torch.int32)
    _int_rows("seen", seen, c.batch)
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    new_lens, new_scores, new_positions = torch.empty_like(lens), torch.empty_like(scores), torch.empty_like(positions)
    need = _lib.LIB.tallax_kv_evict_workspace_size(ctypes.byref(c), min(max(budget, 1), c.table_width * c.page_size))
    ws = _lib.workspace_arg(workspace, lens.device, max(need, 1))
    _lib.check(_lib.LIB.tallax_kv_evict(
        ctypes.byref(c), lens.data_ptr(), scores.data_ptr(), positions.data_ptr(), seen.data_ptr(), budget, recent,
        sinks, new_lens.data_ptr(), new_scores.data_ptr(), new_positions.data_ptr(), ws.data_ptr(), ws.numel(),
        _lib.stream_of(lens)), "kvcache.evict")
    return new_lens, new_scores, new_positions


__all__ = ["append", "decode", "evict"]
