"""Plain 64-bit forms of the operators of one layer's step (kvcache.append_rotated, kvcache.decode_shared,
experts.route) on the host, with how far the device's results may be off from the roundings of its types."""
import math

import numpy as np
import torch

F32 = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, at, frequencies, pair_axes=None, interleaved=False):
    """(rotated x, room): x [tokens, heads, dim] of any float type, at [tokens] or [tokens, axes] whole numbers."""
    n = frequencies.shape[0]
    f = frequencies.double()
    p = at.double()
    p = p[:, None].expand(-1, n) if pair_axes is None else p[:, pair_axes.long().clamp(0, at.shape[1] - 1)]
    angle = (p * f)[:, None]
    c, s = angle.cos(), angle.sin()
    low = torch.arange(n) * 2 if interleaved else torch.arange(n)
    high = low + (1 if interleaved else n)
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    x0, x1 = x[..., low].double(), x[..., high].double()
    y[..., low], y[..., high] = x0 * c - x1 * s, x1 * c + x0 * s
    # cos and sin: their angle (64 bits: 2^-50 of itself and more, here and there), the series (2^-40), their rounding to
    # float32 and then two products and a sum in float32, of at most |x0| + |x1|; and the result's own rounding
    off = angle.abs() * 2.0 ** -49 + 2.0 ** -39 + 4 * F32
    size[..., low] = size[..., high] = (x0.abs() + x1.abs()) * off
    room = size * (1 + 2.0 ** -7)
    if x.dtype != torch.float32:
        turned = torch.zeros(x.shape[-1])
        turned[low], turned[high] = 1, 1
        # bfloat16's smallest step is 2^-133
        room = room + (y.abs() * half_step(x.dtype) * (1 + 2.0 ** -7) + 2.0 ** -134) * turned
    return y, room + 2.0 ** -149 * (room > 0)


def append_rotated(k, v, table, lens, q, k_new, v_new, frequencies, token_positions=None, pair_axes=None,
                   interleaved=False, counts=None, seen=None):
    """(k, v, lens, q) in 64 bits and room for k and q."""
    batch, tokens, _, _ = q.shape
    page, slots = k.shape[2], table.shape[1] * k.shape[2]
    out_k, out_v, out_q = k.double().clone(), v.double().clone(), torch.zeros(q.shape, dtype=torch.float64)
    room_k, room_q = torch.zeros(k.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    new = lens.clone()
    for b in range(batch):
        n = tokens if counts is None else max(0, min(int(counts[b]), tokens))
        start = int(lens[b])
        at = torch.arange(tokens) + (start if seen is None else int(seen[b]))
        if token_positions is not None:
            at = token_positions[b]
        out_q[b, :n], room_q[b, :n] = rotate(q[b, :n], at[:n], frequencies, pair_axes, interleaved)
        turned, room = rotate(k_new[b, :n], at[:n], frequencies, pair_axes, interleaved)
        for t in range(n):
            if start + t >= slots:
                continue
            to = int(table[b, (start + t) // page])
            if 0 <= to < k.shape[0]:
                out_k[to, :, (start + t) % page], room_k[to, :, (start + t) % page] = turned[t], room[t]
                out_v[to, :, (start + t) % page] = v_new[b, t].double()
        new[b] = min(start + n, slots)
    return out_k, out_v, new, out_q, room_k, room_q


def slots_of(pool, table_row, n, page):
    ids = table_row[torch.arange(n) // page].long()
    there = (ids >= 0) & (ids < pool.shape[0])
    return pool[ids.clamp(0, pool.shape[0] - 1), :, torch.arange(n) % page].double()[there], there


def shared_attention(q, k, v, prefix_table, prefix_lens, table, lens, scale, counts=None):
    """(out, lse, room of out, room of lse) of kvcache.decode_shared."""
    b, t, hq, d = q.shape
    _, hkv, page, _ = k.shape
    g, per = hq // hkv, b // prefix_table.shape[0]
    half = half_step(q.dtype)
    low = half if q.dtype == torch.bfloat16 else 0.0  # weights are rounded to bfloat16 before their product
    out = torch.zeros((b, t, hq, d), dtype=torch.float64)
    lse = torch.full((b, t, hq), -math.inf, dtype=torch.float64)
    out_room, lse_room = torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(b):
        p = i // per
        kp, _ = slots_of(k, prefix_table[p], int(prefix_lens[p]), page)
        vp, _ = slots_of(v, prefix_table[p], int(prefix_lens[p]), page)
        n = int(lens[i])
        c = t if counts is None else max(0, min(int(counts[i]), t))
        for j in range(c):
            end = max(0, min(n, n - c + j + 1))
            ko, _ = slots_of(k, table[i], end, page)
            vo, _ = slots_of(v, table[i], end, page)
            kk, vv = torch.cat([kp, ko]), torch.cat([vp, vo])  # [slots, hkv, d]
            m = kk.shape[0]
            if m == 0:
                continue
            qq = q[i, j].double().reshape(hkv, g, d).transpose(0, 1)  # [g, hkv, d]
            x = (qq[:, None] * kk[None]).sum(-1) * scale  # [g, m, hkv]
            z = torch.logsumexp(x, 1)
            w = torch.exp(x - z[:, None])
            o = (w[..., None] * vv[None]).sum(1)
            size = (w[..., None] * vv[None].abs()).sum(1)
            # a score: dim products added in float32 (dim + 1 roundings of at most the sum of their sizes), the scale and
            # its own rounding; in base 2 the exponent's difference is rounded again, exp2 and the weights' sum add a few
            # more (a sum in pieces of chunks: log2 of the slots, at least), and lse takes a logarithm
            dx = ((qq[:, None].abs() * kk[None].abs()).sum(-1) * abs(scale)).amax(1) * (d + 4) * F32 + 4 * F32 * x.abs().amax(1)
            dw = 2 * dx + 32 * F32 + 8 * F32 * math.log2(m + 1)
            r = half * o.abs() * 1.01 + size * (low + 2 * dw[..., None]) * (1 + half)
            out[i, j], out_room[i, j] = o.transpose(0, 1).reshape(hq, d), r.transpose(0, 1).reshape(hq, d)
            lse[i, j] = z.t().reshape(hq)
            lse_room[i, j] = (dw + 4 * F32 * z.abs() + 4 * F32).t().reshape(hq)
    return out, lse, out_room, lse_room


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=None, group_score="max", renormalise=True, scale=1.0):
    """(weights, ids, margin) by sorting, in 64 bits.  logits: float64 values of the device's.  margin: the least distance
    of two different computed values that a choice compared (logits, which are compared as they are, leave nothing open)."""
    tokens, experts = logits.shape
    top_groups = groups if top_groups is None else top_groups
    most = float(np.finfo(np.float32).max)
    weights, ids = np.zeros((tokens, k)), np.zeros((tokens, k), np.int32)
    margin = math.inf
    size = experts // groups
    for t in range(tokens):
        here = logits[t] > -np.inf
        x = np.where(here, np.minimum(logits[t], most), -most)
        with np.errstate(over="ignore"):
            if score == "softmax":
                e = np.where(here, np.exp(x - (x[here].max() if here.any() else 0.0)), 0.0)
                s = e / (e.sum() if e.sum() > 0 else 1.0)
            else:
                s = np.where(here, 1.0 / (1.0 + np.exp(-x)), 0.0)
        if bias is not None:
            here = here & ~np.isnan(bias)
            s = np.where(here, s, 0.0)
            key = s + np.clip(np.nan_to_num(bias, nan=0.0, posinf=most, neginf=-most), -most, most)
        else:
            key = s
        element = key if bias is not None else x
        open_ = np.ones(experts, bool)
        if groups > 1:
            ranks = []
            for gr in range(groups):
                at = slice(gr * size, (gr + 1) * size)
                use = element if group_score == "max" and bias is None else key
                best = sorted(use[at][here[at]], reverse=True)[:2 if group_score == "top2" else 1]
                ranks.append((len(best) > 0, sum(best)))
            order = sorted(range(groups), key=lambda i: (not ranks[i][0], -ranks[i][1], i))
            chosen = set(order[:top_groups])
            open_ = np.array([i // size in chosen for i in range(experts)])
            if group_score == "top2" or bias is not None:
                margin = min(margin, _closest([ranks[i][1] for i in order if ranks[i][0]]))
        order = sorted(np.nonzero(open_)[0], key=lambda i: (not here[i], -element[i] if here[i] else 0.0, i))
        if bias is not None:
            margin = min(margin, _closest([element[i] for i in order if here[i]][:k + 1]))
        ids[t] = order[:k]
        w = s[ids[t]]
        if renormalise:
            w = w / w.sum() if w.sum() > 0 else w * 0
        weights[t] = w * scale
    return weights, ids, margin


def _closest(values):
    """The least distance of neighbours that differ."""
    v = np.asarray(values)
    d = np.abs(np.diff(v))
    return float(d[d > 0].min()) if (d > 0).any() else math.inf
