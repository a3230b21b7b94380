"""Plain 64-bit forms of the serving-step operators (kvcache, speculative) on the host, one sequence, head and
query at a time, and the inputs that their GPU tests share."""
import math

import numpy as np
import torch


def make_cache(rng, batch, kv_heads, dim, page, width, lens, dtype, fill=None, spare=3):
    """(k, v [pages, kv_heads, page, dim], table [batch, width]) on the host.  Pages are in no order; entries past a
    sequence's last page are -1.  fill: the value of every slot that no sequence uses."""
    pages = batch * width + spare
    perm = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int32)
    used = -(-np.asarray(lens) // page)
    table = np.where(np.arange(width)[None] < used[:, None], perm, -1).astype(np.int32)
    pools = []
    for _ in range(2):
        x = torch.from_numpy(rng.standard_normal((pages, kv_heads, page, dim)).astype(np.float32)).to(dtype)
        if fill is not None:
            keep = torch.zeros((pages, page), dtype=torch.bool)
            for b, n in enumerate(lens):
                for s in range(int(n)):
                    keep[int(table[b, s // page]), s % page] = True
            x = torch.where(keep[:, None, :, None], x, torch.tensor(fill, dtype=dtype))
        pools.append(x)
    return pools[0], pools[1], torch.from_numpy(table)


def slots_of(pool, table_row, n, page):
    """[n, kv_heads, dim] in float64 of one sequence, and which of the slots lie in a page of the pool."""
    ids = table_row[torch.arange(n) // page].long()
    there = (ids >= 0) & (ids < pool.shape[0])
    x = pool[ids.clamp(0, pool.shape[0] - 1), :, torch.arange(n) % page].double()
    return x, there


def attention(q, k, v, table, lens, scale, counts=None, scores=None):
    """(out, lse, scores, room) of kvcache.decode.  room: how far the device's out, lse and added weights may be off,
    from the roundings of its types (see below)."""
    b, t, hq, d = q.shape
    _, hkv, page, _ = k.shape
    g = hq // hkv
    half = torch.finfo(q.dtype).eps / 2
    f32 = torch.finfo(torch.float32).eps / 2
    out = torch.zeros((b, t, hq, d), dtype=torch.float64)
    lse = torch.full((b, t, hq), -math.inf, dtype=torch.float64)
    out_room, lse_room = torch.zeros_like(out), torch.zeros_like(lse)
    new = None if scores is None else scores.double().clone()
    new_room = None if scores is None else scores.double().abs() * f32
    for i in range(b):
        n = int(lens[i])
        c = t if counts is None else max(0, min(int(counts[i]), t))
        if n == 0:
            continue
        ks, there = slots_of(k, table[i], n, page)
        vs, _ = slots_of(v, table[i], n, page)
        for j in range(c):
            end = min(n, n - c + j + 1)
            see = torch.nonzero(there[:max(end, 0)])[:, 0]
            if see.numel() == 0:
                continue
            for h in range(hq):
                kk, vv, qq = ks[see, h // g], vs[see, h // g], q[i, j, h].double()
                x = (kk * qq).sum(-1) * scale
                z = torch.logsumexp(x, 0)
                w = torch.exp(x - z)
                out[i, j, h], lse[i, j, h] = (w[:, None] * vv).sum(0), z
                # a score: dim products added in float32 (dim + 1 roundings of at most the sum of their sizes), the
                # scale and its own rounding; in base 2 the exponent's difference is rounded again, exp2 and the
                # weights' sum add a few more, and lse takes a logarithm
                dx = float(((kk.abs() * qq.abs()).sum(-1) * abs(scale)).max()) * (d + 4) * f32 + 4 * f32 * float(x.abs().max())
                dw = 2 * dx + 16 * f32 + 8 * f32 * math.log2(see.numel() + 1)
                size = (w[:, None] * vv.abs()).sum(0)
                # bfloat16 weights are rounded before their product with the values, and out to its type
                out_room[i, j, h] = half * out[i, j, h].abs() * 1.01 + size * ((half if q.dtype == torch.bfloat16 else 0) + 2 * dw)
                # the rounding of out is a half step of what it lies at, not of the exact value
                out_room[i, j, h] += size * half * ((half if q.dtype == torch.bfloat16 else 0) + 2 * dw)
                lse_room[i, j, h] = dw + 4 * f32 * abs(float(z)) + 4 * f32
                if new is not None:
                    new[i, h // g, see] += w
                    new_room[i, h // g, see] += w * (dw + lse_room[i, j, h]) + 4 * f32 * new[i, h // g, see].abs()
    return out, lse, new, (out_room, lse_room, new_room)


def evict(k, v, table, lens, scores, positions, seen, budget, recent, sinks):
    """(k, v, lens, scores, positions) after kvcache.evict, by sorting."""
    k, v = k.clone(), v.clone()
    batch, heads, slots = scores.shape
    page = k.shape[2]
    new_lens = torch.minimum(lens, torch.tensor(budget, dtype=torch.int32)).to(torch.int32)
    new_scores, new_positions = torch.zeros_like(scores), torch.full_like(positions, -1)
    for b in range(batch):
        n, m = int(lens[b]), int(new_lens[b])
        for h in range(heads):
            def key(s):
                p, x = int(positions[b, h, s]), float(scores[b, h, s])
                always = p < sinks or p >= int(seen[b]) - recent
                return (0, s) if always else (2, s) if math.isnan(x) else (1, -x, s)
            keep = set(sorted(range(n), key=key)[:m])
            holes = [s for s in range(m) if s not in keep]
            movers = sorted(s for s in keep if s >= m)
            assert len(holes) == len(movers)
            source = {s: s for s in range(m)}
            source.update(zip(holes, movers))
            for to, frm in source.items():
                new_scores[b, h, to], new_positions[b, h, to] = scores[b, h, frm], positions[b, h, frm]
                pt, pf = int(table[b, to // page]), int(table[b, frm // page])
                if to != frm and 0 <= pt < k.shape[0] and 0 <= pf < k.shape[0]:
                    k[pt, h, to % page] = k[pf, h, frm % page]
                    v[pt, h, to % page] = v[pf, h, frm % page]
    return k, v, new_lens, new_scores, new_positions


def verify(draft, logits, uniforms, noise, probs=None, temperature=None, counts=None):
    """(tokens, accepted) of speculative.verify; every argument a numpy array (logits and probs float64 values of
    the device's), with the margin of the closest comparison, relative to the larger side."""
    batch, rows, vocab = logits.shape
    drafted = rows - 1
    tokens = np.full((batch, rows), -1, np.int32)
    accepted = np.zeros(batch, np.int32)
    margin = math.inf
    for b in range(batch):
        t = float(temperature[b])
        cnt = drafted if counts is None else int(np.clip(counts[b], 0, drafted))
        greedy = np.float32(t) < np.float32(1e-5)

        def p_of(i):
            l = np.where(np.isnan(logits[b, i]), -np.inf, np.minimum(logits[b, i], np.finfo(np.float32).max))
            m = l.max()
            if m == -np.inf:
                return np.zeros(vocab)
            if greedy:
                e = np.zeros(vocab)
                e[int(l.argmax())] = 1
                return e
            with np.errstate(over="ignore"):
                e = np.exp((l - m) / t)
            return e / e.sum()

        n = 0
        while n < cnt:
            x = int(draft[b, n])
            p = p_of(n)[x] if 0 <= x < vocab else 0.0
            if greedy:
                ok = p > 0
            else:
                q = 1.0 if probs is None else float(probs[b, n, x]) if 0 <= x < vocab else 0.0
                a = float(uniforms[b, n]) * q
                ok = a < p
                if p > 0 or a > 0:
                    margin = min(margin, abs(a - p) / max(a, p))
            if not ok:
                break
            n += 1
        p = p_of(n)
        r = p
        if n < cnt and not greedy:
            if probs is not None:
                q = probs[b, n]
            else:
                q = np.zeros(vocab)
                if 0 <= draft[b, n] < vocab:
                    q[draft[b, n]] = 1
            r = np.maximum(p - q, 0)
            if r.max() == 0:
                r = p
        s = r if greedy else r / noise[b].astype(np.float64)
        tokens[b, :n] = draft[b, :n]
        if s.max() > 0:
            tokens[b, n] = int(s.argmax())
            if vocab > 1 and not greedy:
                two = np.partition(s, -2)[-2:]
                margin = min(margin, float((two[1] - two[0]) / two[1]))
        accepted[b] = n
    return tokens, accepted, margin
