"""Workloads of the serving-step operators: a paged key-value cache (append, attention, eviction) and
the verification of drafted tokens.

`run` makes one pass through an operator.  With `own` false it computes the operator's definition from
elementary torch operations; with `own` true it makes the calls of tallax_amd.kvcache and
tallax_amd.speculative.

Layouts: caches [pages, kv_heads, page, dim]; block_table [batch, table] int32, entries past a
sequence's last page are -1; lens [batch] int32 counts the slots in use; scores and positions
[batch, kv_heads, table * page]."""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


def listed():
    return [
        # one interactive user, a short chat, few heads: all latency
        {"name": "decode one short", "op": "decode", "batch": 1, "queries": 1, "heads": 8, "kv_heads": 2, "dim": 64,
         "page": 16, "longest": 200, "dtype": "bf16", "scores": False},
        # a batch of chats at ordinary lengths, their weights added up for a later eviction
        {"name": "decode batch", "op": "decode", "batch": 64, "queries": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "longest": 4096, "dtype": "bf16", "scores": True},
        # few users with long documents: the length has to be split
        {"name": "decode long", "op": "decode", "batch": 4, "queries": 1, "heads": 64, "kv_heads": 8, "dim": 128,
         "page": 64, "longest": 131071, "dtype": "bf16", "scores": False},
        # the target's pass over four drafted tokens and the one before them
        {"name": "decode drafted", "op": "decode", "batch": 32, "queries": 5, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "longest": 8191, "dtype": "bf16", "scores": True},
        # float32, a head per query head, pages that are no power of two
        {"name": "decode f32", "op": "decode", "batch": 9, "queries": 1, "heads": 12, "kv_heads": 12, "dim": 80,
         "page": 24, "longest": 2050, "dtype": "f32", "scores": True},
        # one new token for each sequence of a batch: a scatter that is all latency
        {"name": "append step", "op": "append", "batch": 64, "queries": 1, "kv_heads": 8, "dim": 128, "page": 16,
         "longest": 4096, "dtype": "bf16"},
        # a chunk of a prompt written behind what is there
        {"name": "append chunk", "op": "append", "batch": 8, "queries": 2047, "kv_heads": 8, "dim": 128, "page": 64,
         "longest": 16384, "dtype": "bf16"},
        # every few steps of a running batch: a few tokens over the budget go
        {"name": "evict running", "op": "evict", "batch": 64, "kv_heads": 8, "dim": 128, "page": 16, "longest": 2176,
         "budget": 2048, "dtype": "bf16", "fresh": False},
        # after a long prompt: most of it goes
        {"name": "evict prompt", "op": "evict", "batch": 8, "kv_heads": 8, "dim": 128, "page": 64, "longest": 32768,
         "budget": 4095, "dtype": "bf16", "fresh": True},
        # one user, a small vocabulary
        {"name": "verify one", "op": "verify", "batch": 1, "drafted": 3, "vocab": 32000, "dtype": "bf16",
         "draft": "probs", "greedy": 0},
        # a serving batch at the sampler's vocabulary, the draft model's probabilities at hand
        {"name": "verify batch", "op": "verify", "batch": 64, "drafted": 4, "vocab": 128256, "dtype": "bf16",
         "draft": "probs", "greedy": 0},
        # drafts looked up in the text (no probabilities), some rows greedy, float32 logits, an odd vocabulary
        {"name": "verify lookup", "op": "verify", "batch": 130, "drafted": 7, "vocab": 151937, "dtype": "f32",
         "draft": "tokens", "greedy": 3},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "append", "evict", "verify", "verify"])
    if op == "verify":
        batch, drafted, vocab = _log_int(rng, 1, 256), rng.randint(1, 8), _log_int(rng, 1000, 202000)
        while batch * (drafted + 1) * vocab > 130 * 8 * 151937:
            batch = max(1, batch // 2)
        return {"op": op, "batch": batch, "drafted": drafted, "vocab": vocab, "dtype": rng.choice(["bf16", "f32"]),
                "draft": rng.choice(["probs", "probs", "tokens"]), "greedy": rng.choice([0, 0, 2, 5])}
    dtype = rng.choice(["bf16", "bf16", "f32"])
    c = {"op": op, "batch": _log_int(rng, 1, 128), "kv_heads": rng.choice([1, 2, 4, 5, 8, 16]),
         "dim": rng.choice([64, 80, 96, 128, 128, 192, 256]), "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 256]),
         "longest": _log_int(rng, 33, 131071), "dtype": dtype}
    most = (4 if op == "decode" else 1) * 131071 * 8 * 128 // (_SIZE[dtype] // 2)
    while c["batch"] * c["longest"] * c["kv_heads"] * c["dim"] > most:
        if c["batch"] > 1:
            c["batch"] //= 2
        else:
            c["longest"] //= 2
    if op == "decode":
        c["queries"] = rng.choice([1, 1, 1, rng.randint(2, 9)])
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 7, 8, 8])
        c["scores"] = rng.random() < 0.5
        while c["batch"] * c["longest"] * c["heads"] * c["queries"] > 4 * 131071 * 64:
            if c["batch"] > 1:
                c["batch"] //= 2
            else:
                c["longest"] //= 2
    elif op == "append":
        c["queries"] = rng.choice([1, rng.randint(2, 9), _log_int(rng, 9, max(10, c["longest"] // 2))])
    else:
        c["fresh"] = rng.random() < 0.5
        c["budget"] = max(1, c["longest"] // 8 if c["fresh"] else c["longest"] - rng.randint(1, 1 + c["longest"] // 16))
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _lens(c):
    """Lengths of the sequences, longest first, spread down to a quarter of it; in a batch of 8 or more
    the last place is idle (length 0), as in a serving loop whose batch is not full."""
    b, longest = c["batch"], c["longest"]
    if c["op"] == "evict" and not c["fresh"]:  # all of them a little over the budget
        return [longest - (longest - c["budget"]) * i // b for i in range(b)]
    lens = [longest - (3 * longest // 4) * i // b for i in range(b)]
    if b >= 8 and c["op"] == "decode":
        lens[-1] = 0
    return lens


def _randn(gen, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=_DT[dtype], device="cuda")
    return x.normal_(0.0, scale, generator=gen)


def _cache(c, gen, lens):
    b, ps = c["batch"], c["page"]
    width = -(-c["longest"] // ps)
    if c["op"] == "append":
        width = -(-(c["longest"] + c["queries"]) // ps)
    pages = b * width + 2
    table = torch.randperm(pages, generator=gen, device="cuda")[:b * width].reshape(b, width).to(torch.int32)
    used = (lens + ps - 1) // ps
    if c["op"] == "append":
        used = (lens + c["queries"] + ps - 1) // ps
    table = torch.where(torch.arange(width, device="cuda")[None] < used[:, None], table, -1).to(torch.int32)
    shape = (pages, c["kv_heads"], ps, c["dim"])
    return _randn(gen, shape, c["dtype"]), _randn(gen, shape, c["dtype"]), table.contiguous()


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"op": c["op"]}
    if c["op"] == "verify":
        return _prepare_verify(c, gen, s)
    order = torch.randperm(c["batch"], generator=gen, device="cuda")
    lens = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")[order].contiguous()
    s["k"], s["v"], s["table"] = _cache(c, gen, lens)
    s["lens"], b, hkv = lens, c["batch"], c["kv_heads"]
    slots = s["table"].shape[1] * c["page"]
    if c["op"] == "decode":
        t = c["queries"]
        s["q"] = _randn(gen, (b, t, c["heads"], c["dim"]), c["dtype"], 2.0)
        s["scale"] = c["dim"] ** -0.5
        s["counts"] = None
        if t > 1:  # sequences with fewer drafted tokens than the longest draft
            n = torch.randint(1, t + 1, (b,), generator=gen, device="cuda")
            s["counts"] = torch.minimum(n, lens.long()).to(torch.int32)
        s["scores"] = None
        if c["scores"]:
            s["scores"] = torch.empty((b, hkv, slots), device="cuda").uniform_(0.0, 1.0, generator=gen)
    elif c["op"] == "append":
        shape = (b, c["queries"], hkv, c["dim"])
        s["k_new"], s["v_new"] = _randn(gen, shape, c["dtype"]), _randn(gen, shape, c["dtype"])
        s["scores"] = torch.empty((b, hkv, slots), device="cuda").uniform_(0.0, 1.0, generator=gen)
        s["positions"] = torch.arange(slots, dtype=torch.int32, device="cuda").expand(b, hkv, slots).contiguous()
        s["seen"] = lens + 1000
    else:
        # weights that attention leaves behind: a few tokens have most of it, the newest have had none yet
        w = torch.empty((b, hkv, slots), device="cuda").normal_(0.0, 2.0, generator=gen).exp_()
        at = torch.arange(slots, device="cuda").expand(b, hkv, slots)
        s["scores"] = torch.where(at == lens[:, None, None] - 1, 0.0, w)
        if c["fresh"]:  # nothing has been evicted yet: slots are in the order of the text
            s["positions"], s["seen"] = at.to(torch.int32).contiguous(), lens.clone()
        else:  # earlier evictions have left the slots of each head in an order of its own
            mix = torch.rand((b, hkv, slots), generator=gen, device="cuda").argsort(-1) * 3
            s["positions"] = torch.where(at < c["budget"], mix, 3 * slots + at).to(torch.int32)
            s["seen"] = 3 * slots + lens
        s["budget"] = c["budget"]
        s["recent"], s["sinks"] = c["budget"] // 4, min(4, c["budget"] // 2)
    return s


def _prepare_verify(c, gen, s):
    b, t, v, dt = c["batch"], c["drafted"], c["vocab"], _DT[c["dtype"]]
    s["logits"] = _randn(gen, (b, t + 1, v), c["dtype"], 3.0)
    s["temperature"] = torch.empty(b, device="cuda").uniform_(0.6, 1.2, generator=gen)
    if c["greedy"]:
        s["temperature"][torch.arange(b, device="cuda") % c["greedy"] == 0] = 0.0
    # the draft model is near the target: its logits are the target's with noise
    near = s["logits"][:, :t].float().add_(torch.empty((b, t, v), device="cuda").normal_(0.0, 0.6, generator=gen))
    probs = near.div_(s["temperature"].clamp(min=0.3)[:, None, None]).softmax(-1)
    del near
    race = torch.empty((b, t, v), device="cuda").exponential_(1.0, generator=gen).clamp_(min=1e-20)
    s["draft"] = (probs / race).argmax(-1).to(torch.int32)
    s["probs"] = probs if c["draft"] == "probs" else None
    s["uniforms"] = torch.rand((b, t), generator=gen, device="cuda")
    s["noise"] = torch.empty((b, v), device="cuda").exponential_(1.0, generator=gen).clamp_(min=1e-20)
    counts = torch.full((b,), t, dtype=torch.int32, device="cuda")
    if b > 4:  # some sequences were given fewer drafts, one of them none
        counts[::3] = torch.randint(0, t + 1, (len(range(0, b, 3)),), generator=gen, device="cuda").to(torch.int32)
    s["counts"] = counts
    return s


def run(state):
    s = state
    if own:
        return _run_own(s)
    return {"decode": _decode, "append": _append, "evict": _evict, "verify": _verify}[s["op"]](s)


def _run_own(s):
    from tallax_amd import kvcache, speculative
    if s["op"] == "decode":
        return kvcache.decode(s["q"], s["k"], s["v"], s["table"], s["lens"], scale=s["scale"], counts=s["counts"],
                              scores=s["scores"])
    if s["op"] == "append":
        lens = kvcache.append(s["k"], s["v"], s["table"], s["lens"], s["k_new"], s["v_new"], scores=s["scores"],
                              positions=s["positions"], seen=s["seen"])
        return s["k"], s["v"], lens, s["scores"], s["positions"]
    if s["op"] == "evict":
        lens, scores, positions = kvcache.evict(s["k"], s["v"], s["table"], s["lens"], s["scores"], s["positions"],
                                                s["seen"], budget=s["budget"], recent=s["recent"], sinks=s["sinks"])
        return s["k"], s["v"], lens, scores, positions
    return speculative.verify(s["draft"], s["logits"], s["uniforms"], s["noise"], draft_probs=s["probs"],
                              temperature=s["temperature"], counts=s["counts"])


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _gather(pages, page, off):
    """[batch, kv_heads, slots, dim] in float32 of a cache, from each slot's page and place in it."""
    return pages[page, :, off].permute(0, 2, 1, 3).float()


def _decode(s):
    """Softmax attention of the newest tokens: query t of sequence b sees the slots below
    lens[b] - counts[b] + t + 1; slots whose page is no page of the pool are seen by none."""
    q, k_pages, table = s["q"], s["k"], s["table"]
    b, t, hq, d = q.shape
    pages, hkv, ps, _ = k_pages.shape
    slot = torch.arange(table.shape[1] * ps, device=q.device)
    page = table[:, slot // ps].long()
    there = (page >= 0) & (page < pages)
    page, off = page.clamp(0, pages - 1), slot % ps
    counts = s["counts"] if s["counts"] is not None else torch.full_like(s["lens"], t)
    step = torch.arange(t, device=q.device)
    limit = torch.where(step < counts[:, None], s["lens"][:, None] - counts[:, None] + step + 1, 0)  # [b, t]
    seen = there[:, None] & (slot < limit[..., None]) & (slot < s["lens"][:, None, None])  # [b, t, slots]
    seen = seen[:, None, :, None]
    qg = q.float().reshape(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * (hq // hkv), d)
    x = (qg @ _gather(k_pages, page, off).transpose(-1, -2)) * s["scale"]
    x = x.reshape(b, hkv, t, hq // hkv, -1).masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = (x - top.masked_fill(top == -math.inf, 0.0)).exp()
    total = e.sum(-1, keepdim=True)
    w = e / total.masked_fill(total == 0, 1.0)
    v = _gather(s["v"], page, off)
    v = v.masked_fill(~seen.any(2).reshape(b, 1, -1, 1), 0.0)
    out = w.reshape(b, hkv, t * (hq // hkv), -1) @ v
    out = out.reshape(b, hkv, t, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d)
    lse = (top + total.log()).masked_fill(total == 0, -math.inf)[..., 0].permute(0, 2, 1, 3).reshape(b, t, hq)
    if s["scores"] is None:
        return out.to(q.dtype), lse
    return out.to(q.dtype), lse, s["scores"] + w.sum((2, 3))


def _append(s):
    k_new, table = s["k_new"], s["table"]
    b, t, hkv, _ = k_new.shape
    pages, _, ps, _ = s["k"].shape
    slot = s["lens"][:, None] + torch.arange(t, device=k_new.device)
    page = table.gather(1, (slot // ps).clamp(max=table.shape[1] - 1)).long()
    fits = (slot < table.shape[1] * ps) & (page >= 0) & (page < pages)
    at, step = fits.nonzero(as_tuple=True)
    page, slot = page[at, step], slot[at, step].long()
    s["k"][page, :, slot % ps] = k_new[at, step]
    s["v"][page, :, slot % ps] = s["v_new"][at, step]
    s["scores"][at, :, slot] = 0.0
    s["positions"][at, :, slot] = (s["seen"][at] + step).to(torch.int32)[:, None]
    lens = (s["lens"] + t).clamp(max=table.shape[1] * ps)
    return s["k"], s["v"], lens, s["scores"], s["positions"]


def _evict(s):
    """Keeps `budget` slots of each head: those of the first `sinks` and the last `recent` positions, then the
    largest scores (NaN last, ties: the lowest slot).  Kept slots below the new length stay; the others move, in order,
    into the places that became free."""
    scores, positions, table = s["scores"], s["positions"], s["table"]
    pages, hkv, ps, _ = s["k"].shape
    slots = scores.shape[-1]
    slot = torch.arange(slots, device=scores.device)
    lens = s["lens"][:, None, None]
    new = lens.clamp(max=s["budget"])
    kept_always = (positions < s["sinks"]) | (positions >= s["seen"][:, None, None] - s["recent"])
    key = torch.nan_to_num(scores.double(), nan=-2e300, posinf=1e300, neginf=-1e300)
    key = torch.where(slot < lens, torch.where(kept_always, 2e300, key), -math.inf)
    rank = key.argsort(dim=-1, descending=True, stable=True).argsort(-1)
    keep = rank < new
    hole, mover = ~keep & (slot < new), keep & (slot >= new)
    movers = (~mover).to(torch.int8).argsort(dim=-1, stable=True)
    source = torch.where(hole, movers.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), slot)
    held = slot < new
    new_scores = torch.where(held, scores.gather(-1, source), 0.0)
    new_positions = torch.where(held, positions.gather(-1, source), -1)
    b, h, to = hole.nonzero(as_tuple=True)
    frm = source[b, h, to]
    p_to, p_from = table[b, to // ps].long(), table[b, frm // ps].long()
    fits = ((p_to >= 0) & (p_to < pages) & (p_from >= 0) & (p_from < pages)).nonzero()[:, 0]
    h, p_to, p_from, to, frm = h[fits], p_to[fits], p_from[fits], to[fits], frm[fits]
    s["k"][p_to, h, to % ps] = s["k"][p_from, h, frm % ps]
    s["v"][p_to, h, to % ps] = s["v"][p_from, h, frm % ps]
    return s["k"], s["v"], new[:, 0, 0].contiguous(), new_scores, new_positions


def _first_of_largest(x):
    v = x.shape[-1]
    at = torch.arange(v, device=x.device)
    return torch.where(x == x.amax(-1, keepdim=True), at, v).amin(-1)


def _verify(s):
    """Draft i is accepted while u * q(x) < p(x) (greedy rows: while x is the largest logit); the next token is
    drawn from max(p - q, 0) of the first row that was not accepted, or from p after the last draft, as the
    largest weight / noise.  In 64 bits: a whole number hangs on each comparison."""
    draft, logits = s["draft"], s["logits"].double()
    b, t1, v = logits.shape
    t = t1 - 1
    greedy = s["temperature"] < 1e-5
    best = _first_of_largest(logits)
    tau = torch.where(greedy, 1.0, s["temperature"].double())[:, None, None]
    e = ((logits - logits.amax(-1, keepdim=True)) / tau).exp()
    one = (torch.arange(v, device=draft.device) == best[..., None]).double()
    p = torch.where(greedy[:, None, None], one, e)
    p = p / p.sum(-1, keepdim=True)
    known = (draft >= 0) & (draft < v)
    x = draft.long().clamp(0, v - 1)[..., None]
    px = torch.where(known, p[:, :t].gather(-1, x)[..., 0], 0.0)
    qx = s["probs"].gather(-1, x)[..., 0].double() if s["probs"] is not None else torch.ones_like(px)
    ok = torch.where(greedy[:, None], px > 0, s["uniforms"].double() * qx < px)
    ok &= torch.arange(t, device=draft.device) < s["counts"][:, None]
    n = ok.to(torch.int32).cumprod(-1).sum(-1)
    rows = torch.arange(b, device=draft.device)
    row, last = p[rows, n], (n == s["counts"])[:, None]
    at = n.clamp(max=t - 1)
    q = s["probs"][rows, at].double() if s["probs"] is not None else \
        (torch.arange(v, device=draft.device) == draft[rows, at][:, None]).double()
    rest = torch.where(last | greedy[:, None], row, (row - q).clamp(min=0.0))
    rest = torch.where(rest.amax(-1, keepdim=True) > 0, rest, row)
    token = _first_of_largest(rest / torch.where(greedy[:, None], 1.0, s["noise"].double()))
    step = torch.arange(t1, device=draft.device)
    padded = torch.cat([draft, draft.new_full((b, 1), -1)], 1)
    tokens = torch.where(step < n[:, None], padded, torch.where(step == n[:, None], token[:, None], -1))
    return tokens.to(torch.int32), n.to(torch.int32)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its values in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "verify":
        rows = c["batch"] * (c["drafted"] + 1)
        chosen = c["batch"] * c["vocab"] * (8 if c["draft"] == "probs" else 4)
        return {"bytes": rows * c["vocab"] * _SIZE[c["dtype"]] + chosen, "flops": 3 * rows * c["vocab"]}
    es, lens = _SIZE[c["dtype"]], _lens(c)
    line = c["kv_heads"] * c["dim"] * es  # one token's keys, or values, of all heads
    if c["op"] == "append":
        n = c["batch"] * c["queries"]
        return {"bytes": n * (4 * line + 8 * c["kv_heads"]), "flops": 0}
    if c["op"] == "evict":
        width = -(-c["longest"] // c["page"]) * c["page"]
        # about new / len of the slots past the budget stay, and take the places of others
        moved = sum((n - c["budget"]) * c["budget"] / n for n in lens if n > c["budget"])
        return {"bytes": int(c["kv_heads"] * (8 * sum(lens) + 8 * c["batch"] * width) + 4 * line * moved), "flops": 0}
    kv = 2 * line * sum(lens)
    io = 2 * c["batch"] * c["queries"] * c["heads"] * c["dim"] * es
    extra = 8 * c["kv_heads"] * sum(lens) if c["scores"] else 0
    return {"bytes": kv + io + extra, "flops": 4 * c["queries"] * c["heads"] * c["dim"] * sum(lens)}


def exact(case, seed):
    if case["op"] != "decode":
        return None  # moved values and whole numbers: held to be equal
    s = prepare(case, seed)
    b, t, hq, d = s["q"].shape
    pages, hkv, ps, _ = s["k"].shape
    g = hq // hkv
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((b, t, hq), -math.inf, dtype=torch.float64, device="cuda")
    scores = None if s["scores"] is None else s["scores"].double()
    for i, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        c = t if s["counts"] is None else int(s["counts"][i])
        ids = s["table"][i, :-(-n // ps)].long()
        for h in range(hkv):
            k = s["k"][ids, h].reshape(-1, d)[:n].double()
            v = s["v"][ids, h].reshape(-1, d)[:n].double()
            q = s["q"][i, :c, h * g:(h + 1) * g].reshape(c * g, d).double()
            x = torch.mm(q, k.t().contiguous()) * s["scale"]
            ends = torch.arange(n - c + 1, n + 1, device="cuda").repeat_interleave(g)
            x[torch.arange(n, device="cuda")[None] >= ends[:, None]] = -math.inf
            z = torch.logsumexp(x, -1)
            w = torch.exp(x - z[:, None])
            out[i, :c, h * g:(h + 1) * g] = torch.mm(w, v).reshape(c, g, d)
            lse[i, :c, h * g:(h + 1) * g] = z.reshape(c, g)
            if scores is not None:
                scores[i, h, :n] += w.sum(0)
    return (out, lse) if scores is None else (out, lse, scores)
