"""Workloads of one layer's step in a serving loop: keys written to a paged cache with their positions'
rotation, attention of a batch that shares a prefix, and the choice of experts.

`run` makes one pass through an operator.  With `own` false it computes the operator's definition from
elementary torch operations; with `own` true it makes the calls of tallax_amd.kvcache and
tallax_amd.experts.

Layouts: caches [pages, kv_heads, page, dim]; block_table [batch, table] int32, entries past a
sequence's last page are -1; lens [batch] int32 counts the slots in use; queries, keys and values of new
tokens [batch, tokens, heads, dim], parts of one projection's output."""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


def listed():
    return [
        # one interactive user's next token, few heads: all latency
        {"name": "rotate one", "op": "rotate", "batch": 1, "tokens": 1, "heads": 8, "kv_heads": 2, "dim": 64,
         "pairs": 32, "page": 16, "longest": 200, "dtype": "bf16", "axes": 0, "interleaved": False},
        # one new token for each sequence of a batch
        {"name": "rotate step", "op": "rotate", "batch": 64, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "pairs": 64, "page": 16, "longest": 4096, "dtype": "bf16", "axes": 0, "interleaved": False},
        # chunks of long prompts, far into the text
        {"name": "rotate prompt", "op": "rotate", "batch": 4, "tokens": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
         "pairs": 64, "page": 64, "longest": 131071, "dtype": "bf16", "axes": 0, "interleaved": False},
        # frames of a video with places in time, height and width; part of each head is rotated, neighbours in pairs
        {"name": "rotate video", "op": "rotate", "batch": 3, "tokens": 2501, "heads": 12, "kv_heads": 12, "dim": 80,
         "pairs": 30, "page": 24, "longest": 8192, "dtype": "f32", "axes": 3, "interleaved": True},
        # a few users of one short instruction, few heads
        {"name": "shared short", "op": "shared", "prompts": 1, "batch": 4, "queries": 1, "heads": 8, "kv_heads": 2, "dim": 64,
         "page": 16, "prefix": 500, "longest": 100, "dtype": "bf16"},
        # a batch of chats behind one long instruction
        {"name": "shared batch", "op": "shared", "prompts": 1, "batch": 64, "queries": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "prefix": 8192, "longest": 1024, "dtype": "bf16"},
        # questions about one long document
        {"name": "shared long", "op": "shared", "prompts": 1, "batch": 16, "queries": 1, "heads": 64, "kv_heads": 8,
         "dim": 128, "page": 64, "prefix": 131071, "longest": 300, "dtype": "bf16"},
        # a large batch, drafted tokens to be verified: products of matrices
        {"name": "shared drafted", "op": "shared", "prompts": 1, "batch": 128, "queries": 5, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 32, "prefix": 4099, "longest": 700, "dtype": "bf16"},
        # three samples of each of three prompts; float32, a head per query head, pages that are no power of two
        {"name": "shared f32", "op": "shared", "prompts": 3, "batch": 9, "queries": 1, "heads": 12, "kv_heads": 12,
         "dim": 80, "page": 24, "prefix": 2050, "longest": 333, "dtype": "f32"},
        # one token through a small router
        {"name": "route one", "op": "route", "tokens": 1, "experts": 64, "k": 6, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_score": "max", "renormalise": True, "dtype": "bf16"},
        # a decoding batch, experts in groups, a bias that balances them
        {"name": "route batch", "op": "route", "tokens": 130, "experts": 256, "k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_score": "top2", "renormalise": True, "dtype": "f32"},
        # the tokens of long prompts
        {"name": "route prompts", "op": "route", "tokens": 16384, "experts": 256, "k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "group_score": "top2", "renormalise": True, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "shared", "shared", "shared", "route", "route"])
    if op == "route":
        experts = rng.choice([8, 16, 32, 60, 64, 128, 160, 256, 256, 384, 512])
        groups = rng.choice([1, 1, 4, 4]) if experts < 64 else rng.choice([1, 1, 4, 4 if experts == 60 else 8])
        top = rng.randint(1, groups)
        c = {"op": op, "tokens": _log_int(rng, 1, 16384), "experts": experts,
             "k": rng.randint(1, min(16, experts // groups * top)), "score": rng.choice(["softmax", "sigmoid"]),
             "bias": rng.random() < 0.5, "groups": groups, "top_groups": top,
             "group_score": rng.choice(["max", "top2"]), "renormalise": rng.random() < 0.7,
             "dtype": rng.choice(["bf16", "f32"])}
        while c["tokens"] * experts > 16384 * 256:
            c["tokens"] //= 2
        return c
    dtype = rng.choice(["bf16", "bf16", "f32"])
    c = {"op": op, "batch": _log_int(rng, 1, 128), "kv_heads": rng.choice([1, 2, 4, 5, 8, 16]),
         "dim": rng.choice([64, 80, 96, 128, 128, 192, 256]), "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 256]),
         "dtype": dtype}
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 7, 8, 8])
    if op == "rotate":
        c["pairs"] = rng.choice([c["dim"] // 2, c["dim"] // 2, c["dim"] // 4, rng.randint(1, c["dim"] // 2)])
        c["tokens"] = rng.choice([1, rng.randint(2, 9), _log_int(rng, 9, 8192)])
        c["longest"] = _log_int(rng, 33, 131071)
        c["axes"], c["interleaved"] = rng.choice([0, 0, 1, 3]), rng.random() < 0.3
        most = 16384 * 48 * 128 // (_SIZE[dtype] // 2)
        while c["batch"] * c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] > most:
            if c["batch"] > 1:
                c["batch"] //= 2
            else:
                c["tokens"] //= 2
        most = 4 * 131071 * 8 * 128 // (_SIZE[dtype] // 2)  # the pool
        while c["batch"] * (c["longest"] + c["tokens"]) * c["kv_heads"] * c["dim"] > most:
            c["longest"] = max(c["longest"] // 2, 1)
            if c["longest"] == 1 and c["batch"] > 1:
                c["batch"] //= 2
        return c
    c["queries"] = rng.choice([1, 1, 1, rng.randint(2, 9)])
    c["prefix"], c["longest"] = _log_int(rng, 33, 131071), _log_int(rng, 1, 4096)
    c["longest"] = max(c["longest"], c["queries"])
    c["prompts"] = rng.choice([1, 1, 1, 2, 3, 8])
    size = c["dim"] * (1 if dtype == "bf16" else 4)
    while c["batch"] * c["queries"] * c["heads"] * (c["prefix"] + c["longest"]) * size > 16 * 64 * 131071 * 128 or \
            (c["batch"] * c["longest"] + c["prompts"] * c["prefix"]) * c["kv_heads"] * size > 131071 * 8 * 128:
        if c["batch"] > 1:
            c["batch"] //= 2
        else:
            c["prefix"], c["prompts"] = max(c["prefix"] // 2, 1), 1
    c["prompts"] = min(c["prompts"], c["batch"])
    c["batch"] -= c["batch"] % c["prompts"]
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _lens(c):
    """Lengths of the sequences' own parts, spread from the longest down to a quarter of it; in a batch of
    8 or more the last place of the attention's is idle (length 0, no query)."""
    b, longest = c["batch"], c["longest"]
    lens = [longest - (3 * longest // 4) * i // b for i in range(b)]
    if b >= 8 and c["op"] == "shared":
        lens[-1] = 0
    return lens


def _prefix_lens(c):
    return [c["prefix"] - c["prefix"] // 2 * i // c["prompts"] for i in range(c["prompts"])]


def _randn(gen, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=_DT[dtype], device="cuda")
    return x.normal_(0.0, scale, generator=gen)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"op": c["op"]}
    if c["op"] == "route":
        return _prepare_route(c, gen, s)
    b, ps, hkv = c["batch"], c["page"], c["kv_heads"]
    order = torch.randperm(b, generator=gen, device="cuda")
    lens = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")[order].contiguous()
    new = c["tokens"] if c["op"] == "rotate" else 0
    width = -(-(c["longest"] + new) // ps)
    prompts = c["prompts"] if c["op"] == "shared" else 0
    front = -(-c["prefix"] // ps) if c["op"] == "shared" else 0
    pages = b * width + prompts * front + 2
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = perm[:b * width].reshape(b, width)
    used = (lens + new + ps - 1) // ps
    s["table"] = torch.where(torch.arange(width, device="cuda")[None] < used[:, None], table, -1).to(torch.int32)
    s["k"], s["v"] = (_randn(gen, (pages, hkv, ps, c["dim"]), c["dtype"]) for _ in range(2))
    s["lens"] = lens
    if c["op"] == "shared":
        t = c["queries"]
        begins = torch.tensor(_prefix_lens(c), dtype=torch.int32, device="cuda")
        at = perm[b * width:b * width + prompts * front].reshape(prompts, front)
        used = (begins + ps - 1) // ps
        s["prefix"] = torch.where(torch.arange(front, device="cuda")[None] < used[:, None], at, -1).to(torch.int32)
        s["prefix_lens"] = begins
        s["q"] = _randn(gen, (b, t, c["heads"], c["dim"]), c["dtype"], 2.0)
        s["scale"] = c["dim"] ** -0.5
        n = torch.randint(1, t + 1, (b,), generator=gen, device="cuda")  # some have fewer drafted tokens
        s["counts"] = torch.minimum(n, lens.long()).to(torch.int32)
        return s
    heads, t = c["heads"], c["tokens"]
    qkv = _randn(gen, (b, t, heads + 2 * hkv, c["dim"]), c["dtype"], 2.0)
    s["q"], s["k_new"], s["v_new"] = qkv[:, :, :heads], qkv[:, :, heads:heads + hkv], qkv[:, :, heads + hkv:]
    pairs = c["pairs"]
    f = 1000000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    s["frequencies"], s["interleaved"] = f.float(), c["interleaved"]
    s["positions"], s["pair_axes"] = None, None
    if c["axes"] == 1:  # the text goes on from where each sequence is, after what has been evicted
        away = torch.randint(0, 1000000, (b, 1), generator=gen, device="cuda")
        s["positions"] = (away + torch.arange(t, device="cuda")).to(torch.int32)
    elif c["axes"] == 3:  # frames of 20 by 36 patches, behind the text
        i = torch.arange(t, device="cuda")
        grid = torch.stack([i // 720, i % 720 // 36, i % 36], -1)
        s["positions"] = (grid[None] + lens[:, None, None]).to(torch.int32).contiguous()
        s["pair_axes"] = (torch.arange(pairs, device="cuda") % 3).to(torch.int32)
    return s


def _prepare_route(c, gen, s):
    s["logits"] = _randn(gen, (c["tokens"], c["experts"]), c["dtype"], 1.5)
    s["bias"] = None
    if c["bias"]:  # what balancing has come to
        s["bias"] = torch.empty(c["experts"], device="cuda").normal_(0.0, 0.05, generator=gen)
    s["k"] = c["k"]
    s["how"] = {n: c[n] for n in ("score", "groups", "top_groups", "group_score", "renormalise")}
    s["how"]["scale"] = 2.5 if c["score"] == "sigmoid" else 1.0
    return s


def run(state):
    s = state
    if own:
        return _run_own(s)
    return {"rotate": _rotate, "shared": _shared, "route": _route}[s["op"]](s)


def _run_own(s):
    from tallax_amd import experts, kvcache
    if s["op"] == "rotate":
        lens, q = kvcache.append_rotated(s["k"], s["v"], s["table"], s["lens"], s["q"], s["k_new"], s["v_new"],
                                         s["frequencies"], token_positions=s["positions"], pair_axes=s["pair_axes"],
                                         interleaved=s["interleaved"])
        return s["k"], s["v"], lens, q
    if s["op"] == "shared":
        return kvcache.decode_shared(s["q"], s["k"], s["v"], s["prefix"], s["prefix_lens"], s["table"],
                                     s["lens"], scale=s["scale"], counts=s["counts"])
    return experts.route(s["logits"], s["k"], bias=s["bias"], **s["how"])


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _rotate(s):
    """Writes the values and the rotated keys behind each sequence; the rotated queries.  Angles in 64 bits."""
    table, q = s["table"], s["q"]
    b, t, _, d = q.shape
    pages, _, ps, _ = s["k"].shape
    step = torch.arange(t, device=q.device)
    slot = s["lens"][:, None] + step
    at = slot if s["positions"] is None else s["positions"]
    f = s["frequencies"].double()
    pairs = f.shape[0]
    at = at[..., s["pair_axes"].long()] if s["pair_axes"] is not None else at[..., None].expand(b, t, pairs)
    angle = at.double() * f
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    low = slice(0, 2 * pairs, 2) if s["interleaved"] else slice(0, pairs)
    high = slice(1, 2 * pairs, 2) if s["interleaved"] else slice(pairs, 2 * pairs)

    def turned(x):
        y = x.float().clone()
        x0, x1 = y[..., low].clone(), y[..., high].clone()
        y[..., low] = x0 * cos - x1 * sin
        y[..., high] = x1 * cos + x0 * sin
        return y.to(x.dtype)

    page = table.gather(1, (slot // ps).clamp(max=table.shape[1] - 1)).long()
    fits = (slot < table.shape[1] * ps) & (page >= 0) & (page < pages)
    i, j = fits.nonzero(as_tuple=True)
    page, slot = page[i, j], slot[i, j].long()
    s["k"][page, :, slot % ps] = turned(s["k_new"])[i, j]
    s["v"][page, :, slot % ps] = s["v_new"][i, j]
    return s["k"], s["v"], (s["lens"] + t).clamp(max=table.shape[1] * ps), turned(q)


def _slots(s, table, lens, limit):
    """Keys and values [hkv, rows of table, slots, d] in float32, and which slots each of limit [rows, n] sees."""
    pages, _, ps, _ = s["k"].shape
    slot = torch.arange(table.shape[1] * ps, device=table.device)
    page = table[:, slot // ps].long()
    held = (page >= 0) & (page < pages) & (slot < lens[:, None])
    page, off = page.clamp(0, pages - 1), slot % ps
    k, v = (c[page, :, off].permute(2, 0, 1, 3).float() for c in (s["k"], s["v"]))
    return k, v.masked_fill(~held[..., None], 0.0), held[:, None] & (slot < limit[..., None])


def _shared(s):
    """Softmax attention over a prefix, which all queries of its sequences see, and each sequence's own slots: query t
    of counts[b] sees those below lens[b] - counts[b] + t + 1.  Sequences b of one prefix follow one another."""
    q, lens, counts = s["q"], s["lens"], s["counts"]
    b, t, hq, d = q.shape
    hkv, prompts = s["k"].shape[1], s["prefix"].shape[0]
    g = hq // hkv
    step = torch.arange(t, device=q.device)
    rows = q.float().reshape(b, t, hkv, g, d).permute(2, 0, 1, 3, 4).reshape(hkv, b, t * g, d)
    whole = s["prefix_lens"][:, None]
    kp, vp, seen = _slots(s, s["prefix"], s["prefix_lens"], whole)
    x = (rows.reshape(hkv, prompts, -1, d) @ kp.transpose(-1, -2)) * s["scale"]
    x = x.masked_fill(~seen, -math.inf).reshape(hkv, b, t * g, -1)
    limit = torch.minimum(lens[:, None] - counts[:, None] + step + 1, lens[:, None])
    ko, vo, seen = _slots(s, s["table"], lens, limit)
    y = (rows @ ko.transpose(-1, -2)) * s["scale"]
    y = y.masked_fill(~seen.repeat_interleave(g, 1)[None], -math.inf)
    top = torch.maximum(x.amax(-1, keepdim=True), y.amax(-1, keepdim=True))
    base = top.masked_fill(top == -math.inf, 0.0)
    x, y = (x - base).exp(), (y - base).exp()
    total = x.sum(-1, keepdim=True) + y.sum(-1, keepdim=True)
    out = (x.reshape(hkv, prompts, b // prompts * t * g, -1) @ vp).reshape(hkv, b, t * g, d) + y @ vo
    out = out / total.masked_fill(total == 0, 1.0)
    lse = (top + total.log()).masked_fill(total == 0, -math.inf)
    none = (step >= counts[:, None]).repeat_interleave(g, 1)[None, ..., None]  # a query that does not count
    out, lse = out.masked_fill(none, 0.0), lse.masked_fill(none, -math.inf)
    out = out.reshape(hkv, b, t, g, d).permute(1, 2, 0, 3, 4).reshape(b, t, hq, d)
    return out.to(q.dtype), lse.reshape(hkv, b, t, g).permute(1, 2, 0, 3).reshape(b, t, hq).contiguous()


def _route(s):
    """The k experts of the largest scores plus bias, of the groups that are ranked first; their scores.  In 64 bits:
    a whole number hangs on each comparison."""
    x, how = s["logits"].double(), s["how"]
    tokens, experts = x.shape
    if how["score"] == "softmax":
        e = (x - x.amax(-1, keepdim=True)).exp()
        score = e / e.sum(-1, keepdim=True)
    else:
        score = 1.0 / (1.0 + (-x).exp())
    key = score if s["bias"] is None else score + s["bias"].double()
    if how["groups"] > 1:
        by_group = key.reshape(tokens, how["groups"], -1)
        best = by_group.sort(dim=-1, descending=True)[0]
        n = 2 if how["group_score"] == "top2" and best.shape[-1] > 1 else 1
        first = best[..., :n].sum(-1).argsort(dim=-1, descending=True, stable=True)[:, :how["top_groups"]]
        kept = (torch.arange(how["groups"], device=x.device)[:, None] == first[:, None]).any(-1)
        key = by_group.masked_fill(~kept[..., None], -math.inf).reshape(tokens, experts)
    ids = key.argsort(dim=-1, descending=True, stable=True)[:, :s["k"]]
    w = score.gather(-1, ids)
    if how["renormalise"]:
        w = w / w.sum(-1, keepdim=True)
    return (w * how["scale"]).float(), ids.to(torch.int32)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its values in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "route":
        n = c["tokens"] * c["experts"]
        return {"bytes": n * _SIZE[c["dtype"]] + c["tokens"] * c["k"] * 8, "flops": 4 * n}
    es = _SIZE[c["dtype"]]
    if c["op"] == "rotate":
        n = c["batch"] * c["tokens"]
        return {"bytes": 2 * n * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] * es,
                "flops": 6 * n * (c["heads"] + c["kv_heads"]) * c["pairs"]}
    begins = sum(_prefix_lens(c))
    slots = begins + sum(_lens(c))
    rows = c["batch"] * c["queries"] * c["heads"]
    flops = 4 * c["dim"] * c["queries"] * c["heads"] * (c["batch"] // c["prompts"] * begins + sum(_lens(c)))
    return {"bytes": 2 * c["kv_heads"] * c["dim"] * es * slots + 2 * rows * c["dim"] * es + 4 * rows, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "shared": _exact_shared, "route": _exact_route}[case["op"]](s)


def _exact_rotate(s):
    """Turned as complex numbers, one sequence at a time; values are only moved."""
    pools, q = s["k"].double(), s["q"]
    b, t, _, d = q.shape
    ps, n = pools.shape[2], s["frequencies"].shape[0]
    out = q.double()
    for i in range(b):
        place = torch.arange(t, device="cuda", dtype=torch.int64) + int(s["lens"][i])
        p = place if s["positions"] is None else s["positions"][i].long()
        p = p[:, s["pair_axes"].long()] if p.dim() == 2 else p[:, None]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), p * s["frequencies"].double())
        done = []
        for x in (q[i].double(), s["k_new"][i].double()):
            if s["interleaved"]:
                z = torch.complex(x[..., 0:2 * n:2].contiguous(), x[..., 1:2 * n:2].contiguous()) * turn[:, None]
                first = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * turn[:, None]
                first = torch.cat([z.real, z.imag], -1)
            done.append(torch.cat([first, x[..., 2 * n:]], -1))
        out[i] = done[0]
        pools[s["table"][i].long()[place // ps], :, place % ps] = done[1]
    return pools, None, None, out


def _exact_shared(s):
    """One sequence and kv head at a time, over its prefix and its own slots as one list."""
    b, t, hq, d = s["q"].shape
    _, hkv, ps, _ = s["k"].shape
    g, prompts = hq // hkv, s["prefix"].shape[0]
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((b, t, hq), -math.inf, dtype=torch.float64, device="cuda")
    lens, counts, begins = s["lens"].tolist(), s["counts"].tolist(), s["prefix_lens"].tolist()
    for h in range(hkv):
        for i, (n, c) in enumerate(zip(lens, counts)):
            at = i // (b // prompts)
            p = begins[at]
            if i % (b // prompts) == 0:
                ids = s["prefix"][at, :-(-p // ps)].long()
                front = [x[ids, h].reshape(-1, d)[:p].double() for x in (s["k"], s["v"])]
            if c == 0:
                continue
            ids = s["table"][i, :-(-n // ps)].long()
            k, v = (torch.cat([f, x[ids, h].reshape(-1, d)[:n].double()]) for f, x in zip(front, (s["k"], s["v"])))
            q = s["q"][i, :c, h * g:(h + 1) * g].reshape(c * g, d).double()
            x = torch.mm(q, k.t().contiguous()) * s["scale"]
            ends = torch.arange(p + n - c + 1, p + n + 1, device="cuda").repeat_interleave(g)
            x[torch.arange(p + n, device="cuda")[None] >= ends[:, None]] = -math.inf
            z = torch.logsumexp(x, -1)
            out[i, :c, h * g:(h + 1) * g] = torch.mm(torch.exp(x - z[:, None]), v).reshape(c, g, d)
            lse[i, :c, h * g:(h + 1) * g] = z.reshape(c, g)
    return out, lse


def _first_of_largest(x):
    n = x.shape[-1]
    return torch.where(x == x.amax(-1, keepdim=True), torch.arange(n, device=x.device), n).amin(-1)


def _exact_route(s):
    """Groups and experts picked one after another, as the largest of those that are left."""
    x, how = s["logits"].double(), s["how"]
    tokens, experts = x.shape
    score = torch.softmax(x, -1) if how["score"] == "softmax" else torch.sigmoid(x)
    key = score.clone() if s["bias"] is None else score + s["bias"].double()
    row = torch.arange(tokens, device="cuda")
    size = experts // how["groups"]
    if how["groups"] > 1:
        rank = key.reshape(tokens, how["groups"], size).topk(min(2, size), -1)[0]
        rank = rank.sum(-1) if how["group_score"] == "top2" else rank[..., 0].clone()
        open_ = torch.zeros((tokens, how["groups"]), dtype=torch.bool, device="cuda")
        for _ in range(how["top_groups"]):
            first = _first_of_largest(rank)
            open_[row, first] = True
            rank[row, first] = -math.inf
        key[~open_.repeat_interleave(size, -1)] = -math.inf
    ids = torch.zeros((tokens, s["k"]), dtype=torch.int64, device="cuda")
    for j in range(s["k"]):
        ids[:, j] = _first_of_largest(key)
        key[row, ids[:, j]] = -math.inf
    w = score[row[:, None], ids]
    if how["renormalise"]:
        w = w / w.sum(-1, keepdim=True)
    return w * how["scale"], ids.to(torch.int32)
