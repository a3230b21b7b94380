"""GPU: each of kvcache.decode_shared's kernels and their instances, by tables that reach them (asserted), against
attention over both parts in 64 bits."""
import math

import numpy as np
import pytest
import torch

from tests import layer_ref as L
from tests import shared_paths as S
from tests.test_gpu_shared import _both, _check, _make, _run

pytestmark = pytest.mark.gpu


def _args(c, rng, lens, begins, fill=math.nan):
    """Inputs of the lengths, in tables of the case's width."""
    q, k, v, prefix, begins, table, lens = _make(rng, lens, begins, c.queries, c.group * c.kv_heads, c.kv_heads, c.dim,
                                                 c.page, c.dtype, fill=fill)

    def wide(t, width):
        pad = torch.full((t.shape[0], max(width - t.shape[1], 0)), -1, dtype=torch.int32)
        return torch.cat([t[:, :width], pad], 1).contiguous()

    assert c.plan()[:3] == [c.path, c.rg, c.mt]
    return q, k, v, wide(prefix, c.prefix_pages), begins, wide(table, c.own_pages), lens


def _lens(c, most=150):
    most = min(most, c.own_pages * c.page - c.queries)
    lens = [0 if i % 11 == 5 else c.queries + i * 37 % most for i in range(c.batch)]
    lens[0] = c.queries + most - 1
    return lens


def _begins(c, most=333):
    return [(min(most, c.prefix_pages * c.page), 70, 0, 1, 129)[i % 5] for i in range(c.prompts)]


@pytest.mark.parametrize("case", S.cases() + S.cases_of_pages() + S.cases_of_dims(), ids=repr)
def test_each_path(gpu, case):
    """Lengths of none, counts of none and too many, pages that are missing, unused slots of NaN; the same bits twice."""
    rng = np.random.default_rng(case.dim + case.batch)
    args = _args(case, rng, _lens(case), _begins(case))
    q, k, v, prefix, begins, table, own = args
    first = _both(gpu, args)
    assert all(torch.equal(a, b) for a, b in zip(first, _run(gpu, args), strict=True))
    counts = torch.from_numpy(rng.integers(-1, case.queries + 3, case.batch).astype(np.int32))
    table, prefix = table.clone(), prefix.clone()
    prefix[0, :2] = torch.tensor([-1, 99999], dtype=torch.int32)[:prefix.shape[1]]
    table[0, 0] = -1
    table[-1] = 99999
    _both(gpu, (q, k, v, prefix, begins, table, own), counts=counts)


@pytest.mark.parametrize("case", S.cases_of_many_rows(), ids=repr)
def test_the_most_rows(gpu, case):
    rng = np.random.default_rng(case.batch)
    args = _args(case, rng, [1300, 700][:case.batch], [70])
    _both(gpu, args)
    _both(gpu, args, counts=torch.tensor([1023, 5][:case.batch], dtype=torch.int32))


@pytest.mark.parametrize("case", [c for c in S.cases() if c.dim in (64, 192)], ids=repr)
def test_each_path_with_one_part(gpu, case):
    rng = np.random.default_rng(case.dim + case.batch)
    q, k, v, prefix, begins, table, own = _args(case, rng, _lens(case, 40), _begins(case, 100))
    _both(gpu, (q, k, v, prefix, begins * 0, table, own))
    _both(gpu, (q, k, v, prefix, begins, table, own * 0))
    out, lse = _both(gpu, (q, k, v, prefix, begins * 0, table, own * 0))
    assert not bool(out.any()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("case", [c for c in S.cases() if c.queries > 1 or c.dim == 128], ids=repr)
def test_each_path_with_values_that_are_not_finite(gpu, case):
    """A value reaches the queries that see its slot, and none else."""
    c = case
    rng = np.random.default_rng(c.dim)
    lens = [c.queries + 20] * c.batch
    lens[1 % c.batch] = 1  # its first queries see the prefix alone
    if c.own_pages * c.page < lens[0]:
        lens = [min(n, c.own_pages * c.page) for n in lens]
    args = _args(c, rng, lens, [min(100, c.prefix_pages * c.page)] * c.prompts)
    q, k, v, prefix, begins, table, own = args
    bad = torch.zeros(q.shape, dtype=torch.bool)
    per = c.batch // c.prompts

    def spoil(row, slot, kvh, d, value, where):
        v[int(row[slot // S.PAGE]), kvh, slot % S.PAGE, d] = value
        bad[where + (slice(kvh * c.group, (kvh + 1) * c.group), d)] = True

    p = c.prompts - 1
    every = slice(None)
    spoil(prefix[p], 97, c.kv_heads - 1, 5, math.inf, (slice(p * per, (p + 1) * per), every))
    spoil(table[0], lens[0] - 1, 0, c.dim - 1, math.nan, (slice(0, 1), slice(c.queries - 1, c.queries)))  # the newest slot
    last = c.batch - 1
    if last > 1:
        spoil(table[last], 0, 0, 7, -math.inf, (slice(last, last + 1), every))
        first = max(0, c.queries - 1)
        spoil(table[1], 0, c.kv_heads - 1, 3, math.inf, (slice(1, 2), slice(first, c.queries)))
    out, lse = _run(gpu, args)
    assert torch.equal(~torch.isfinite(out.cpu().float()), bad)
    assert bool(torch.isfinite(lse).all())


def _long(q, k, v, prefix, begins, table, lens, scale):
    """Attention in 64 bits on the card, a sequence's kv head at a time; every query counts.  (out, lse, room of out, room
    of lse): the rooms as layer_ref.shared_attention derives them."""
    b, t, hq, d = q.shape
    hkv, per = k.shape[1], b // prefix.shape[0]
    g = hq // hkv
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device=q.device)
    lse = torch.zeros((b, t, hq), dtype=torch.float64, device=q.device)
    out_room, lse_room = torch.zeros_like(out), torch.zeros_like(lse)
    half = L.half_step(q.dtype)
    low = half if q.dtype == torch.bfloat16 else 0.0
    for p in range(prefix.shape[0]):
        n = int(begins[p])
        at = torch.arange(n, device=q.device)
        for h in range(hkv):
            kp, vp = (x[prefix[p, at // S.PAGE].long(), h, at % S.PAGE].double() for x in (k, v))
            for i in range(p * per, (p + 1) * per):
                m = int(lens[i])
                own = torch.arange(m, device=q.device)
                ko, vo = (x[table[i, own // S.PAGE].long(), h, own % S.PAGE].double() for x in (k, v))
                kk, vv = torch.cat([kp, ko]), torch.cat([vp, vo])
                qq = q[i, :, h * g:(h + 1) * g].reshape(t * g, d).double()
                x = torch.mm(qq, kk.t().contiguous()) * scale
                dx = torch.mm(qq.abs(), kk.abs().t().contiguous()).amax(-1) * scale * (d + 4) * L.F32 + 4 * L.F32 * x.abs().amax(-1)
                dw = 2 * dx + 32 * L.F32 + 8 * L.F32 * math.log2(n + m + 1)
                ends = n + m - t + 1 + torch.arange(t, device=q.device).repeat_interleave(g)
                x[torch.arange(n + m, device=q.device)[None] >= ends[:, None]] = -math.inf
                z = torch.logsumexp(x, -1)
                w, at_h = torch.exp(x - z[:, None]), slice(h * g, (h + 1) * g)
                o, size = torch.mm(w, vv), torch.mm(w, vv.abs())
                room = half * o.abs() * 1.01 + size * (low + 2 * dw[:, None]) * (1 + half)
                out[i, :, at_h], out_room[i, :, at_h] = o.reshape(t, g, d), room.reshape(t, g, d)
                lse[i, :, at_h], lse_room[i, :, at_h] = z.reshape(t, g), (dw + 4 * L.F32 * z.abs() + 4 * L.F32).reshape(t, g)
    return out, lse, out_room, lse_room


@pytest.mark.parametrize("case", [c for c in S.cases() if c.dim == 128 and c.prompts <= 10], ids=repr)
def test_each_path_over_many_chunks(gpu, case):
    """Lengths that fill what the tables hold, or thousands of slots of it, so that every chunk has its part."""
    from tallax_amd import kvcache
    c = case
    # of the widest tables a few chunks
    most, longest = min(c.prefix_pages, 2600), min(c.own_pages, 60)
    gen = torch.Generator(device=gpu)
    gen.manual_seed(c.batch)
    pages = c.batch * longest + c.prompts * most
    k, v = (torch.randn((pages, c.kv_heads, S.PAGE, c.dim), generator=gen, device=gpu).to(c.dtype) for _ in range(2))
    q = torch.randn((c.batch, c.queries, c.group * c.kv_heads, c.dim), generator=gen, device=gpu).to(c.dtype)
    perm = torch.randperm(pages, generator=gen, device=gpu).to(torch.int32)
    prefix = torch.full((c.prompts, c.prefix_pages), -1, dtype=torch.int32, device=gpu)
    prefix[:, :most] = perm[:c.prompts * most].reshape(c.prompts, most)
    table = torch.full((c.batch, c.own_pages), -1, dtype=torch.int32, device=gpu)
    table[:, :longest] = perm[c.prompts * most:].reshape(c.batch, longest)
    begins = torch.tensor([most * S.PAGE - 7 - i for i in range(c.prompts)], dtype=torch.int32, device=gpu)
    lens = torch.tensor([max(c.queries, longest * S.PAGE - i * 13) for i in range(c.batch)], dtype=torch.int32, device=gpu)
    got = kvcache.decode_shared(q, k, v, prefix, begins, table, lens)
    _check(got, [x.cpu() for x in _long(q, k, v, prefix, begins, table, lens, c.dim ** -0.5)])
