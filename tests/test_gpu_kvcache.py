"""GPU: kvcache.append, decode and evict against plain 64-bit forms on the host: lengths from 0 and 1 up, pages that end inside a tile,
head layouts, ragged queries, places that nothing may read, pools past 4 GiB, streams and graphs."""
import numpy as np
import pytest
import torch

from tests import serving_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _bits(t):
    return t.contiguous().cpu().view(torch.int16 if t.dtype == torch.bfloat16 else torch.int32)


def _same(xs, ys):
    return all(x.dtype == y.dtype and torch.equal(_bits(x), _bits(y)) for x, y in zip(xs, ys, strict=True))


def _check(got, want, room, what):
    got, want = got.double().cpu(), want
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = (got - want).abs()[fine]
    over = off > room[fine]
    assert not over.any(), (what, float(off[over].max()), float(room[fine][over].min()), int(over.sum()))


def _inputs(seed, dtype, b, t, hq, hkv, d, page, lens, counts, fill=float("nan"), extra=1):
    rng = np.random.default_rng(seed)
    width = -(-max(lens) // page) + extra
    k, v, table = R.make_cache(rng, b, hkv, d, page, width, lens, DT[dtype], fill=fill)
    q = torch.from_numpy((rng.standard_normal((b, t, hq, d)) * 2).astype(np.float32)).to(DT[dtype])
    scores = torch.from_numpy(rng.random((b, hkv, width * page)).astype(np.float32))
    lens = torch.tensor(lens, dtype=torch.int32)
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    return q, k, v, table, lens, counts, scores


def _decode(gpu, q, k, v, table, lens, counts=None, scores=None, **more):
    from tallax_amd import kvcache
    up = [x.to(gpu) if x is not None else None for x in (q, k, v, table, lens, counts, scores)]
    return kvcache.decode(*up[:5], counts=up[5], scores=up[6], **more)


DECODE = [
    # batch, queries, heads, kv_heads, dim, page, lens, counts
    (1, 1, 1, 1, 64, 16, [1], None),
    (3, 1, 8, 2, 64, 16, [33, 0, 1], None),
    (3, 1, 4, 4, 128, 1, [130, 31, 32], None),
    (2, 3, 8, 2, 80, 24, [300, 2], [3, 2]),
    (3, 5, 32, 8, 128, 32, [700, 129, 64], [5, 0, 1]),
    (2, 9, 16, 2, 256, 100, [513, 8], [9, 4]),
    (4, 2, 14, 2, 96, 8, [65, 63, 1, 0], None),
    (2, 1, 5, 5, 8, 16, [50, 17], None),
    (1, 16, 8, 1, 128, 64, [1000], None),
    (2, 1, 64, 1, 128, 16, [2500, 257], None),
    (2, 4, 24, 3, 192, 7, [411, 255], [4, 9]),
    (2, 7, 40, 8, 72, 48, [97, 600], [1, 6]),
    (9, 1, 12, 12, 80, 24, [1, 2, 15, 16, 17, 127, 128, 129, 0], None),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", DECODE, ids=lambda c: "x".join(map(str, c[:6])))
def test_decode(gpu, dtype, case):
    b, t, hq, hkv, d, page, lens, counts = case
    q, k, v, table, lens, counts, scores = _inputs(1, dtype, b, t, hq, hkv, d, page, lens, counts)
    want = R.attention(q, k, v, table, lens, d ** -0.5, counts, scores)
    out, lse, new = _decode(gpu, q, k, v, table, lens, counts, scores)
    _check(out, want[0], want[3][0], "out")
    _check(lse, want[1], want[3][1], "lse")
    _check(new, want[2], want[3][2], "scores")
    out2, lse2 = _decode(gpu, q, k, v, table, lens, counts)
    assert torch.equal(_bits(out), _bits(out2)) and torch.equal(_bits(lse), _bits(lse2))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [16, 24, 128])
def test_decode_long_is_split_and_joined(gpu, dtype, page):
    lens = [9000, 1, 0, 4097, 8192, 256, 257]
    q, k, v, table, lens, _, scores = _inputs(2, dtype, 7, 1, 8, 2, 64, page, lens, None, fill=None)
    want = R.attention(q, k, v, table, lens, 0.3, None, scores)
    out, lse, new = _decode(gpu, q, k, v, table, lens, None, scores, scale=0.3, max_len=9000)
    _check(out, want[0], want[3][0], "out")
    _check(lse, want[1], want[3][1], "lse")
    _check(new, want[2], want[3][2], "scores")


def test_decode_max_len_cuts(gpu):
    q, k, v, table, lens, _, scores = _inputs(3, "bf16", 2, 1, 4, 2, 64, 16, [300, 90], None)
    cut = torch.clamp(lens, max=100)
    want = R.attention(q, k, v, table, cut, 0.125, None, scores)
    out, lse, new = _decode(gpu, q, k, v, table, lens, None, scores, max_len=100)
    _check(out, want[0], want[3][0], "out")
    _check(lse, want[1], want[3][1], "lse")
    _check(new, want[2], want[3][2], "scores")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [32, 5])
def test_decode_skips_what_is_no_page(gpu, dtype, page):
    q, k, v, table, lens, counts, scores = _inputs(4, dtype, 3, 2, 8, 2, 128, page, [200, 100, 64], [2, 2, 1])
    table[0, 1], table[0, 3] = -1, k.shape[0]
    table[1, :] = -7  # no slot of this sequence is anywhere
    table[2, 0] = 2 ** 31 - 1
    want = R.attention(q, k, v, table, lens, 128 ** -0.5, counts, scores)
    out, lse, new = _decode(gpu, q, k, v, table, lens, counts, scores)
    _check(out, want[0], want[3][0], "out")
    _check(lse, want[1], want[3][1], "lse")
    _check(new, want[2], want[3][2], "scores")
    assert float(out[1].float().abs().max()) == 0 and bool((lse[1] == -float("inf")).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_decode_values_of_unseen_tokens_do_not_leak(gpu, dtype, bad):
    """The last two tokens' keys and values are not finite: only the queries that see them may show it."""
    q, k, v, table, lens, counts, scores = _inputs(5, dtype, 2, 4, 8, 2, 64, 16, [150, 70], [4, 3], fill=bad)
    for b in range(2):
        for s in (int(lens[b]) - 2, int(lens[b]) - 1):
            v[table[b, s // 16], :, s % 16, 5] = bad
    want = R.attention(q, k, v, table, lens, 0.125, counts)
    out, lse = _decode(gpu, q, k, v, table, lens, counts)
    seen_bad = torch.zeros((2, 4), dtype=torch.bool)
    seen_bad[0, 2:] = True
    seen_bad[1, 1:3] = True
    got = out.double().cpu()
    assert not torch.isfinite(got[seen_bad][..., 5]).any()
    ok = got.clone()
    ok[seen_bad] = 0
    clean = want[0].clone()
    clean[seen_bad] = 0
    _check(ok, clean, want[3][0].nan_to_num(0.0), "out")
    keys = k.clone()
    for b in range(2):
        s = int(lens[b]) - 1
        keys[table[b, s // 16], :, s % 16, 3] = bad
    out, lse = _decode(gpu, q, keys, R_clean(v, table, lens), table, lens, counts)
    assert torch.isfinite(out[0, :3].float()).all() and torch.isfinite(lse[0, :3]).all()
    assert torch.isfinite(out[1, :2].float()).all() and torch.isfinite(lse[1, :2]).all()


def R_clean(v, table, lens):
    v = v.clone()
    for b in range(len(lens)):
        for s in (int(lens[b]) - 2, int(lens[b]) - 1):
            v[table[b, s // 16], :, s % 16, 5] = 1.0
    return v


def test_decode_scores_at_the_ends_of_the_range(gpu):
    """Keys that make scores of +-1e4 and beyond: the running maximum has to carry them."""
    q, k, v, table, lens, _, scores = _inputs(6, "f32", 2, 1, 4, 2, 64, 16, [600, 40], None)
    k = k * torch.where(torch.rand((k.shape[0], 1, 16, 1), generator=torch.Generator().manual_seed(1)) < 0.1, 300.0, 1.0)
    want = R.attention(q, k, v, table, lens, 1.0, None, scores)
    out, lse, new = _decode(gpu, q, k, v, table, lens, None, scores, scale=1.0)
    _check(out, want[0], want[3][0], "out")
    _check(lse, want[1], want[3][1], "lse")
    _check(new, want[2], want[3][2], "scores")


def test_decode_layouts(gpu):
    """Pools with slots before heads, pools inside a larger one, q as a part of a projection's output."""
    q, k, v, table, lens, counts, scores = _inputs(7, "bf16", 3, 2, 8, 4, 64, 16, [100, 40, 7], None)
    out, lse, new = _decode(gpu, q, k, v, table, lens, None, scores)
    by_slot = [x.transpose(1, 2).contiguous().to(gpu).transpose(1, 2) for x in (k, v)]
    both = torch.stack([k, v], 1).to(gpu)
    wide = torch.zeros((3, 2, 8 * 64 + 128), dtype=torch.bfloat16, device=gpu)
    wide[..., 64:64 + 512] = q.reshape(3, 2, 512).to(gpu)
    odd = torch.zeros((3, 2, 8 * 64 + 3), dtype=torch.bfloat16, device=gpu)
    odd[..., 3:] = q.reshape(3, 2, 512).to(gpu)
    for qq in (q.to(gpu), wide[..., 64:576].unflatten(-1, (8, 64)), odd[..., 3:].unflatten(-1, (8, 64))):
        for kk, vv in (by_slot, (both[:, 0], both[:, 1]), (k.to(gpu), by_slot[1])):
            o, l, s = _decode(gpu, qq, kk, vv, table, lens, None, scores)
            assert torch.equal(_bits(o), _bits(out)) and torch.equal(_bits(l), _bits(lse))
            assert torch.equal(_bits(s), _bits(new))


def test_decode_pool_past_4_gib(gpu):
    page, hkv, d = 64, 8, 128
    pages = (5 << 30) // (page * hkv * d * 2)
    big = [torch.empty((pages, hkv, page, d), dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    q, k, v, table, lens, _, scores = _inputs(8, "bf16", 1, 1, 16, hkv, d, page, [300], None, fill=None)
    ids = torch.where(table >= 0, table, 0).long()
    at = pages - 1 - torch.arange(table.shape[1]) * 3
    for x, small in zip(big, (k, v)):
        x[at.to(gpu)] = small[ids[0]].to(gpu)
    far = torch.where(table >= 0, at[None].to(torch.int32), table).to(torch.int32)
    out, lse, new = _decode(gpu, q, k, v, table, lens, None, scores)
    o, l, s = _decode(gpu, q, big[0], big[1], far, lens, None, scores)
    assert torch.equal(_bits(o), _bits(out)) and torch.equal(_bits(l), _bits(lse)) and torch.equal(_bits(s), _bits(new))


def test_decode_in_place_scores_streams_and_graph(gpu):
    from tallax_amd import kvcache
    q, k, v, table, lens, counts, scores = [
        x.to(gpu) if x is not None else None
        for x in _inputs(9, "bf16", 4, 3, 8, 2, 128, 16, [700, 33, 1, 0], [3, 1, 1, 0])]
    out, lse, new = kvcache.decode(q, k, v, table, lens, counts=counts, scores=scores)
    again = kvcache.decode(q, k, v, table, lens, counts=counts, scores=scores)
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip((out, lse, new), again))
    own = scores.clone()
    _, _, same = kvcache.decode(q, k, v, table, lens, counts=counts, scores=own, out_scores=own)
    assert same is own and torch.equal(_bits(own), _bits(new))
    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream())
    ws = torch.empty(8 << 20, dtype=torch.uint8, device=gpu)
    with torch.cuda.stream(side):
        there = kvcache.decode(q, k, v, table, lens, counts=counts, scores=scores, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip((out, lse, new), there))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = kvcache.decode(q, k, v, table, lens, counts=counts, scores=scores, workspace=ws)
    for rep in range(3):
        q.copy_(torch.randn(q.shape, device=gpu))
        lens.copy_(torch.tensor([701 + rep, 40 * rep, 5, rep], dtype=torch.int32).clamp(max=table.shape[1] * 16))
        table.copy_(torch.where(table < 0, 0, table))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured]
        want = kvcache.decode(q, k, v, table, lens, counts=counts, scores=scores)
        torch.cuda.synchronize()
        assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(got, want)), rep


APPEND = [
    # batch, tokens, kv_heads, dim, page, lens, counts
    (1, 1, 1, 8, 1, [0], None),
    (3, 1, 8, 128, 16, [15, 16, 17], None),
    (4, 5, 2, 80, 24, [20, 0, 47, 3], [5, 0, 2, 9]),
    (2, 130, 3, 64, 64, [1, 100], None),
    (2, 0, 3, 64, 64, [1, 100], None),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: "x".join(map(str, c[:5])))
def test_append(gpu, dtype, case):
    from tallax_amd import kvcache
    b, t, hkv, d, page, lens, counts = case
    rng = np.random.default_rng(10)
    width = -(-(max(lens) + t) // page)  # of the longest; others may run past nothing, but not past the table
    k, v, table = R.make_cache(rng, b, hkv, d, page, max(width, 1), [n + t for n in lens], DT[dtype])
    if b > 1 and width > 1:
        table[1, lens[1] // page] = -1  # its tokens are dropped
    new = [torch.from_numpy(rng.standard_normal((b, t, hkv, d)).astype(np.float32)).to(DT[dtype]) for _ in range(2)]
    slots = table.shape[1] * page
    scores = torch.from_numpy(rng.random((b, hkv, slots)).astype(np.float32))
    positions = torch.from_numpy(rng.integers(0, 100, (b, hkv, slots)).astype(np.int32))
    lens, seen = torch.tensor(lens, dtype=torch.int32), torch.arange(b, dtype=torch.int32) * 1000 + 50
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    want = [x.clone() for x in (k, v, scores, positions)]
    want_lens = lens.clone()
    for i in range(b):
        n = t if counts is None else min(counts[i], t)
        want_lens[i] = min(int(lens[i]) + n, slots)
        for j in range(n):
            s = int(lens[i]) + j
            p = int(table[i, s // page]) if s < slots else -1
            if p < 0:
                continue
            want[0][p, :, s % page], want[1][p, :, s % page] = new[0][i, j], new[1][i, j]
            want[2][i, :, s], want[3][i, :, s] = 0.0, int(seen[i]) + j
    got = [x.to(gpu) for x in (k, v, scores, positions)]
    up = [x.to(gpu) for x in (table, lens, new[0], new[1], seen)]
    cnt = None if cnt is None else cnt.to(gpu)
    out = kvcache.append(got[0], got[1], *up[:4], counts=cnt, scores=got[2], positions=got[3], seen=up[4])
    assert torch.equal(out.cpu(), want_lens)
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(got, want))
    got = [x.to(gpu) for x in (k, v)]
    views = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in got]
    kvcache.append(views[0], views[1], *up[:4], counts=cnt)
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(views, want))


def test_append_past_the_table_is_dropped(gpu):
    from tallax_amd import kvcache
    k, v = (torch.zeros((2, 1, 4, 8), device=gpu) for _ in range(2))
    table = torch.tensor([[1]], dtype=torch.int32, device=gpu)
    lens = torch.tensor([3], dtype=torch.int32, device=gpu)
    new = torch.ones((1, 5, 1, 8), device=gpu)
    assert kvcache.append(k, v, table, lens, new, new).tolist() == [4]
    assert float(k.sum()) == 8 and float(k[1, 0, 3].sum()) == 8


EVICT = [
    # batch, kv_heads, dim, page, lens, budget, recent, sinks
    (1, 1, 8, 1, [1], 1, 0, 0),
    (3, 2, 64, 16, [100, 33, 0], 32, 8, 4),
    (2, 3, 80, 24, [500, 499], 498, 100, 4),
    (2, 2, 128, 64, [1500, 2100], 300, 0, 0),
    (2, 8, 64, 7, [64, 65], 64, 64, 0),
    (1, 1, 64, 16, [5000], 1, 1, 0),
    (2, 1, 64, 16, [4100, 1025], 1024, 0, 1024),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["spread", "ties", "strange", "equal"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: "x".join(map(str, c[:4])) + "_%d" % c[5])
def test_evict(gpu, dtype, kind, case):
    from tallax_amd import kvcache
    b, hkv, d, page, lens, budget, recent, sinks = case
    rng = np.random.default_rng(11)
    width = -(-max(lens) // page) + 1
    k, v, table = R.make_cache(rng, b, hkv, d, page, width, lens, DT[dtype])
    slots = width * page
    scores = rng.standard_normal((b, hkv, slots)).astype(np.float32)
    if kind == "ties":
        scores = np.round(scores)
    elif kind == "equal":
        scores[:] = 0.25
    elif kind == "strange":
        at = rng.random(scores.shape)
        scores = np.where(at < 0.2, np.nan, np.where(at < 0.4, np.inf, np.where(at < 0.6, -np.inf, scores)))
        scores = np.where(at > 0.9, -0.0, np.where(at > 0.8, 0.0, scores)).astype(np.float32)
    positions = np.stack([np.stack([rng.permutation(slots) for _ in range(hkv)]) for _ in range(b)]).astype(np.int32)
    lens = torch.tensor(lens, dtype=torch.int32)
    seen = torch.full((b,), slots, dtype=torch.int32)
    scores, positions = torch.from_numpy(scores), torch.from_numpy(positions)
    if width > 4:
        table[0, 1] = -1
    want = R.evict(k, v, table, lens, scores, positions, seen, budget, recent, sinks)
    up = [x.to(gpu) for x in (k, v, table, lens, scores, positions, seen)]
    got = kvcache.evict(*up, budget=budget, recent=recent, sinks=sinks)
    ok = [_same([x], [y]) for x, y in zip((up[0], up[1], *got), want)]
    assert all(ok), ok
    # sources are not written: the same call again gives the same cache
    again = kvcache.evict(*up, budget=budget, recent=recent, sinks=sinks)
    ok = [_same([x], [y]) for x, y in zip((up[0], up[1], *again), want)]
    assert all(ok), ok


def test_evict_negative_positions_and_layout(gpu):
    """All positions inside the first `sinks`: more are always kept than the budget holds, so the lowest slots stay."""
    from tallax_amd import kvcache
    rng = np.random.default_rng(12)
    k, v, table = R.make_cache(rng, 1, 2, 64, 16, 4, [60], torch.bfloat16)
    scores = torch.from_numpy(rng.random((1, 2, 64)).astype(np.float32))
    positions = torch.full((1, 2, 64), -5, dtype=torch.int32)
    lens, seen = torch.tensor([60], dtype=torch.int32), torch.tensor([60], dtype=torch.int32)
    want = R.evict(k, v, table, lens, scores, positions, seen, 20, 0, 4)
    kk, vv = (x.transpose(1, 2).contiguous().to(gpu).transpose(1, 2) for x in (k, v))
    got = kvcache.evict(kk, vv, *[x.to(gpu) for x in (table, lens, scores, positions, seen)], budget=20, sinks=4)
    assert torch.equal(_bits(got[1]), _bits(want[3])) and torch.equal(_bits(kk), _bits(want[0]))
    assert torch.equal(_bits(vv), _bits(want[1]))


def test_evict_and_append_in_a_graph(gpu):
    from tallax_amd import kvcache
    rng = np.random.default_rng(13)
    lens_list = [300, 64, 200]
    k0, v0, table = R.make_cache(rng, 3, 2, 64, 16, 20, lens_list, torch.bfloat16)
    k, v, table = k0.to(gpu), v0.to(gpu), table.to(gpu)
    lens = torch.tensor(lens_list, dtype=torch.int32, device=gpu)
    scores = torch.rand((3, 2, 320), device=gpu)
    positions = torch.arange(320, dtype=torch.int32, device=gpu).expand(3, 2, 320).contiguous()
    new = torch.randn((3, 2, 2, 64), device=gpu).to(torch.bfloat16)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)

    def step():
        a = kvcache.evict(k, v, table, lens, scores, positions, lens, budget=64, recent=8, sinks=2, workspace=ws)
        return a + (kvcache.append(k, v, table, a[0], new, new, scores=a[1], positions=a[2], seen=lens),)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for rep in range(3):
        scores.uniform_()
        k.copy_(k0)
        v.copy_(v0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured + (k, v)]
        k.copy_(k0)
        v.copy_(v0)
        want = step() + (k, v)
        torch.cuda.synchronize()
        assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(got, want)), rep


def test_refusals(gpu):
    from tallax_amd import kvcache
    k, v = (torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    table = torch.zeros((3, 2), dtype=torch.int32, device=gpu)
    lens = torch.ones(3, dtype=torch.int32, device=gpu)
    q = torch.zeros((3, 1, 4, 64), dtype=torch.bfloat16, device=gpu)
    scores = torch.zeros((3, 2, 32), device=gpu)
    positions = torch.zeros((3, 2, 32), dtype=torch.int32, device=gpu)
    kvcache.decode(q, k, v, table, lens, scores=scores)
    for bad in (dict(q=q[:2]), dict(q=q.float()), dict(q=q[:, :, :3]), dict(q=q[..., :32]), dict(q=q[:, :0]),
                dict(k_pages=k[:, :1]), dict(k_pages=k.float()), dict(k_pages=k.cpu()), dict(lens=lens.long()),
                dict(lens=lens[:2]), dict(block_table=table.long()), dict(block_table=table.t()),
                dict(scores=scores[..., :16]), dict(scores=scores.double()), dict(counts=lens[:2]),
                dict(max_len=33), dict(max_len=-1), dict(scale=float("nan")), dict(out_scores=scores),
                dict(workspace=torch.zeros(4, device=gpu), scores=scores)):
        args = dict(q=q, k_pages=k, v_pages=v, block_table=table, lens=lens)
        with pytest.raises(ValueError):
            kvcache.decode(**{**args, **bad})
    with pytest.raises(NotImplementedError):
        kvcache.decode(q.half(), k.half(), v.half(), table, lens)
    with pytest.raises(NotImplementedError):
        kvcache.decode(q[..., :60].contiguous(), k[..., :60].contiguous(), v[..., :60].contiguous(), table, lens)
    odd = torch.zeros((4, 2, 16, 66), dtype=torch.bfloat16, device=gpu)[..., 1:65]
    with pytest.raises(NotImplementedError):  # not on 16 bytes: a pool is never copied
        kvcache.decode(q, odd, v, table, lens)
    with pytest.raises(ValueError):
        kvcache.decode(q, k[..., ::2], v[..., ::2], table, lens)
    for bad in (dict(k_new=q[..., :32]), dict(scores=scores), dict(scores=scores, positions=positions),
                dict(k_new=torch.zeros((3, 1, 2, 64), device=gpu))):
        n = torch.zeros((3, 1, 2, 64), dtype=torch.bfloat16, device=gpu)
        with pytest.raises(ValueError):
            kvcache.append(**{**dict(k_pages=k, v_pages=v, block_table=table, lens=lens, k_new=n, v_new=n), **bad})
    for bad in (dict(budget=0), dict(budget=4, recent=3, sinks=2), dict(budget=4, recent=-1), dict(budget=-3)):
        with pytest.raises(ValueError):
            kvcache.evict(k, v, table, lens, scores, positions, lens, **bad)


def test_empty_batches_and_tables(gpu):
    from tallax_amd import kvcache
    k, v = (torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    for batch, width in ((0, 2), (2, 0)):
        table = torch.zeros((batch, width), dtype=torch.int32, device=gpu)
        lens = torch.zeros(batch, dtype=torch.int32, device=gpu)
        q = torch.ones((batch, 2, 4, 64), dtype=torch.bfloat16, device=gpu)
        scores = torch.zeros((batch, 2, width * 16), device=gpu)
        positions = torch.zeros((batch, 2, width * 16), dtype=torch.int32, device=gpu)
        out, lse, new = kvcache.decode(q, k, v, table, lens, scores=scores)
        assert out.shape == q.shape and bool((out == 0).all()) and bool((lse == -float("inf")).all())
        n = torch.ones((batch, 1, 2, 64), dtype=torch.bfloat16, device=gpu)
        assert kvcache.append(k, v, table, lens, n, n).tolist() == [0] * batch
        assert kvcache.evict(k, v, table, lens, scores, positions, lens, budget=3)[0].tolist() == [0] * batch
    assert float(k.float().abs().max()) == 0


def test_decode_max_len_cuts_several_queries(gpu):
    """A length above max_len is taken as max_len for every query of a draft, not for the last alone."""
    q, k, v, table, lens, counts, scores = _inputs(14, "bf16", 3, 4, 8, 2, 64, 16, [300, 90, 101], [4, 2, 3])
    cut = torch.clamp(lens, max=100)
    want = R.attention(q, k, v, table, cut, 0.125, counts, scores)
    out, lse, new = _decode(gpu, q, k, v, table, lens, counts, scores, max_len=100)
    _check(out, want[0], want[3][0], "out")
    _check(lse, want[1], want[3][1], "lse")
    _check(new, want[2], want[3][2], "scores")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", [(2, 9, 32, 4, 128, 16, [300, 70], [9, 5]), (1, 5, 24, 2, 256, 24, [290], None),
                                  (2, 3, 33, 3, 200, 8, [130, 259], [3, 1]), (1, 12, 16, 2, 16, 5, [77], None)],
                         ids=lambda c: "x".join(map(str, c[:6])))
def test_decode_many_rows(gpu, dtype, case):
    """More rows of a kv head than one workgroup takes, some of them not a whole tile, all dims."""
    b, t, hq, hkv, d, page, lens, counts = case
    q, k, v, table, lens, counts, scores = _inputs(15, dtype, b, t, hq, hkv, d, page, lens, counts)
    want = R.attention(q, k, v, table, lens, d ** -0.5, counts, scores)
    out, lse, new = _decode(gpu, q, k, v, table, lens, counts, scores)
    _check(out, want[0], want[3][0], "out")
    _check(lse, want[1], want[3][1], "lse")
    _check(new, want[2], want[3][2], "scores")


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("f32", 80), ("f32", 256)])
def test_decode_values_that_are_not_finite(gpu, dtype, dim):
    """Values of the newest tokens of 8 queries that are infinite or NaN, in more than one place and with both signs:
    each query shows those it sees, in the places they have, and nothing else changes."""
    q, k, v, table, lens, counts, _ = _inputs(16, dtype, 2, 8, 8, 2, dim, 16, [140, 75], [8, 6])
    clean = R.attention(q, k, v, table, lens, 0.125, counts)
    bad = v.clone()
    at = {(0, 139): (5, float("inf")), (0, 137): (7, float("-inf")), (0, 133): (dim - 1, float("nan")),
          (1, 74): (0, float("nan")), (1, 73): (0, float("inf")), (1, 70): (3, float("-inf"))}
    for (b, s), (d, x) in at.items():
        bad[table[b, s // 16], :, s % 16, d] = x
    out, lse = _decode(gpu, q, k, bad, table, lens, counts, scale=0.125)
    got, want, room = out.double().cpu(), clean[0].clone(), clean[3][0].clone()
    for b, n in ((0, 8), (1, 6)):
        for t in range(n):
            end = int(lens[b]) - n + t + 1
            for d in {d for (bb, s), (d, _) in at.items() if bb == b}:
                xs = [x for (bb, s), (dd, x) in at.items() if bb == b and dd == d and s < end]
                hidden = [s for (bb, s), (dd, x) in at.items() if bb == b and dd == d and s >= end]
                if xs:
                    want[b, t, :, d] = sum(xs[1:], xs[0])
                    room[b, t, :, d] = 0
                elif hidden:
                    assert torch.isfinite(got[b, t, :, d]).all()
    _check(got, want, room, "out")
    _check(lse, clean[1], clean[3][1], "lse")


@pytest.mark.parametrize("cap,lens,budget", [(40000, [39999, 33000], 35000), (70000, [70000, 20], 4097)])
@pytest.mark.parametrize("kind", ["spread", "ties"])
def test_evict_long_rows(gpu, cap, lens, budget, kind):
    """More slots than a workgroup holds at once, against a stable sort."""
    from tallax_amd import kvcache
    rng = np.random.default_rng(17)
    page, b, hkv = 100, len(lens), 2
    width = cap // page
    k = torch.arange(b * width * hkv * page, dtype=torch.int32).reshape(b * width, hkv, page, 1)
    k = k.repeat(1, 1, 1, 8).to(torch.float32).contiguous()  # below 2^24: exact
    v = -k
    table = torch.from_numpy(rng.permutation(b * width).reshape(b, width).astype(np.int32))
    scores = rng.standard_normal((b, hkv, cap)).astype(np.float32)
    if kind == "ties":
        scores = np.round(scores)
    positions = np.broadcast_to(np.arange(cap, dtype=np.int32), (b, hkv, cap)).copy()
    up = [x.to(gpu) for x in (k.clone(), v.clone(), table, torch.tensor(lens, dtype=torch.int32),
                              torch.from_numpy(scores), torch.from_numpy(positions),
                              torch.tensor(lens, dtype=torch.int32))]
    got = kvcache.evict(*up, budget=budget, recent=100, sinks=4)
    kk, vv = up[0].cpu(), up[1].cpu()
    for i, n in enumerate(lens):
        m = min(n, budget)
        assert int(got[0][i]) == m
        for h in range(hkv):
            key = scores[i, h, :n].astype(np.float64)
            key[:4] = key[n - 100:n] = 1e9
            keep = np.zeros(n, bool)
            keep[np.argsort(-key, kind="stable")[:m]] = True
            source = np.arange(m)
            source[~keep[:m]] = np.arange(n)[keep & (np.arange(n) >= m)]
            want_s, want_p = np.zeros(cap, np.float32), np.full(cap, -1, np.int32)
            want_s[:m], want_p[:m] = scores[i, h, source], positions[i, h, source]
            assert np.array_equal(got[1][i, h].cpu().numpy(), want_s)
            assert np.array_equal(got[2][i, h].cpu().numpy(), want_p)
            slot = torch.arange(m)
            src = torch.from_numpy(source)
            to = kk[table[i, slot // page].long(), h, slot % page, 0]
            assert torch.equal(to, k[table[i, src // page].long(), h, src % page, 0])
            assert torch.equal(vv[table[i, slot // page].long(), h, slot % page, 3], -to)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_keys_that_weigh_nothing(gpu, dtype):
    """Scores of -inf: such slots get no weight, and a query whose every score is -inf gives 0 and -inf."""
    q, k, v, table, lens, _, scores = _inputs(18, dtype, 3, 1, 8, 2, 64, 16, [300, 40, 500], None)
    q[..., 0] = 1.0
    k[..., 0] = k[..., 0].nan_to_num(0.0)
    for b, slots in ((0, range(0, 300, 3)), (1, range(40)), (2, range(0, 256))):
        for s in slots:
            k[table[b, s // 16], :, s % 16, 0] = -float("inf")
    out, lse, new = _decode(gpu, q, k, v, table, lens, None, scores, scale=0.125)
    for i in (0, 2):  # the same as without those slots
        n = int(lens[i])
        keep = torch.tensor([t for t in range(n) if not (t % 3 == 0 if i == 0 else t < 256)])
        pages = -(-len(keep) // 16)
        pools = []
        for x in (k, v):
            dense = torch.zeros((pages * 16, 2, 64), dtype=x.dtype)
            dense[:len(keep)] = x[table[i, keep // 16].long(), :, keep % 16]
            pools.append(dense.reshape(pages, 16, 2, 64).transpose(1, 2))
        left = torch.zeros((1, 2, pages * 16))
        left[0, :, :len(keep)] = scores[i][:, keep]
        want = R.attention(q[i:i + 1], *pools, torch.arange(pages, dtype=torch.int32)[None],
                           torch.tensor([len(keep)], dtype=torch.int32), 0.125, None, left)
        _check(out[i:i + 1], want[0], want[3][0], "out")
        _check(lse[i:i + 1], want[1], want[3][1], "lse")
        got = new[i].cpu()
        _check(got[:, keep], want[2][0][:, :len(keep)], want[3][2][0][:, :len(keep)], "scores")
        rest = torch.ones(scores.shape[2], dtype=torch.bool)
        rest[keep] = False
        assert torch.equal(got[:, rest], scores[i][:, rest])
    assert float(out[1].float().abs().max()) == 0 and bool((lse[1] == -float("inf")).all())
    assert torch.equal(new[1].cpu(), scores[1])


@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_decode_scales(gpu, scale):
    q, k, v, table, lens, counts, scores = _inputs(19, "bf16", 2, 2, 8, 2, 128, 16, [290, 17], [2, 1])
    want = R.attention(q, k, v, table, lens, scale, counts, scores)
    out, lse, new = _decode(gpu, q, k, v, table, lens, counts, scores, scale=scale)
    _check(out, want[0], want[3][0], "out")
    _check(lse, want[1], want[3][1], "lse")
    _check(new, want[2], want[3][2], "scores")
