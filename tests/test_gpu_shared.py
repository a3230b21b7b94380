"""GPU: kvcache.decode_shared against attention over both parts in 64 bits, at the sizes, types and masks where it can
go wrong."""
import math

import numpy as np
import pytest
import torch

from tests import layer_ref as L
from tests import serving_ref as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _make(rng, lens, begins, queries, heads, kv_heads, dim, page, dtype, q_scale=1.5, fill=None):
    """q, pools, prefix table and lengths, table and lengths on the host; prefixes lie in the same pools."""
    batch, prompts = len(lens), len(begins)
    all_lens = list(lens) + list(begins)
    width = max(1, max(-(-n // page) for n in all_lens))
    k, v, table = R.make_cache(rng, batch + prompts, kv_heads, dim, page, width, all_lens, dtype, fill=fill)
    q = torch.from_numpy(rng.standard_normal((batch, queries, heads, dim)).astype(np.float32) * q_scale).to(dtype)
    t = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    own = max(1, max(-(-n // page) for n in lens))
    return q, k, v, table[batch:].contiguous(), t(begins), table[:batch, :own].contiguous(), t(lens)


def _run(gpu, args, scale=None, counts=None, **kw):
    from tallax_amd import kvcache
    d = [x.to(gpu) for x in args]
    return kvcache.decode_shared(*d, scale=scale, counts=None if counts is None else counts.to(gpu), **kw)


def _check(got, want):
    out, lse, out_room, lse_room = want
    for x, y, room in ((got[0], out, out_room), (got[1], lse, lse_room)):
        x = x.cpu().double()
        same = x == y  # -inf among them
        off = (x - y).abs()
        ok = same | (off <= room)
        assert bool(ok.all()), (float(off[~ok].max()), float((off / room)[~ok].max()), int((~ok).sum()))


def _both(gpu, args, scale=None, counts=None, **kw):
    q, dim = args[0], args[0].shape[-1]
    want = L.shared_attention(q, args[1], args[2], args[3], args[4].tolist(), args[5], args[6].tolist(),
                              dim ** -0.5 if scale is None else scale, counts)
    got = _run(gpu, args, scale, counts, **kw)
    _check(got, want)
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch,prompts,queries,heads,kv_heads,dim,page,prefix,longest", [
    (1, 1, 1, 1, 1, 8, 1, 1, 1), (4, 1, 1, 8, 2, 64, 16, 500, 100), (3, 3, 1, 6, 3, 80, 24, 130, 40),
    (5, 1, 3, 10, 5, 96, 8, 333, 17), (9, 1, 1, 32, 4, 128, 16, 700, 200), (17, 1, 1, 16, 2, 128, 32, 257, 33),
    (24, 2, 1, 7, 1, 64, 100, 1000, 5), (6, 2, 5, 8, 2, 128, 16, 300, 60), (40, 1, 1, 8, 2, 256, 16, 300, 20),
    (3, 1, 1, 16, 2, 256, 8, 400, 64), (2, 1, 9, 24, 2, 192, 16, 200, 40), (33, 1, 1, 4, 1, 40, 16, 2100, 9),
    (64, 1, 2, 8, 4, 64, 16, 515, 12), (12, 1, 1, 12, 12, 72, 24, 90, 30), (70, 1, 1, 6, 2, 128, 16, 400, 3)])
def test_shapes(gpu, dtype, batch, prompts, queries, heads, kv_heads, dim, page, prefix, longest):
    rng = np.random.default_rng(batch * 100 + dim)
    lens = [max(queries, longest - longest * 3 // 4 * i // batch) for i in range(batch)]
    begins = [prefix - prefix // 2 * i // prompts for i in range(prompts)]
    args = _make(rng, lens, begins, queries, heads, kv_heads, dim, page, dtype)
    counts = torch.from_numpy(rng.integers(0, queries + 1, batch).astype(np.int32))
    _both(gpu, args)
    _both(gpu, args, counts=counts)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 260])
def test_rows_around_the_tiles(gpu, dtype, rows):
    rng = np.random.default_rng(rows)
    args = _make(rng, [3] * rows, [150], 1, 1, 1, 64, 16, dtype)
    _both(gpu, args)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch", [4, 40, 80])
def test_prefix_lengths_around_the_tiles(gpu, dtype, dim, batch):
    rng = np.random.default_rng(dim + batch)
    for prefix in (1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513):
        args = _make(rng, [2] * batch, [prefix], 1, 1, 1, dim, 16, dtype)
        _both(gpu, args)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_parts_of_length_zero(gpu, dtype):
    """No prefix, nothing of its own, neither: what there is, or 0 and -inf."""
    rng = np.random.default_rng(3)
    args = _make(rng, [0, 5, 0, 9], [0, 40], 1, 4, 2, 64, 8, dtype)
    out, lse = _both(gpu, args)
    assert not bool(out[0].any()) and bool((lse[0] == -math.inf).all())
    _both(gpu, args, counts=torch.tensor([1, 0, 1, -4], dtype=torch.int32))
    q, k, v, prefix, begins, table, lens = args
    empty = torch.zeros_like(lens)
    _both(gpu, (q, k, v, prefix, begins, table[:, :0].contiguous(), empty))  # a table of no width
    _both(gpu, (q, k, v, prefix[:, :0].contiguous(), begins * 0, table, lens))
    _both(gpu, (q, k, v, prefix[:, :0].contiguous(), begins * 0, table[:, :0].contiguous(), empty))
    # queries in front of their sequence's first slot see the prefix alone
    _both(gpu, (q, k, v, prefix, begins, table, lens))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch", [3, 40, 130])
def test_pages_that_are_not_there(gpu, dtype, batch):
    rng = np.random.default_rng(4)
    args = _make(rng, [20] * batch, [300], 1, 2, 1, 64, 8, dtype)
    q, k, v, prefix, begins, table, lens = args
    prefix = prefix.clone()
    prefix[0, [0, 3, 7, 8, 30]] = torch.tensor([-1, 99999, -5, k.shape[0], -1], dtype=torch.int32)
    table = table.clone()
    table[0] = -1
    _both(gpu, (q, k, v, prefix, begins, table, lens))
    out, lse = _both(gpu, (q, k, v, prefix * 0 - 1, begins, table, lens))
    assert not bool(out[0].any()) and bool((lse[0] == -math.inf).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch", [3, 40, 130])
@pytest.mark.parametrize("dim", [40, 64, 128, 256])
def test_unused_slots_do_not_matter(gpu, dtype, batch, dim):
    """Slots past the lengths, and the pages of others, hold NaN."""
    rng = np.random.default_rng(5)
    args = _make(rng, [20 + i % 3 for i in range(batch)], [77], 1, 2, 1, dim, 16, dtype, fill=math.nan)
    _both(gpu, args)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch", [3, 40, 130])
def test_values_that_are_not_finite(gpu, dtype, batch):
    """In the prefix every query of its sequences sees them, and none of the other prefix's; keys of -inf weigh nothing."""
    rng = np.random.default_rng(6)
    q, k, v, prefix, begins, table, lens = _make(rng, [6] * (2 * batch), [100, 90], 1, 2, 1, 64, 16, dtype)
    v[int(prefix[0, 2]), 0, 3, 5] = math.inf
    v[int(table[1, 0]), 0, 2, 9] = math.nan
    out, _ = _run(gpu, (q, k, v, prefix, begins, table, lens))
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[:batch, ..., 5] = True
    bad[1, ..., 9] = True
    assert torch.equal(~torch.isfinite(out.cpu().float()), bad)
    q, k, v, prefix, begins, table, lens = _make(rng, [6] * (2 * batch), [100, 90], 1, 2, 1, 64, 16, dtype)
    q = q.abs() + 0.1
    want = L.shared_attention(q, k, v, prefix[:, 1:], [84, 74], table, lens.tolist(), 0.125)
    k[prefix[:, 0].long(), 0, :, 11] = -math.inf
    _check(_run(gpu, (q, k, v, prefix, begins, table, lens), 0.125), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-30])
def test_scales(gpu, dtype, scale):
    rng = np.random.default_rng(7)
    for batch in (2, 40, 70):
        args = _make(rng, [7] * batch, [130], 1, 2, 1, 64, 16, dtype, q_scale=1.0)
        _both(gpu, args, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_that_grow_and_shrink(gpu, dtype):
    """The running maximum moves in every tile, or only in the first; scores of hundreds."""
    rng = np.random.default_rng(8)
    for batch in (2, 40):
        for slope in (0.5, -0.5, 0.0):
            q, k, v, prefix, begins, table, lens = _make(rng, [40] * batch, [600], 1, 2, 1, 64, 8, dtype)
            q[..., 0] = 8.0
            for i in range(600):
                k[int(prefix[0, i // 8]), 0, i % 8, 0] = slope * i
            _both(gpu, (q, k, v, prefix, begins, table, lens))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(gpu, dtype):
    """Pools with heads and slots in the other order, queries as a part of something larger, off 16 bytes, or not dense."""
    from tallax_amd import kvcache
    rng = np.random.default_rng(9)
    args = _make(rng, [20, 9, 4], [100], 2, 4, 2, 48, 8, dtype)
    q, k, v, *rest = (x.to(gpu) for x in args)
    want = kvcache.decode_shared(q, k, v, *rest)
    _check(want, L.shared_attention(args[0], args[1], args[2], args[3], [100], args[5], [20, 9, 4], 48 ** -0.5))
    k2, v2 = (y.transpose(1, 2).contiguous().transpose(1, 2) for y in (k, v))
    big = torch.zeros((3, 2, 12, 48), dtype=dtype, device=gpu)
    big[:, :, 4:8] = q
    odd = torch.empty(q.numel() + 1, dtype=dtype, device=gpu)[1:].view(q.shape).copy_(q)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    loose = q.transpose(2, 3).contiguous().transpose(2, 3)
    for qq, kk, vv in ((q, k2, v2), (big[:, :, 4:8], k, v), (odd, k, v), (turned, k2, v), (loose, k, v2)):
        assert all(torch.equal(a, b) for a, b in zip(kvcache.decode_shared(qq, kk, vv, *rest), want, strict=True))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bounds_on_the_lengths(gpu, dtype):
    """max_prefix and max_len change how the work is split, not what comes out; larger lengths are taken as them."""
    rng = np.random.default_rng(10)
    q, k, v, prefix, begins, table, lens = _make(rng, [30, 12, 25], [400], 1, 4, 2, 64, 8, dtype)
    wide = torch.cat([prefix, torch.full((1, 300), -1, dtype=torch.int32)], 1)
    _both(gpu, (q, k, v, wide, begins, table, lens))
    _both(gpu, (q, k, v, wide, begins, table, lens), max_prefix=400, max_len=30)
    cut = L.shared_attention(q, k, v, prefix, [99], table, [10, 10, 10], 0.125)
    _check(_run(gpu, (q, k, v, wide, begins, table, lens), max_prefix=99, max_len=10), cut)
    none = L.shared_attention(q, k, v, prefix, [0], table, [0, 0, 0], 0.125)
    _check(_run(gpu, (q, k, v, wide, begins, table, lens), max_prefix=0, max_len=0), none)
    below = (q, k, v, prefix, begins * 0 - 5, table, lens * 0 - 3)
    _check(_run(gpu, below), none)


def test_one_sequence_without_a_prefix_is_decode(gpu):
    """Where there is no prefix the results are decode's."""
    from tallax_amd import kvcache
    rng = np.random.default_rng(11)
    q, k, v, prefix, begins, table, lens = (x.to(gpu) for x in _make(rng, [300, 200], [1], 3, 4, 2, 64, 8, F32))
    want = kvcache.decode(q, k, v, table, lens)
    got = kvcache.decode_shared(q, k, v, prefix, begins * 0, table, lens)
    for a, b in zip(got, want, strict=True):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-6)


def test_workspaces(gpu):
    rng = np.random.default_rng(12)
    args = _make(rng, [30, 12, 25], [400], 1, 4, 2, 64, 8, F32)
    want = _run(gpu, args)
    buf = torch.empty(1 << 24, dtype=torch.uint8, device=gpu)
    for off in (16, 48):
        buf.fill_(0xff)
        assert all(torch.equal(x, y) for x, y in zip(_run(gpu, args, workspace=buf[off:]), want, strict=True))
    for off in (1, 8, 12):
        with pytest.raises(ValueError, match="16 bytes"):
            _run(gpu, args, workspace=buf[off:])
    with pytest.raises(ValueError, match="smaller"):
        _run(gpu, args, workspace=buf[:64])


def test_refusals(gpu):
    rng = np.random.default_rng(13)
    q, k, v, prefix, begins, table, lens = args = _make(rng, [30, 12, 25], [400], 1, 4, 2, 64, 8, F32)
    for bad in ((q[:2], *args[1:]), (q[..., :32], *args[1:]), (q.bfloat16(), *args[1:]), (q[:, :, :3], *args[1:]),
                (q, k, v, prefix[0], *args[4:]), (q, k, v, prefix.long(), *args[4:]), (q, k, v, prefix, begins.long(), *args[5:]),
                (q, k, v, prefix, torch.cat([begins, begins]), *args[5:]),
                (q, k, v, prefix.repeat(2, 1), begins.repeat(2), *args[5:]), (q, k, v, prefix[:0], begins[:0], *args[5:]),
                (q, k, v, prefix, begins, table, lens[:2])):
        with pytest.raises(ValueError):
            _run(gpu, bad)
    for kw in (dict(scale=math.inf), dict(scale=math.nan), dict(max_len=-1), dict(max_len=33), dict(max_prefix=-1),
               dict(max_prefix=401)):
        with pytest.raises(ValueError):
            _run(gpu, args, **kw)
    with pytest.raises(ValueError):
        _run(gpu, args, counts=lens[:2])
    from tallax_amd import kvcache
    d = [x.to(gpu) for x in args]
    for i, bad in ((0, q), (3, d[3].repeat(1, 2)[:, ::2]), (4, begins), (5, table), (0, None)):
        with pytest.raises(ValueError):
            kvcache.decode_shared(*d[:i], bad, *d[i + 1:])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,queries,group", [(64, 1, 3), (128, 1, 2), (128, 3, 2), (128, 5, 4), (256, 1, 2), (80, 2, 12),
                                               (192, 2, 3), (64, 1, 18)])
def test_many_sequences(gpu, dtype, dim, queries, group):
    """Enough of them that the workgroup of a sequence's own slots makes the outputs: lengths of zero, tables of several
    pages, counts of none and too many, pages that are missing, a prefix that is empty."""
    rng = np.random.default_rng(dim + queries)
    batch, kv_heads = 132, 2
    lens = [0 if i % 11 == 5 else queries + (i * 7) % 150 for i in range(batch)]
    args = _make(rng, lens, [333, 0, 70], queries, kv_heads * group, kv_heads, dim, 16, dtype, fill=math.nan)
    q, k, v, prefix, begins, table, own = args
    counts = torch.from_numpy(rng.integers(-1, queries + 3, batch).astype(np.int32))
    _both(gpu, args, counts=counts)
    table, prefix = table.clone(), prefix.clone()
    table[3], table[7, 0], prefix[0, [1, 5]] = -1, 99999, -1
    out, lse = _both(gpu, (q, k, v, prefix, begins, table, own))
    _both(gpu, (q, k, v, prefix, begins * 0, table, own))
    _both(gpu, (q, k, v, prefix, begins, table, own * 0))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_sequences_with_values_that_are_not_finite(gpu, dtype):
    rng = np.random.default_rng(14)
    q, k, v, prefix, begins, table, lens = _make(rng, [20] * 140, [100, 90], 2, 4, 2, 64, 16, dtype)
    v[int(prefix[1, 2]), 1, 3, 5] = math.inf  # seen by the second prefix's sequences, by kv head 1
    v[int(table[1, 1]), 0, 3, 9] = math.nan   # slot 19: seen by the last query alone
    v[int(table[2, 0]), 0, 3, 7] = -math.inf
    out, _ = _run(gpu, (q, k, v, prefix, begins, table, lens))
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[70:, :, 2:, 5] = True
    bad[1, 1, :2, 9] = True
    bad[2, :, :2, 7] = True
    assert torch.equal(~torch.isfinite(out.cpu().float()), bad)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,queries,group", [(64, 1, 5), (64, 1, 20), (64, 3, 3), (128, 1, 6), (128, 3, 2), (128, 5, 4),
                                               (256, 1, 5), (256, 2, 12), (80, 2, 12), (192, 2, 3)])
def test_one_launch(gpu, dtype, dim, queries, group):
    """Too few sequences to make the outputs, too many rows for the kernel of few, and tiles that fill less than the card:
    a prefix's tiles and the sequences' own slots side by side, in one chunk of these and in several."""
    rng = np.random.default_rng(dim + queries)
    batch, kv_heads = 39, 2
    for longest in (150, 900):
        lens = [0 if i % 11 == 5 else queries + (i * 7) % longest for i in range(batch)]
        lens[0] = longest
        args = _make(rng, lens, [333, 0, 1070], queries, kv_heads * group, kv_heads, dim, 16, dtype, fill=math.nan)
        q, k, v, prefix, begins, table, own = args
        counts = torch.from_numpy(rng.integers(-1, queries + 3, batch).astype(np.int32))
        _both(gpu, args, counts=counts)
        table, prefix = table.clone(), prefix.clone()
        table[3], table[7, 0], prefix[0, [1, 5]] = -1, 99999, -1
        _both(gpu, (q, k, v, prefix, begins, table, own))
        _both(gpu, (q, k, v, prefix, begins * 0, table, own))
    _both(gpu, (q, k, v, prefix, begins, table, own * 0))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_launch_with_values_that_are_not_finite(gpu, dtype):
    rng = np.random.default_rng(15)
    q, k, v, prefix, begins, table, lens = _make(rng, [20] * 40, [100, 90], 2, 4, 2, 64, 16, dtype)
    v[int(prefix[1, 2]), 1, 3, 5] = math.inf  # seen by the second prefix's sequences, by kv head 1
    v[int(table[1, 1]), 0, 3, 9] = math.nan   # slot 19: seen by the last query alone
    v[int(table[2, 0]), 0, 3, 7] = -math.inf
    out, _ = _run(gpu, (q, k, v, prefix, begins, table, lens))
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[20:, :, 2:, 5] = True
    bad[1, 1, :2, 9] = True
    bad[2, :, :2, 7] = True
    assert torch.equal(~torch.isfinite(out.cpu().float()), bad)


def _wide(args, slots=6000):
    """The same with room for many slots in the tables, by which both parts are split."""
    q, k, v, prefix, begins, table, lens = args
    pad = torch.full((prefix.shape[0], -(-slots // k.shape[2])), -1, dtype=torch.int32)
    return q, k, v, torch.cat([prefix, pad], 1).contiguous(), begins, table, lens


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 16, 17, 31, 32, 33, 64, 65, 129, 260])
def test_wide_tables_rows_around_the_tiles(gpu, dtype, rows):
    rng = np.random.default_rng(rows)
    for slots in (2000, 20000):
        _both(gpu, _wide(_make(rng, [3] * rows, [150], 1, 1, 1, 64, 16, dtype), slots))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch", [4, 40, 80])
def test_wide_tables_prefixes_around_the_tiles(gpu, dtype, dim, batch):
    rng = np.random.default_rng(dim + batch)
    for prefix in (1, 31, 33, 64, 65, 127, 129, 257, 513):
        _both(gpu, _wide(_make(rng, [2] * batch, [prefix], 1, 1, 1, dim, 16, dtype)))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch", [3, 40, 130])
@pytest.mark.parametrize("dim", [40, 64, 128, 256])
def test_wide_tables_unused_slots_and_pages(gpu, dtype, batch, dim):
    rng = np.random.default_rng(5)
    args = _wide(_make(rng, [20 + i % 3 for i in range(batch)], [77], 1, 2, 1, dim, 16, dtype, fill=math.nan))
    _both(gpu, args)
    q, k, v, prefix, begins, table, lens = args
    prefix, table = prefix.clone(), table.clone()
    prefix[0, [0, 3]] = torch.tensor([-1, 99999], dtype=torch.int32)
    table[0] = -1
    _both(gpu, (q, k, v, prefix, begins, table, lens))
    _both(gpu, (q, k, v, prefix, begins * 0, table, lens))
    _both(gpu, (q, k, v, prefix, begins, table, lens * 0))
    out, lse = _both(gpu, (q, k, v, prefix * 0 - 1, begins, table * 0 - 1, lens))
    assert not bool(out.any()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch", [3, 40, 130])
@pytest.mark.parametrize("wide", [False, True])
def test_queries_in_front_of_their_first_slot(gpu, dtype, batch, wide):
    """More queries than own slots: the first see the prefix alone, those from counts on nothing; values that are not
    finite reach those that see them."""
    rng = np.random.default_rng(16)
    lens = [i % 5 for i in range(2 * batch)]
    q, k, v, prefix, begins, table, own = _make(rng, lens, [100, 90], 4, 4, 2, 64, 16, dtype, fill=math.nan)
    args = q, k, v, prefix, begins, table, own
    args = _wide(args) if wide else args
    _both(gpu, args)
    counts = torch.tensor([(3 * i) % 7 - 1 for i in range(2 * batch)], dtype=torch.int32)
    _both(gpu, args, counts=counts)
    v[int(table[4, 0]), 0, 3, 9] = math.inf  # sequence 4's newest slot: its last query's alone
    v[int(prefix[0, 2]), 1, 3, 5] = math.nan
    out, _ = _run(gpu, args)
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[:batch, :, 2:, 5] = True
    bad[4, 3, :2, 9] = True
    assert torch.equal(~torch.isfinite(out.cpu().float()), bad)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-30])
def test_wide_tables_scales(gpu, dtype, scale):
    rng = np.random.default_rng(17)
    for batch in (2, 40, 140):
        args = _wide(_make(rng, [7] * batch, [130], 1, 4, 2, 64, 16, dtype, q_scale=1.0))
        _both(gpu, args, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch", [2, 40, 140])
def test_wide_tables_scores_that_grow_and_shrink(gpu, dtype, batch):
    rng = np.random.default_rng(18)
    for slope in (0.5, -0.5):
        q, k, v, prefix, begins, table, lens = _make(rng, [40] * batch, [1500], 1, 4, 2, 64, 8, dtype)
        q[..., 0] = 8.0
        for i in range(1500):
            k[int(prefix[0, i // 8]), 0, i % 8, 0] = slope * i
        _both(gpu, (q, k, v, prefix, begins, table, lens))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch", [3, 30, 130])
def test_wide_tables_layouts(gpu, dtype, batch):
    from tallax_amd import kvcache
    rng = np.random.default_rng(19)
    args = _wide(_make(rng, [9 + i % 9 for i in range(batch)], [500], 2, 4, 2, 48, 8, dtype))
    want = _both(gpu, args)
    q, k, v, *rest = (x.to(gpu) for x in args)
    k2, v2 = (y.transpose(1, 2).contiguous().transpose(1, 2) for y in (k, v))
    big = torch.zeros((batch, 2, 12, 48), dtype=dtype, device=gpu)
    big[:, :, 4:8] = q
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    for qq, kk, vv in ((q, k2, v2), (big[:, :, 4:8], k, v), (turned, k2, v)):
        assert all(torch.equal(a, b) for a, b in zip(kvcache.decode_shared(qq, kk, vv, *rest), want, strict=True))
