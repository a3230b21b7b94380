"""GPU: kvcache.append_rotated against its formula in 64 bits, at the layouts, types and masks where it can go wrong."""
import numpy as np
import pytest
import torch

from tests import layer_ref as L
from tests import serving_ref as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _tokens(rng, batch, tokens, heads, kv_heads, dim, dtype):
    x = torch.from_numpy(rng.standard_normal((batch, tokens, heads + 2 * kv_heads, dim)).astype(np.float32) * 2).to(dtype)
    return x, (x[:, :, :heads], x[:, :, heads:heads + kv_heads], x[:, :, heads + kv_heads:])


def _parts(x, heads, kv_heads):
    return x[:, :, :heads], x[:, :, heads:heads + kv_heads], x[:, :, heads + kv_heads:]


def _frequencies(pairs, base=1e4):
    return (base ** (-np.arange(pairs) / pairs)).astype(np.float32)


def _check(got, want, rooms):
    k, v, lens, q = got
    wk, wv, wl, wq = want
    assert torch.equal(lens.cpu(), wl)
    assert torch.equal(v.cpu().double(), wv)
    for name, x, y, room in (("q", q, wq, rooms[1]), ("k", k, wk, rooms[0])):
        off = (x.cpu().double() - y).abs()
        worst = (off - room).max() if off.numel() else torch.tensor(0.0)
        assert bool((off <= room).all()), (name, float(worst), float(off.max()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch,tokens,heads,kv_heads,dim,pairs,page", [
    (1, 1, 8, 2, 64, 32, 16), (3, 5, 6, 3, 128, 64, 8), (2, 7, 4, 4, 80, 40, 24), (2, 3, 5, 1, 40, 17, 1),
    (1, 33, 7, 7, 256, 128, 100), (5, 1, 2, 2, 8, 4, 3), (2, 9, 3, 1, 72, 36, 16), (4, 2, 4, 2, 128, 16, 16),
    (2, 2, 3, 2, 96, 1, 8), (1, 4, 48, 16, 192, 96, 32)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_shapes(gpu, dtype, batch, tokens, heads, kv_heads, dim, pairs, page, interleaved):
    from tallax_amd import kvcache
    rng = np.random.default_rng(1000 * batch + dim + pairs)
    lens = rng.integers(0, 30, batch)
    width = -(-(30 + tokens) // page)
    k, v, table = R.make_cache(rng, batch, kv_heads, dim, page, width, lens + tokens, dtype)
    x, (q, kn, vn) = _tokens(rng, batch, tokens, heads, kv_heads, dim, dtype)
    f = torch.from_numpy(_frequencies(pairs))
    lens_t = torch.tensor(lens, dtype=torch.int32)
    *want, room_k, room_q = L.append_rotated(k, v, table, lens_t, q, kn, vn, f, interleaved=interleaved)
    dk, dv = k.to(gpu), v.to(gpu)
    new, out = kvcache.append_rotated(dk, dv, table.to(gpu), lens_t.to(gpu), *_parts(x.to(gpu), heads, kv_heads),
                                      f.to(gpu), interleaved=interleaved)
    _check((dk, dv, new, out), want, (room_k, room_q))


def _case(gpu, rng, batch=3, tokens=6, heads=4, kv_heads=2, dim=64, pairs=24, page=8, dtype=BF16, lens=(5, 0, 21), **kw):
    """One call of the operator and the same of the plain form."""
    from tallax_amd import kvcache
    spare = kw.pop("table", None)
    width = -(-(max(lens) + tokens) // page)
    k, v, table = R.make_cache(rng, batch, kv_heads, dim, page, width, np.asarray(lens) + tokens, dtype)
    if spare is not None:
        table = spare(table)
    x, (q, kn, vn) = _tokens(rng, batch, tokens, heads, kv_heads, dim, dtype)
    f = torch.from_numpy(kw.pop("frequencies", _frequencies(pairs)))
    lens_t = torch.tensor(lens, dtype=torch.int32)
    *want, room_k, room_q = L.append_rotated(k, v, table, lens_t, q, kn, vn, f, **kw)
    dk, dv = k.to(gpu), v.to(gpu)
    moved = {n: y.to(gpu) if isinstance(y, torch.Tensor) else y for n, y in kw.items()}
    new, out = kvcache.append_rotated(dk, dv, table.to(gpu), lens_t.to(gpu), *_parts(x.to(gpu), heads, kv_heads),
                                      f.to(gpu), **moved)
    _check((dk, dv, new, out), want, (room_k, room_q))
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_several_axes(gpu, dtype, interleaved):
    rng = np.random.default_rng(2)
    places = torch.from_numpy(rng.integers(-50, 5000, (3, 6, 3)).astype(np.int32))
    for axes in (np.arange(24) % 3, np.repeat([0, 1, 2], 8), rng.integers(-2, 6, 24)):  # out of range: clamped
        _case(gpu, rng, dtype=dtype, token_positions=places, pair_axes=torch.from_numpy(axes.astype(np.int32)),
              interleaved=interleaved)
    _case(gpu, rng, dtype=dtype, token_positions=places[..., :1].contiguous(), pair_axes=torch.zeros(24, dtype=torch.int32))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_far_and_strange_positions(gpu, dtype):
    rng = np.random.default_rng(3)
    far = torch.tensor([[0, 1, -1, 131071, 1000003, 2 ** 24 + 1], [2 ** 31 - 1, -2 ** 31, 7, 2 ** 30, 12345678, 99999999],
                        [5, 5, 5, 4, 3, 2]], dtype=torch.int32)
    _case(gpu, rng, dtype=dtype, token_positions=far)
    _case(gpu, rng, dtype=dtype, token_positions=far, frequencies=np.linspace(0.0, 3.2, 24).astype(np.float32))


@pytest.mark.parametrize("tokens", [1, 6, 130])
def test_counts_and_seen(gpu, tokens):
    rng = np.random.default_rng(4)
    for counts in ([0, 1, tokens], [-3, tokens + 5, tokens // 2]):
        c = torch.tensor(counts, dtype=torch.int32)
        out = _case(gpu, rng, tokens=tokens, counts=c)
        for b, n in enumerate(counts):
            assert not bool(out[b, max(n, 0):].any())
        _case(gpu, rng, tokens=tokens, counts=c, seen=torch.tensor([700, 0, 31], dtype=torch.int32))


def test_tokens_that_have_no_slot(gpu):
    """Past the table's end, in no page, or in a page that is none of the pool: dropped, their queries rotated."""
    rng = np.random.default_rng(5)

    def spoil(table):
        t = table.clone()
        t[0, 1], t[1, 0], t[2, -1] = -1, 9999, -7
        return t
    _case(gpu, rng, table=spoil)
    _case(gpu, rng, table=lambda t: t[:, :2].contiguous(), lens=(5, 0, 12))
    _case(gpu, rng, table=lambda t: t[:, :0].contiguous(), lens=(0, 0, 0))


def test_scores_and_positions(gpu):
    from tallax_amd import kvcache
    rng = np.random.default_rng(6)
    k, v, table = R.make_cache(rng, 2, 2, 64, 8, 4, [20, 9], F32)
    x, _ = _tokens(rng, 2, 3, 4, 2, 64, F32)
    q, kn, vn = _parts(x.to(gpu), 4, 2)
    lens = torch.tensor([17, 6], dtype=torch.int32, device=gpu)
    seen = torch.tensor([170, 60], dtype=torch.int32, device=gpu)
    both = []
    for rotated in (False, True):
        dk, dv, t = k.to(gpu), v.to(gpu), table.to(gpu)
        scores = torch.full((2, 2, 32), 5.0, device=gpu)
        positions = torch.full((2, 2, 32), 77, dtype=torch.int32, device=gpu)
        kw = dict(scores=scores, positions=positions, seen=seen)
        if rotated:
            new, _ = kvcache.append_rotated(dk, dv, t, lens, q, kn, vn, torch.zeros(32, device=gpu), **kw)
        else:
            new = kvcache.append(dk, dv, t, lens, kn, vn, **kw)
        both.append((dk, dv, new, scores, positions))
    assert all(torch.equal(a, b) for a, b in zip(*both, strict=True))  # angles of 0: the append without rotation


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(gpu, dtype):
    """Pools with heads and slots in the other order, inputs at odd addresses and strides."""
    from tallax_amd import kvcache
    rng = np.random.default_rng(7)
    k, v, table = R.make_cache(rng, 2, 2, 48, 8, 4, [20, 9], dtype)
    x, _ = _tokens(rng, 2, 5, 4, 2, 48, dtype)
    lens = torch.tensor([12, 3], dtype=torch.int32, device=gpu)
    f = torch.from_numpy(_frequencies(24)).to(gpu)
    want = None
    for layout in range(4):
        dk, dv = k.to(gpu), v.to(gpu)
        q, kn, vn = _parts(x.to(gpu), 4, 2)
        places = None
        if layout == 1:
            dk, dv = (y.transpose(1, 2).contiguous().transpose(1, 2) for y in (dk, dv))
        if layout == 2:  # off 16 bytes, and the last axis not dense
            odd = torch.empty(x.numel() + 1, dtype=dtype, device=gpu)[1:].view(x.shape).copy_(x)
            q, kn, vn = _parts(odd, 4, 2)
            q = q.transpose(2, 3).contiguous().transpose(2, 3)
        if layout == 3:
            q, kn, vn = (y.transpose(1, 2).contiguous().transpose(1, 2) for y in (q, kn, vn))
            places = (lens[:, None] + torch.arange(5, device=gpu)).to(torch.int32).t().contiguous().t()
        new, out = kvcache.append_rotated(dk, dv, table.to(gpu), lens, q, kn, vn, f, token_positions=places)
        assert out.is_contiguous()
        got = (dk, dv, new, out)
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True)), layout


def test_values_that_are_not_finite(gpu):
    """A rotated pair that holds one has what the formula gives; other elements and tokens do not see it."""
    from tallax_amd import kvcache
    rng = np.random.default_rng(8)
    k, v, table = R.make_cache(rng, 1, 1, 64, 8, 4, [20], BF16)
    x, _ = _tokens(rng, 1, 3, 1, 1, 64, BF16)
    x[0, 1, 0, 5], x[0, 1, 1, 33], x[0, 1, 2, 7], x[0, 2, 0, 63] = np.inf, np.nan, -np.inf, np.nan
    lens = torch.tensor([10], dtype=torch.int32, device=gpu)
    f = torch.from_numpy(_frequencies(24)).to(gpu)
    dk, dv = k.to(gpu), v.to(gpu)
    _, out = kvcache.append_rotated(dk, dv, table.to(gpu), lens, *_parts(x.to(gpu), 1, 1), f)
    bad = torch.zeros((3, 64), dtype=torch.bool)
    bad[1, [5, 29]] = bad[2, 63] = True
    assert torch.equal(~torch.isfinite(out[0, :, 0].cpu().float()), bad)
    page, off = int(table[0, 1]), 3
    key = dk[page, 0, off].cpu().float()
    assert (~torch.isfinite(key)).nonzero()[:, 0].tolist() == [9, 33]
    assert float(dv[page, 0, off, 7]) == -np.inf


def test_no_tokens_and_no_sequences(gpu):
    from tallax_amd import kvcache
    rng = np.random.default_rng(9)
    k, v, table = (y.to(gpu) for y in R.make_cache(rng, 2, 2, 64, 8, 4, [20, 9], F32))
    lens = torch.tensor([12, 3], dtype=torch.int32, device=gpu)
    f = torch.ones(32, device=gpu)
    x = torch.zeros((2, 0, 8, 64), device=gpu)
    before = k.clone()
    new, out = kvcache.append_rotated(k, v, table, lens, *_parts(x, 4, 2), f)
    assert torch.equal(new, lens) and out.shape == (2, 0, 4, 64) and torch.equal(k, before)
    x = torch.zeros((0, 3, 8, 64), device=gpu)
    new, out = kvcache.append_rotated(k, v, table[:0], lens[:0], *_parts(x, 4, 2), f)
    assert new.shape == (0,) and out.shape == (0, 3, 4, 64)


def test_refusals(gpu):
    from tallax_amd import kvcache
    rng = np.random.default_rng(10)
    k, v, table = (y.to(gpu) for y in R.make_cache(rng, 2, 2, 64, 8, 4, [20, 9], F32))
    lens = torch.tensor([12, 3], dtype=torch.int32, device=gpu)
    x = torch.zeros((2, 3, 8, 64), device=gpu)
    q, kn, vn = _parts(x, 4, 2)
    f = torch.ones(32, device=gpu)
    i32 = dict(dtype=torch.int32, device=gpu)
    good = dict(q=q, k_new=kn, v_new=vn, frequencies=f)
    for over in (dict(q=q[:1]), dict(q=q[:, :2]), dict(q=q[..., :32]), dict(q=q.bfloat16()), dict(k_new=kn[:, :, :1]),
                 dict(v_new=vn[:, :2]), dict(k_new=kn.bfloat16()), dict(frequencies=torch.ones(33, device=gpu)),
                 dict(frequencies=f.double()), dict(frequencies=f[:0]), dict(frequencies=f[None]), dict(q=q.cpu()),
                 dict(token_positions=torch.zeros((2, 3))), dict(token_positions=torch.zeros((2, 4), **i32)),
                 dict(token_positions=torch.zeros((2, 3, 1), **i32)), dict(pair_axes=torch.zeros(32, **i32)),
                 dict(token_positions=torch.zeros((2, 3), **i32), pair_axes=torch.zeros(32, **i32)),
                 dict(token_positions=torch.zeros((2, 3, 0), **i32), pair_axes=torch.zeros(32, **i32)),
                 dict(token_positions=torch.zeros((2, 3, 2), **i32), pair_axes=torch.zeros(31, **i32)),
                 dict(counts=lens[:1]), dict(seen=lens.long()), dict(scores=torch.zeros((2, 2, 32), device=gpu))):
        a = {**good, **over}
        with pytest.raises(ValueError):
            kvcache.append_rotated(k, v, table, lens, a.pop("q"), a.pop("k_new"), a.pop("v_new"), a.pop("frequencies"), **a)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,pairs", [(128, 33), (80, 20), (80, 36), (192, 65), (96, 9), (128, 60), (24, 8), (40, 16),
                                       (128, 63), (24, 9), (256, 124), (16, 5)])
def test_halves_off_the_vectors(gpu, dtype, dim, pairs):
    """Halves of any number of pairs, also with tokens that do not count and tokens that have no slot."""
    rng = np.random.default_rng(dim + pairs)
    for tokens, heads, kv_heads in ((1, 4, 2), (9, 8, 8), (3, 40, 20)):
        counts = torch.tensor([tokens, 0, tokens - 1], dtype=torch.int32)
        _case(gpu, rng, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, pairs=pairs, dtype=dtype)
        out = _case(gpu, rng, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, pairs=pairs, dtype=dtype, counts=counts)
        assert not bool(out[1].any()) and not bool(out[2, -1].any())

        def cut(table):
            table = table.clone()
            table[:, 1] = -1
            return table

        _case(gpu, rng, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, pairs=pairs, dtype=dtype, table=cut)
