"""Host checks of kvcache.append_rotated, kvcache.decode_shared and experts.route (no GPU): every refusal comes before a
launch, workspaces are as documented, and the plain forms that the GPU tests compare with agree with other ways to them."""
import ctypes
import math

import numpy as np
import torch

from tests import layer_ref as L
from tests import serving_ref as R
from tests.test_serving_host import _cache


def _rotate(c, lens=4, counts=None, scores=None, positions=None, seen=None, out_q=16, out=8, q=16, k=16, v=16, tokens=1,
            heads=4, batch_at=(256, 128, 128), token_at=(256, 128, 128), head_at=(64, 64, 64), f=16, pairs=32,
            neighbours=0, places=None, axes=1, pair_axes=None):
    from tallax_amd import _lib
    three = ctypes.c_int64 * 3
    fresh = _lib.KvTokens(q, k, v, tokens, heads, three(*batch_at), three(*token_at), three(*head_at))
    turn = _lib.Rotation(f, pairs, neighbours, places, axes, pair_axes)
    return _lib.LIB.tallax_kv_append_rotated(ctypes.byref(c), lens, counts, ctypes.byref(fresh), ctypes.byref(turn),
                                             scores, positions, seen, out_q, out, None)


def test_append_rotated_refuses_on_the_host():
    from tallax_amd import _lib
    inv, uns = _lib.INVALID_ARGUMENT, _lib.UNSUPPORTED
    assert _rotate(_cache(dim=60)) == uns and _rotate(_cache(kv_heads=0)) == inv
    c = _cache()
    for kw, st in ((dict(lens=None), inv), (dict(out=4), inv), (dict(out=None), inv), (dict(out_q=None), inv),
                   (dict(q=None), inv), (dict(k=None), inv), (dict(v=None), inv), (dict(f=None), inv),
                   (dict(tokens=-1), inv), (dict(tokens=1 << 25), inv), (dict(heads=0), inv), (dict(heads=70000), uns),
                   (dict(pairs=0), inv), (dict(pairs=33), inv), (dict(axes=0), inv), (dict(axes=2000), uns),
                   (dict(axes=3), inv), (dict(axes=3, places=4), inv), (dict(axes=3, pair_axes=4), inv),
                   (dict(scores=4), inv), (dict(positions=4), inv), (dict(scores=4, positions=4), inv),
                   (dict(q=24), uns), (dict(k=24), uns), (dict(v=17), uns), (dict(out_q=24), uns),
                   (dict(head_at=(60, 64, 64)), uns), (dict(token_at=(256, -128, 128)), uns),
                   (dict(batch_at=(256, 128, 4)), uns), (dict(tokens=(1 << 23) + 1), inv),
                   (dict(head_at=(1 << 31, 64, 64)), uns), (dict(token_at=(1 << 35, 128, 128)), uns)):
        assert _rotate(c, **kw) == st, kw
        assert _lib.LIB.tallax_last_error()
    assert _lib.LIB.tallax_kv_append_rotated(ctypes.byref(c), 4, None, None, None, None, None, None, 16, 8, None) == inv
    assert _rotate(_cache(batch=0)) == _lib.OK


def _shared(c, **over):
    from tallax_amd import _lib
    a = dict(table=4096, prefixes=1, width=4, prefix_lens=4, q=16, qb=256, qt=256, qh=64, queries=1, heads=4, scale=0.125,
             lens=4, counts=None, max_prefix=64, max_len=64, out=16, lse=4, ws=256, nws=1 << 30, stream=None)
    a.update(over)
    return _lib.LIB.tallax_kv_decode_shared(ctypes.byref(c), *a.values())


def test_decode_shared_refuses_on_the_host():
    from tallax_amd import _lib
    inv, uns = _lib.INVALID_ARGUMENT, _lib.UNSUPPORTED
    for over, st in ((dict(dtype=2), uns), (dict(dim=264), uns), (dict(page_size=0), inv), (dict(k=None), inv),
                     (dict(k_stride_slot=65), uns), (dict(k=None, table_width=0), inv)):
        assert _shared(_cache(**over), max_len=0) == st, over
    c = _cache()
    for over, st in ((dict(queries=0), inv), (dict(queries=2000), inv), (dict(heads=3), inv), (dict(heads=0), inv),
                     (dict(prefixes=0), inv), (dict(prefixes=2), inv), (dict(prefixes=-1), inv), (dict(width=-1), inv),
                     (dict(width=1 << 22), uns), (dict(queries=1024, heads=64), uns), (dict(scale=math.nan), inv),
                     (dict(scale=math.inf), inv), (dict(scale=1e39), inv), (dict(q=None), inv), (dict(lens=None), inv),
                     (dict(out=None), inv), (dict(prefix_lens=None), inv), (dict(table=None), inv), (dict(q=18), uns),
                     (dict(qh=63), uns), (dict(qb=-256), uns), (dict(out=24), uns), (dict(max_len=65), inv),
                     (dict(max_len=-1), inv), (dict(max_prefix=65), inv), (dict(max_prefix=-1), inv),
                     (dict(width=512, max_prefix=8192, ws=None), _lib.WORKSPACE_TOO_SMALL),
                     (dict(width=512, max_prefix=8192, nws=64), _lib.WORKSPACE_TOO_SMALL),
                     (dict(width=512, max_prefix=8192, ws=264), inv)):
        assert _shared(c, **over) == st, over
        assert _lib.LIB.tallax_last_error()
    far = dict(dim=8, page_size=1, kv_heads=1, k_stride_page=24, v_stride_page=24, k_stride_slot=8, v_stride_slot=8)
    assert _shared(_cache(pages=2 ** 31 - 1, **far), heads=1, max_len=4, max_prefix=4) == uns
    assert b"2^32" in _lib.LIB.tallax_last_error()
    many = _cache(batch=65535, pages=1 << 20)
    assert _shared(many, queries=256, heads=2, qt=128, nws=1 << 62) == uns
    assert b"workgroups" in _lib.LIB.tallax_last_error()
    assert _shared(_cache(batch=0), prefixes=0) == _lib.OK
    size = _lib.LIB.tallax_kv_decode_shared_workspace_size
    assert size(ctypes.byref(c), 2, 4, 1, 4, 64, 64) == 0 == size(ctypes.byref(c), 1, 4, 0, 4, 64, 64)
    assert size(ctypes.byref(c), 3, 4, 1, 4, 64, 64) == 0  # short ones need none
    assert size(ctypes.byref(c), 3, 512, 1, 4, 8192, 64) > 0
    assert size(ctypes.byref(c), 1, 512, 1, 4, -1, -1) == size(ctypes.byref(c), 1, 512, 1, 4, 8192, 64) > 0


def _route(**over):
    from tallax_amd import _lib
    a = dict(logits=16, dt=0, tokens=4, experts=64, stride=64, k=6, sigmoid=0, bias=None, groups=8, top_groups=4,
             group_top=2, renormalise=1, scale=1.0, weights=16, ids=16, stream=None)
    a.update(over)
    return _lib.LIB.tallax_route(*a.values())


def test_route_refuses_on_the_host():
    from tallax_amd import _lib
    inv, uns = _lib.INVALID_ARGUMENT, _lib.UNSUPPORTED
    for kw, st in ((dict(dt=2), uns), (dict(tokens=-1), inv), (dict(experts=0), inv), (dict(experts=65), inv),
                   (dict(groups=0), inv), (dict(groups=7), inv), (dict(top_groups=0), inv), (dict(top_groups=9), inv),
                   (dict(k=0), inv), (dict(k=33), inv), (dict(group_top=3), inv), (dict(stride=-1), inv),
                   (dict(scale=math.nan), inv), (dict(scale=math.inf), inv), (dict(scale=1e39), inv),
                   (dict(experts=2048), uns), (dict(experts=1024, groups=128, top_groups=128), uns),
                   (dict(experts=1024, groups=1, top_groups=1, k=65), uns), (dict(tokens=(1 << 25) + 1), uns),
                   (dict(logits=None), inv),
                   (dict(weights=None), inv), (dict(ids=None), inv)):
        assert _route(**kw) == st, kw
        assert _lib.LIB.tallax_last_error()
    assert _route(tokens=0, logits=None) == _lib.OK


def test_python_refusals_that_need_no_gpu():
    import pytest
    from tallax_amd import experts, kvcache
    x = torch.zeros(4, 8)
    for call in (lambda: experts.route(x, 2), lambda: experts.route(None, 2),
                 lambda: kvcache.append_rotated(*[x] * 8), lambda: kvcache.decode_shared(*[x] * 7)):
        with pytest.raises(ValueError, match="must be torch tensors"):
            call()


def test_rotation_reference_is_a_complex_product():
    rng = np.random.default_rng(0)
    x = torch.from_numpy(rng.standard_normal((5, 2, 16)).astype(np.float32))
    f = torch.from_numpy(rng.uniform(0.1, 1, 6).astype(np.float32))
    at = torch.tensor([0, 1, 7, 1000, -3], dtype=torch.int32)
    for interleaved in (False, True):
        y, _ = L.rotate(x, at, f, None, interleaved)
        low = torch.arange(6) * 2 if interleaved else torch.arange(6)
        high = low + 1 if interleaved else low + 6
        z = torch.complex(x[..., low].double(), x[..., high].double())
        z = z * torch.exp(1j * (at.double()[:, None] * f.double()))[:, None]
        assert torch.allclose(y[..., low], z.real) and torch.allclose(y[..., high], z.imag)
        assert torch.equal(y[..., 12:], x[..., 12:].double())
    assert torch.equal(L.rotate(x, at[:1].expand(5), f)[0], x.double())
    places = torch.stack([at, at * 2, at * 0], 1)
    axes = torch.tensor([0, 1, 2, 0, 1, 7])
    y, _ = L.rotate(x, places, f, axes)
    for i, a in enumerate((0, 1, 2, 0, 1, 2)):
        want, _ = L.rotate(x, places[:, a], f)
        assert torch.equal(y[..., [i, i + 6]], want[..., [i, i + 6]])


def test_shared_reference_is_attention_over_both_parts():
    """As serving_ref's attention over a cache that holds the prefix again in front of every sequence."""
    rng = np.random.default_rng(1)
    lens, begins, page = [9, 3, 17, 8], [13, 30], 8
    k, v, table = R.make_cache(rng, 4, 2, 16, page, 3, lens, torch.float32, spare=40)
    free = [i for i in range(k.shape[0]) if i not in set(table.flatten().tolist())]
    prefix = torch.full((2, 4), -1, dtype=torch.int32)
    prefix[0, :2], prefix[1, :4] = torch.tensor(free[:2]), torch.tensor(free[2:6])
    q = torch.from_numpy(rng.standard_normal((4, 2, 4, 16)))
    out, lse, _, _ = L.shared_attention(q, k, v, prefix, begins, table, lens, 0.25)
    flat_k, flat_v = (x.transpose(1, 2).reshape(-1, 2, 1, 16) for x in (k, v))  # pages of one slot
    rows = []
    for b, n in enumerate(lens):
        slots = [int(prefix[b // 2, s // page]) * page + s % page for s in range(begins[b // 2])]
        rows.append(slots + [int(table[b, s // page]) * page + s % page for s in range(n)])
    width = max(map(len, rows))
    whole = torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32)
    want, want_lse, _, _ = R.attention(q, flat_k, flat_v, whole, [len(r) for r in rows], 0.25)
    assert torch.allclose(out, want) and torch.allclose(lse, want_lse)


def test_route_reference_on_small_cases():
    x = np.array([[0.0, 2.0, 1.0, -1.0, 2.0, -np.inf]])
    w, ids, _ = L.route(x, 3, renormalise=False)
    p = np.exp(x[0]) / np.exp(x[0]).sum()
    assert ids[0].tolist() == [1, 4, 2] and np.allclose(w[0], p[[1, 4, 2]])
    w, ids, _ = L.route(x, 2, "sigmoid", bias=np.array([0.5, 0, 0, 0.8, 0, 9.0]))
    s = 1 / (1 + np.exp(-x[0]))
    assert ids[0].tolist() == [3, 0] and np.allclose(w[0], s[[3, 0]] / (s[3] + s[0]))
    # groups of two: sums 2 (of scores .5 + .88), .73 + .27, .88 and nothing
    _, ids, _ = L.route(x, 2, "sigmoid", groups=3, top_groups=1, group_score="top2")
    assert ids[0].tolist() == [1, 0]
    _, ids, _ = L.route(x, 4, "sigmoid", groups=3, top_groups=2, group_score="max")
    assert ids[0].tolist() == [1, 4, 0, 5]
    w, ids, _ = L.route(np.full((1, 4), -np.inf), 2, groups=2, top_groups=1)
    assert ids[0].tolist() == [0, 1] and (w == 0).all()
