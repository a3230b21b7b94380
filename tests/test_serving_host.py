"""Host checks of the serving-step entry points (no GPU): every refusal comes before a launch, workspaces are as
documented, and the plain forms that the GPU tests compare with agree with a dense computation."""
import math

import numpy as np
import torch

from tests import serving_ref as R


def _cache(**over):
    from tallax_amd import _lib
    f = dict(k=4096, v=8192, dtype=_lib.BF16, dim=64, pages=10, kv_heads=2, page_size=16, k_stride_page=2048,
             k_stride_head=1024, k_stride_slot=64, v_stride_page=2048, v_stride_head=1024, v_stride_slot=64,
             block_table=4096, batch=3, table_width=4)
    f.update(over)
    return _lib.KvCache(**f)


def _decode(c, **over):
    import ctypes
    from tallax_amd import _lib
    a = dict(q=16, qb=256, qt=256, qh=64, queries=1, heads=4, scale=0.125, lens=4, counts=None, max_len=64,
             scores=None, out=16, lse=4, out_scores=None, ws=None, nws=0, stream=None)
    a.update(over)
    return _lib.LIB.tallax_kv_decode(ctypes.byref(c), *a.values())


def test_decode_refuses_on_the_host():
    from tallax_amd import _lib
    inv, uns = _lib.INVALID_ARGUMENT, _lib.UNSUPPORTED
    for over, st in ((dict(dtype=2), uns), (dict(dim=60), uns), (dict(dim=264), uns), (dict(dim=0), uns),
                     (dict(pages=-1), inv), (dict(kv_heads=0), inv), (dict(page_size=0), inv), (dict(k=None), inv),
                     (dict(block_table=None), inv), (dict(k=4098), uns), (dict(k_stride_slot=65), uns),
                     (dict(v_stride_page=-2048), uns), (dict(batch=70000), uns), (dict(page_size=1 << 21), uns),
                     (dict(table_width=1 << 22), uns), (dict(pages=1 << 31), uns), (dict(k_stride_slot=1 << 27), uns)):
        assert _decode(_cache(**over)) == st, over
        assert _lib.LIB.tallax_last_error()
    c = _cache()
    for over, st in ((dict(queries=0), inv), (dict(queries=2000), inv), (dict(heads=3), inv), (dict(heads=0), inv),
                     (dict(q=None), inv), (dict(lens=None), inv), (dict(out=None), inv), (dict(max_len=65), inv),
                     (dict(max_len=-1), inv), (dict(scale=math.nan), inv), (dict(scale=math.inf), inv),
                     (dict(scores=4), inv), (dict(out_scores=4), inv), (dict(q=18), uns), (dict(qh=63), uns),
                     (dict(qb=-256), uns), (dict(queries=1024, heads=64), uns),
                     (dict(scores=4, out_scores=4), _lib.WORKSPACE_TOO_SMALL)):
        assert _decode(c, **over) == st, over
    assert _decode(_cache(batch=0)) == _lib.OK


def test_decode_refuses_pools_past_its_offsets():
    from tallax_amd import _lib
    far = dict(dim=8, page_size=1, kv_heads=1, k_stride_page=24, v_stride_page=24, k_stride_slot=8, v_stride_slot=8)
    assert _decode(_cache(pages=2 ** 31 - 1, **far), heads=1, max_len=4, q=None) == _lib.INVALID_ARGUMENT
    assert _decode(_cache(pages=2 ** 31 - 1, **far), heads=1, max_len=4) == _lib.UNSUPPORTED  # 2^31 x 48 bytes
    assert b"2^32" in _lib.LIB.tallax_last_error()


def test_append_evict_refuse_on_the_host():
    import ctypes
    from tallax_amd import _lib
    L, inv, uns, c = _lib.LIB, _lib.INVALID_ARGUMENT, _lib.UNSUPPORTED, ctypes.byref(_cache())
    app = lambda lens=4, cnt=None, k=16, v=16, t=1, s=None, p=None, seen=None, out=8: \
        L.tallax_kv_append(c, lens, cnt, k, v, t, s, p, seen, out, None)  # noqa: E731
    for kw, st in ((dict(lens=None), inv), (dict(out=4), inv), (dict(k=None), inv), (dict(t=-1), inv),
                   (dict(s=4), inv), (dict(s=4, p=4), inv), (dict(k=24), uns)):
        assert app(**kw) == st, kw
    ev = lambda budget=8, recent=0, sinks=0, lens=4, sc=4, os=8, ws=256, n=1 << 20: \
        L.tallax_kv_evict(c, lens, sc, 4, 4, budget, recent, sinks, 4, os, 8, ws, n, None)  # noqa: E731
    for kw, st in ((dict(budget=0), inv), (dict(recent=-1), inv), (dict(sinks=9), inv), (dict(recent=5, sinks=4), inv),
                   (dict(lens=None), inv), (dict(sc=None), inv), (dict(os=4), inv),
                   (dict(ws=None), _lib.WORKSPACE_TOO_SMALL), (dict(n=100), _lib.WORKSPACE_TOO_SMALL)):
        assert ev(**kw) == st, kw
    assert L.tallax_kv_evict_workspace_size(c, 8) == 6 * 17 * 4


def test_verify_refuses_on_the_host():
    from tallax_amd import _lib
    L, inv, uns = _lib.LIB, _lib.INVALID_ARGUMENT, _lib.UNSUPPORTED

    def ver(draft=4, logits=4, dt=0, b=2, t=3, v=100, counts=None, temp=4, probs=None, qdt=0, u=4, noise=4, tok=4,
            acc=4, ws=256, n=1 << 20):
        return L.tallax_verify(draft, logits, dt, b, t, v, counts, temp, probs, qdt, u, noise, tok, acc, ws, n, None)

    for kw, st in ((dict(v=0), inv), (dict(b=-1), inv), (dict(t=64), uns), (dict(b=20000), uns), (dict(dt=2), uns),
                   (dict(probs=4, qdt=2), uns), (dict(draft=None), inv), (dict(temp=None), inv), (dict(u=None), inv),
                   (dict(noise=None), inv), (dict(tok=None), inv), (dict(ws=None), _lib.WORKSPACE_TOO_SMALL),
                   (dict(n=64), _lib.WORKSPACE_TOO_SMALL)):
        assert ver(**kw) == st, kw
    assert ver(b=0) == _lib.OK


def test_attention_reference_is_dense_attention():
    rng = np.random.default_rng(0)
    lens = [37, 5]
    k, v, table = R.make_cache(rng, 2, 2, 16, 8, 6, lens, torch.float32)
    q = torch.from_numpy(rng.standard_normal((2, 3, 4, 16)))
    scores = torch.zeros((2, 2, 48))
    out, lse, new, _ = R.attention(q, k, v, table, torch.tensor(lens), 0.25, None, scores)
    for b, n in enumerate(lens):
        ks = torch.stack([k[table[b, s // 8], :, s % 8] for s in range(n)]).double()
        vs = torch.stack([v[table[b, s // 8], :, s % 8] for s in range(n)]).double()
        x = torch.einsum("thd,shd->hts", q[b], ks.repeat_interleave(2, 1)) * 0.25
        x = x.masked_fill(torch.arange(n) > torch.arange(n - 3, n)[:, None], -math.inf)
        w = x.softmax(-1)
        assert torch.allclose(out[b], torch.einsum("hts,shd->thd", w, vs.repeat_interleave(2, 1)))
        assert torch.allclose(lse[b], x.logsumexp(-1).t())
        assert torch.allclose(new[b, :, :n], w.sum(1).reshape(2, 2, n).sum(1))
    assert torch.allclose(new.sum((1, 2)), torch.full((2,), 12.0, dtype=torch.float64))


def test_verify_reference_keeps_the_target():
    """Summed over what the draft may be, the first token has the target's distribution exactly: min(p, q) accepted
    plus the refused mass spread as max(p - q, 0)."""
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((1, 2, 6))
    p = np.exp(logits[0, 0]) / np.exp(logits[0, 0]).sum()
    q = rng.dirichlet(np.ones(6))
    n = 4000
    draft = rng.choice(6, (n, 1), p=q).astype(np.int32)
    tokens, _, _ = R.verify(draft, np.repeat(logits, n, 0), rng.random((n, 1)), rng.exponential(size=(n, 6)),
                            np.repeat(q[None, None], n, 0), np.ones(n))
    freq = np.bincount(tokens[:, 0], minlength=6) / n
    assert (np.abs(freq - p) < 5 * np.sqrt(p * (1 - p) / n)).all()


def test_evict_reference_on_a_small_case():
    k = torch.arange(8.0).reshape(1, 1, 8, 1)
    table = torch.zeros((1, 1), dtype=torch.int32)
    scores = torch.tensor([[[0.1, 5.0, 0.2, 0.3, 9.0, 0.0, 7.0, 1.0]]])
    pos = torch.arange(8, dtype=torch.int32).reshape(1, 1, 8)
    lens = torch.tensor([7], dtype=torch.int32)
    kk, _, n, s, p = R.evict(k, k, table, lens, scores, pos, lens, 4, 1, 1)
    # kept: position 0 (sink), 6 (newest), then scores 9 (slot 4) and 5 (slot 1); 4 and 6 move into 2 and 3
    assert n.tolist() == [4] and p[0, 0].tolist() == [0, 1, 4, 6, -1, -1, -1, -1]
    assert kk.flatten().tolist() == [0.0, 1.0, 4.0, 6.0, 4.0, 5.0, 6.0, 7.0]
    assert torch.equal(s[0, 0, :4], torch.tensor([0.1, 5.0, 9.0, 7.0]))
