"""GPU: experts.route against sorting in 64 bits: ids are equal, weights within their roundings."""
import numpy as np
import pytest
import torch

from tests import layer_ref as L
from tests.gpu_util import host_values, to_dev

pytestmark = pytest.mark.gpu


def _run(gpu, x, k, dtype="f32", bias=None, **kw):
    from tallax_amd import experts
    b = None if bias is None else torch.from_numpy(np.asarray(bias, np.float32)).to(gpu)
    w, ids = experts.route(to_dev(x, dtype, gpu), k, bias=b, **kw)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and w.shape == ids.shape == (x.shape[0], k)
    return w.cpu().numpy(), ids.cpu().numpy()


def _check(gpu, x, k, dtype="f32", bias=None, **kw):
    values = host_values(x.astype(np.float32), dtype).astype(np.float64)
    b = None if bias is None else np.asarray(bias, np.float32).astype(np.float64)
    want, ids, margin = L.route(values, k, bias=b, **kw)
    assert margin > 1e-13  # the device's 64-bit scores are off by less, so no choice is left open
    w, got = _run(gpu, x.astype(np.float32), k, dtype, bias, **kw)
    assert np.array_equal(got, ids), np.nonzero((got != ids).any(1))[0][:5]
    # a score in float32 (an exponential, a sum or a quotient: 8 half steps), a sum of k, a quotient, the scale; 2^-149:
    # the smallest step
    room = np.abs(want) * 32 * L.F32 + 2.0 ** -148
    assert (np.abs(w - want) <= room).all(), (np.abs(w - want) / room).max()
    return w, got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 8, 2), (3, 64, 6), (130, 60, 4), (65, 128, 8), (7, 160, 6),
                                              (33, 256, 8), (5, 384, 16), (9, 512, 10), (2, 1024, 64), (4, 700, 5), (1000, 16, 1)])
def test_shapes(gpu, dtype, score, tokens, experts, k):
    rng = np.random.default_rng(tokens + experts)
    x = rng.standard_normal((tokens, experts)) * 1.5
    for bias in (None, rng.standard_normal(experts) * 0.05):
        for renormalise, scale in ((True, 1.0), (False, 2.5)):
            _check(gpu, x, k, dtype, bias, score=score, renormalise=renormalise, scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("experts,groups,top_groups,k", [(64, 8, 3, 6), (60, 4, 2, 6), (256, 8, 4, 8), (160, 8, 3, 6),
                                                         (16, 16, 5, 3), (64, 64, 7, 7), (1024, 32, 3, 20), (12, 2, 1, 6),
                                                         (256, 4, 4, 8), (512, 8, 1, 64), (96, 3, 2, 8)])
def test_groups(gpu, dtype, score, group_score, experts, groups, top_groups, k):
    rng = np.random.default_rng(experts + groups)
    x = rng.standard_normal((37, experts)) * 1.5
    for bias in (None, rng.standard_normal(experts) * 0.05):
        _check(gpu, x, k, dtype, bias, score=score, groups=groups, top_groups=top_groups, group_score=group_score)


def test_defaults_are_a_softmax_top_k(gpu):
    """Without groups and bias the ids are tax.top_k's."""
    from tallax_amd import experts, tax
    rng = np.random.default_rng(1)
    x = to_dev((rng.standard_normal((50, 128)) * 2).astype(np.float32), "bf16", gpu)
    _, ids = experts.route(x, 8)
    assert torch.equal(ids, tax.top_k(x, 8)[1])
    w, _ = experts.route(x, 8)
    assert torch.allclose(w.sum(-1), torch.ones(50, device=gpu), atol=1e-6)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_ties_go_to_the_lowest(gpu, score, bias):
    rng = np.random.default_rng(2)
    x = rng.integers(-1, 2, (40, 96)).astype(np.float32)
    b = np.full(96, 0.25) if bias else None
    for groups, top in ((1, 1), (8, 3), (6, 6)):
        for how in ("max", "top2"):
            _check(gpu, x, 8, "f32", b, score=score, groups=groups, top_groups=top, group_score=how)
    _check(gpu, np.zeros((3, 96)), 12, "f32", b, score=score, groups=8, top_groups=2)


@pytest.mark.parametrize("bias", [False, True])
def test_scores_next_to_each_other(gpu, bias):
    """Logits that differ in their last bit, far from 0, where 32-bit scores tie, and biases that nearly cancel them."""
    rng = np.random.default_rng(3)
    base = rng.choice([0.0, 3.0, 9.0, -9.0], (60, 1)).astype(np.float32)
    x = np.tile(base, (1, 64))
    steps = rng.integers(0, 4, x.shape)
    for i in range(3):
        x = np.where(steps > i, np.nextafter(x, np.float32(99)), x).astype(np.float32)
    b = rng.choice([0.0, 2.0 ** -25, 2.0 ** -24], 64).astype(np.float32) if bias else None
    for score in ("sigmoid", "softmax"):
        _check(gpu, x, 8, "f32", b, score=score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_experts_that_are_not_there(gpu, score):
    """-inf, NaN and the type's lowest value among the logits, whole rows and groups of them, more chosen than there are."""
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((48, 64)) * 1.5).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 5:] = -np.inf
    x[3, ::2] = np.nan
    x[4, :56] = -np.inf
    x[5, 8:] = np.finfo(np.float32).min
    x[6] = np.finfo(np.float32).min
    x[7, 9] = np.inf
    x[8, [3, 40]] = np.inf
    x[9] = 100.0
    x[10, 1:] = -200.0
    x[11] = np.where(np.arange(64) % 8 == 0, x[11], -np.inf)
    bias = rng.standard_normal(64) * 0.05
    strange = bias.copy()
    strange[[3, 17]], strange[20], strange[21] = np.nan, np.inf, -np.inf
    for b in (None, bias, strange):
        for groups, top in ((1, 1), (8, 2)):
            for how in ("max", "top2"):
                kw = dict(score=score, groups=groups, top_groups=top, group_score=how)
                values = x.astype(np.float64)
                want, ids, margin = L.route(values, 8, bias=None if b is None else np.asarray(b, np.float32).astype(np.float64), **kw)
                w, got = _run(gpu, x, 8, "f32", b, **kw)
                assert np.array_equal(got, ids)
                assert (np.abs(w - want) <= np.abs(want) * 32 * L.F32 + 2.0 ** -148).all()
                assert np.isfinite(w).all()


def test_rows_at_any_stride(gpu):
    from tallax_amd import experts
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((21, 200)) * 1.5).astype(np.float32)
    for dtype in ("f32", "bf16"):
        d = to_dev(x, dtype, gpu)
        want = experts.route(d[:, 3:63].contiguous(), 5)
        for y in (d[:, 3:63], d.t().contiguous().t()[:, 3:63]):
            assert all(torch.equal(a, b) for a, b in zip(experts.route(y, 5), want, strict=True))
        one = d[:1, 3:63].expand(9, 60)
        got = experts.route(one, 5)
        assert all(torch.equal(a, b[:1].expand(9, 5)) for a, b in zip(got, want, strict=True))


def test_many_tokens(gpu):
    """More workgroups than the card holds at once; every row is as it is alone."""
    from tallax_amd import experts
    gen = torch.Generator(device=gpu)
    gen.manual_seed(6)
    x = torch.randn((20001, 96), generator=gen, device=gpu)
    b = torch.randn(96, generator=gen, device=gpu) * 0.05
    kw = dict(score="sigmoid", bias=b, groups=4, top_groups=2, group_score="top2")
    w, ids = experts.route(x, 6, **kw)
    for i in (0, 1, 777, 20000):
        w1, i1 = experts.route(x[i:i + 1], 6, **kw)
        assert torch.equal(w1, w[i:i + 1]) and torch.equal(i1, ids[i:i + 1])
    assert int(ids.min()) >= 0 and int(ids.max()) < 96
    assert bool((ids.sort(-1)[0].diff(dim=-1) > 0).all())
    w, ids = experts.route(x[:0], 6)
    assert w.shape == ids.shape == (0, 6)


def test_refusals(gpu):
    from tallax_amd import experts
    x = torch.zeros((4, 64), device=gpu)
    for kw in (dict(k=0), dict(k=65), dict(k=4, groups=7), dict(k=4, groups=0), dict(k=9, groups=8, top_groups=1),
               dict(k=4, groups=8, top_groups=9), dict(k=4, score="tanh"), dict(k=4, score=None),
               dict(k=4, group_score="sum"), dict(k=4, bias=torch.zeros(63, device=gpu)),
               dict(k=4, bias=torch.zeros(64, device=gpu).double()), dict(k=4, scale=float("nan")), dict(k=-1)):
        with pytest.raises(ValueError):
            experts.route(x, **kw)
    for y in (x[0], x.cpu(), x[:, :0]):
        with pytest.raises(ValueError):
            experts.route(y, 4)
    for y in (x.half(), x.int(), torch.zeros((4, 1025), device=gpu)):
        with pytest.raises(NotImplementedError):
            experts.route(y, 4)


def test_zeros_of_both_signs_tie(gpu):
    rng = np.random.default_rng(7)
    x = rng.choice([0.0, -0.0, 1e-30, -1.0], (50, 64)).astype(np.float32)
    for dtype in ("f32", "bf16"):
        for score in ("softmax", "sigmoid"):
            _check(gpu, x, 8, dtype, None, score=score)
            _check(gpu, x, 8, dtype, None, score=score, groups=8, top_groups=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_logits_and_biases(gpu, dtype):
    """Scores that saturate, that vanish, and biases far larger than them."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((40, 128)) * 30
    for score in ("softmax", "sigmoid"):
        for bias in (None, rng.standard_normal(128) * 100, rng.integers(-3, 4, 128) * 0.5):
            for groups, top in ((1, 1), (16, 4), (4, 1)):
                for how in ("max", "top2"):
                    kw = dict(score=score, groups=groups, top_groups=top, group_score=how)
                    values = host_values(x.astype(np.float32), dtype).astype(np.float64)
                    b = None if bias is None else np.asarray(bias, np.float32).astype(np.float64)
                    want, ids, margin = L.route(values, 8, bias=b, **kw)
                    w, got = _run(gpu, x.astype(np.float32), 8, dtype, bias, **kw)
                    if margin > 1e-13:
                        assert np.array_equal(got, ids), kw
                        assert (np.abs(w - want) <= np.abs(want) * 32 * L.F32 + 2.0 ** -148).all()
                    assert np.isfinite(w).all()


@pytest.mark.parametrize("k", [6, 7, 8, 15, 16])
@pytest.mark.parametrize("bias", [False, True])
def test_neighbours_that_rise_by_the_smallest_steps(gpu, k, bias):
    """The largest experts lie next to each other, and more of them than are chosen differ in their last bits alone."""
    x = np.full((9, 512), -3.0, np.float32)
    for t in range(9):
        x[t, 32 * t:32 * t + 32] = 1.0 + np.arange(32) * 2.0 ** -23
    b = np.zeros(512) if bias else None
    for groups, top in ((1, 1), (8, 2)):
        for score in ("softmax", "sigmoid"):
            _check(gpu, x, k, "f32", b, score=score, groups=groups, top_groups=top)
