"""GPU: experts.route where its 32-bit keys, ranks and sums leave a choice open, and where scores are far from 1."""
import numpy as np
import pytest
import torch

from tests import layer_ref as L
from tests.gpu_util import host_values
from tests.test_gpu_route import _check, _run

pytestmark = pytest.mark.gpu


def _rows(gpu, x, k, dtype="f32", bias=None, least=1.0, **kw):
    """As _check, row by row: those whose border leaves nothing open (a share of `least` of them, at least)."""
    values = host_values(x.astype(np.float32), dtype).astype(np.float64)
    b = None if bias is None else np.asarray(bias, np.float32).astype(np.float64)
    w, got = _run(gpu, x.astype(np.float32), k, dtype, bias, **kw)
    assert np.isfinite(w).all()
    checked = 0
    for t in range(len(x)):
        want, ids, margin = L.route(values[t:t + 1], k, bias=b, **kw)
        if margin <= 1e-13:  # the device's 64-bit scores are off by less
            continue
        checked += 1
        assert np.array_equal(got[t], ids[0]), (t, got[t], ids[0])
        assert (np.abs(w[t] - want[0]) <= np.abs(want[0]) * 32 * L.F32 + 2.0 ** -148).all(), t
    assert checked >= least * len(x), checked
    return w, got


# --- bfloat16 keys that hold the expert's number ---------------------------------------------------------------
@pytest.mark.parametrize("logits,groups,top_groups,k,want", [
    ([-1.0, -1.0, 149 / 1024, -10.0], 2, 1, 2, [0, 1]),  # ranks .5379 and .5364
    ([-1.40625, 1.0546875, -0.31835938, -1.9609375, 1.7890625, -1.0625, 0.578125, -0.859375], 4, 2, 3, [4, 1, 5])])
def test_ranks_of_negative_logits_by_hand(gpu, logits, groups, top_groups, k, want):
    x = np.tile(np.asarray(logits, np.float32), (5, 1))
    _, ids = _check(gpu, x, k, "bf16", score="sigmoid", groups=groups, top_groups=top_groups, group_score="top2")
    assert (ids == want).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("mean,spread", [(-3.0, 0.5), (-3.0, 1.5), (-8.0, 1.0), (0.0, 1.5)])
@pytest.mark.parametrize("experts,groups,top_groups,k", [(16, 8, 4, 3), (32, 16, 5, 6), (24, 8, 3, 4), (256, 8, 4, 8),
                                                         (60, 4, 2, 6), (48, 3, 1, 10)])
def test_ranks_of_negative_logits(gpu, score, mean, spread, experts, groups, top_groups, k):
    rng = np.random.default_rng(experts + groups)
    x = rng.standard_normal((1500, experts)) * spread + mean
    _rows(gpu, x, k, "bf16", score=score, groups=groups, top_groups=top_groups, group_score="top2", least=0.99)


# --- ranks past float32 -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("order", [0, 1, 2])
def test_ranks_past_float32(gpu, dtype, score, sign, order):
    """Biases whose sum of two leaves float32 (an infinite one counts as the largest number): ranks still differ."""
    rng = np.random.default_rng(order)
    x = rng.standard_normal((40, 16))
    small = np.asarray([3.0e38, 3.2e38, 2.1e38, 2.0e38])[np.roll(np.arange(4), order)]
    bias = np.zeros((4, 4)) if sign > 0 else np.full((4, 4), -np.inf)
    bias[:, 2], bias[:, 1] = sign * np.inf, sign * small
    for top_groups in (1, 2, 3):
        _check(gpu, x, 4 * top_groups, dtype, bias.reshape(-1), score=score, groups=4, top_groups=top_groups,
               group_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_masked_group_before_one_that_is_not_there(gpu, score):
    """A group whose biases are -inf ranks before one without an expert, whatever their numbers."""
    x = np.random.default_rng(1).standard_normal((24, 32))
    x[:, :8] = -np.inf
    bias = np.zeros(32)
    bias[8:16] = -np.inf
    bias[16:24] = -3.0e38
    for top_groups in (2, 3):
        for how in ("max", "top2"):
            _check(gpu, x, 8, "f32", bias, score=score, groups=4, top_groups=top_groups, group_score=how)
            _check(gpu, x, 8 * top_groups, "f32", bias, score=score, groups=4, top_groups=top_groups, group_score=how)


# --- scores far from 1 ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("low,high", [(-692.0, -680.0), (-699.9, -691.0), (-720.0, -695.0), (-745.0, -690.0)])
def test_sigmoids_that_64_bits_just_hold(gpu, dtype, low, high):
    """Weights of scores of 1e-300: a power's range is not left where scores still have a sum."""
    rng = np.random.default_rng(2)
    x = np.full((50, 64), -900.0)
    for t in range(50):
        x[t, rng.choice(64, 12, replace=False)] = rng.uniform(low, high, 12)
    _check(gpu, x, 8, dtype, score="sigmoid")


def test_softmax_weights_far_below_the_largest(gpu):
    """The largest logit is not chosen; the chosen ones are e^-690 and less of it."""
    rng = np.random.default_rng(3)
    x = np.full((30, 64), -800.0)
    bias = np.zeros(64)
    bias[0] = -2.0
    bias[8:16] = 1.0 + np.arange(8) / 8
    x[:, 0] = 0.0
    for low, high in ((-680.0, -600.0), (-699.0, -691.0), (-703.0, -685.0)):
        x[:, 8:16] = rng.uniform(low, high, (30, 8))
        _check(gpu, x, 8, "f32", bias)


def test_large_logits_and_biases_row_by_row(gpu):
    """Scores that saturate, that vanish, and biases far larger than them: each row whose border is not open."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((40, 128)) * 30
    for dtype in ("f32", "bf16"):
        for score in ("softmax", "sigmoid"):
            for bias in (None, rng.standard_normal(128) * 100, rng.integers(-3, 4, 128) * 0.5):
                for groups, top in ((1, 1), (16, 4), (4, 1)):
                    for how in ("max", "top2"):
                        _border(gpu, x, 8, dtype, bias, score=score, groups=groups, top_groups=top, group_score=how)


def _border(gpu, x, k, dtype, bias, **kw):
    """Rows by what decides: the last group that is open against the first that is not, and each choice against the
    next.  Those apart by more than 1e-13, or equal, have to come out; of others what comes out is as good to 1e-12."""
    values = host_values(x.astype(np.float32), dtype).astype(np.float64)
    b = None if bias is None else np.asarray(bias, np.float32).astype(np.float64)
    w, got = _run(gpu, x.astype(np.float32), k, dtype, bias, **kw)
    want, ids, _ = L.route(values, k, bias=b, **kw)
    size, closed = x.shape[1] // kw["groups"], 0
    for t in range(len(x)):
        v = values[t]
        s = np.exp(v - v.max()) / np.exp(v - v.max()).sum() if kw["score"] == "softmax" else 1.0 / (1.0 + np.exp(-v))
        key = s if b is None else s + b
        element = v if b is None else key
        use = element if kw["group_score"] == "max" and b is None else key
        n = 2 if kw["group_score"] == "top2" else 1
        rank = np.sort(use.reshape(-1, size), -1)[:, ::-1][:, :n].sum(-1)
        order = np.argsort(-rank, kind="stable")
        gap = rank[order[kw["top_groups"] - 1]] - rank[order[kw["top_groups"]]] if kw["top_groups"] < kw["groups"] else 1.0
        open_ = np.isin(np.arange(x.shape[1]) // size, order[:kw["top_groups"]])
        # equal ranks: of scores and biases that are the same numbers, or of scores that are 1 (e^-40 is below 2^-54)
        both = order[kw["top_groups"] - 1:kw["top_groups"] + 1]
        ones = np.sort(v.reshape(-1, size)[both], -1)[:, ::-1][:, :n].min() > 40.0
        sure = (gap == 0.0 and (b is not None or ones)) or gap > 1e-13
        if b is not None:
            d = -np.diff(np.sort(-np.where(open_, element, -np.inf))[:k + 1])
            d = np.abs(d[np.isfinite(d)])
            sure = sure and bool(((d == 0) | (d > 1e-13)).all())
        if sure:
            closed += 1
            assert np.array_equal(got[t], ids[t]), (t, kw)
            assert (np.abs(w[t] - want[t]) <= np.abs(want[t]) * 32 * L.F32 + 2.0 ** -148).all(), (t, kw)
            continue
        taken = sorted({int(g) for g in got[t] // size})
        assert len(taken) <= kw["top_groups"] and len(set(got[t].tolist())) == k
        assert all(rank[g] >= rank[order[kw["top_groups"] - 1]] - 1e-12 for g in taken)
        assert (np.diff(element[got[t]]) <= 1e-12).all()
        share = s[got[t]] / max(s[got[t]].sum(), 1e-300)
        assert (np.abs(w[t] - share) <= 32 * L.F32 * share + 2.0 ** -40).all()
    assert closed >= 6, (closed, kw)  # of 40: sums of two that saturate leave the most open


# --- the softmax's sum ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("experts,groups,group_score", [(1024, 1, "max"), (1017, 9, "max"), (1017, 9, "top2"), (1023, 3, "max"),
                                                        (512, 1, "max"), (256, 1, "max")])
def test_a_sum_whose_small_terms_are_lost(gpu, dtype, experts, groups, group_score):
    """Terms of less than half a step of a float32 sum, as many as a lane holds: their scores' order hangs on them."""
    size = experts // groups
    x = np.full((9, experts), -200.0)
    lane = 116 if groups == 9 else 88 if groups == 3 else experts // 16
    x[:, 1:min(lane, size)] = -16.75  # e^-16.75 = 5.3e-8, which 1 in float32 does not feel
    x[:, 0] = 0.0
    other = size if groups > 1 else experts - 1
    lost = (min(lane, size) - 1) * np.exp(-16.75)  # the first expert's score is 1 less this
    for part in (0.3, 0.6, 0.9, 1.1, 1.5):
        bias = np.full(experts, -5.0)
        bias[0], bias[other] = -1.0, -part * lost
        _check(gpu, x, 1, dtype, bias, groups=groups, top_groups=1, group_score=group_score)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("experts,k,groups", [(64, 6, 1), (256, 8, 8), (1024, 16, 1), (700, 5, 4), (60, 20, 1)])
@pytest.mark.parametrize("renormalise", [False, True])
def test_weights_are_rounded_once(gpu, dtype, experts, k, groups, renormalise):
    """A weight is its score in 64 bits, rounded to float32: by which way a token goes its bits do not differ by more."""
    rng = np.random.default_rng(experts)
    for spread in (0.2, 1.5, 6.0):
        x = rng.standard_normal((60, experts)) * spread
        for bias in (None, rng.standard_normal(experts) * 0.05):
            kw = dict(renormalise=renormalise, groups=groups, top_groups=max(1, groups // 2))
            values = host_values(x.astype(np.float32), dtype).astype(np.float64)
            want, ids, margin = L.route(values, k, bias=None if bias is None else bias.astype(np.float32).astype(np.float64), **kw)
            assert margin > 1e-13
            w, got = _run(gpu, x.astype(np.float32), k, dtype, bias, **kw)
            assert np.array_equal(got, ids)
            # half a step of float32, and 2^-30 for an exponential of 2^-32, a sum of those and a quotient of 2^-40
            assert (np.abs(w - want) <= np.abs(want) * (L.F32 + 2.0 ** -30) + 2.0 ** -149).all()


# --- rows, and what is beside them ----------------------------------------------------------------------------------
def test_a_row_is_what_it_is_alone(gpu):
    """A token whose last choice is open beside others changes no bit of theirs."""
    from tallax_amd import experts
    rng = np.random.default_rng(9)
    x = rng.standard_normal((16000, 256)).astype(np.float32)
    bias = np.zeros(256, np.float32)
    biased = rng.choice(255, 8, replace=False)
    bias[biased] = 0.3
    # every fourth token: expert 255's score is the others' and 0.3, as near as float32 comes: (e^v - 1) / (e^v + 255) = .3
    near = np.zeros(256, np.float32)
    b = float(np.float32(0.3))
    near[255] = np.log((1 + 255 * b) / (1 - b))
    x[::4] = near
    d, bias_d = torch.from_numpy(x).to(gpu), torch.from_numpy(bias).to(gpu)
    w, ids = experts.route(d, 8, bias=bias_d)
    rest = torch.arange(16000, device=gpu) % 4 != 0
    alone = experts.route(d[rest].contiguous(), 8, bias=bias_d)
    assert torch.equal(ids[rest], alone[1]) and torch.equal(w[rest], alone[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,k", [(1017, 9, 2, 16), (1017, 9, 5, 7), (1023, 3, 1, 8), (1023, 3, 2, 16),
                                                         (1020, 5, 2, 8), (1015, 7, 3, 16)])
def test_groups_of_many_experts_to_a_lane(gpu, dtype, score, experts, groups, top_groups, k):
    rng = np.random.default_rng(experts + top_groups)
    x = rng.standard_normal((37, experts)) * 1.5
    for bias in (None, rng.standard_normal(experts) * 0.05):
        for how in ("max", "top2"):
            _rows(gpu, x, k, dtype, bias, score=score, groups=groups, top_groups=top_groups, group_score=how, least=0.9)


def test_rows_that_lie_far_apart(gpu):
    """Rows more than 2^31 elements from each other, and one row of a stride that is never taken."""
    from tallax_amd import experts
    rng = np.random.default_rng(11)
    stride = 2 ** 31 + 40
    x = torch.from_numpy(rng.standard_normal((2, 64)).astype(np.float32)).to(gpu).bfloat16()
    far = torch.empty(stride + 64, dtype=torch.bfloat16, device=gpu)
    rows = far.as_strided((2, 64), (stride, 1))
    rows.copy_(x)
    want = experts.route(x, 6)
    assert all(torch.equal(a, b) for a, b in zip(experts.route(rows, 6), want, strict=True))
    one = x[:1].as_strided((1, 64), (2 ** 35, 1))
    assert all(torch.equal(a, b[:1]) for a, b in zip(experts.route(one, 6), want, strict=True))
