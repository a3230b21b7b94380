"""GPU: speculative.verify against its definition in 64 bits on the host, and the distribution it has to keep."""
import numpy as np
import pytest
import torch

from oracle import tallax_oracle as O
from tests import serving_ref as R

pytestmark = pytest.mark.gpu


def _round(x, dtype):
    return O.round_to_dtype(x.astype(np.float32), dtype).astype(np.float32)


def _dev(x, dtype, gpu):
    return torch.from_numpy(np.ascontiguousarray(x)).to(gpu).to(torch.bfloat16 if dtype == "bf16" else torch.float32)


def _inputs(seed, batch, drafted, vocab, dtype, qdtype, near=0.6):
    rng = np.random.default_rng(seed)
    logits = _round(rng.standard_normal((batch, drafted + 1, vocab)) * 3, dtype)
    temp = rng.uniform(0.5, 1.3, batch).astype(np.float32)
    l = (logits[:, :drafted] + near * rng.standard_normal((batch, drafted, vocab))) / temp[:, None, None]
    e = np.exp(l - l.max(-1, keepdims=True)) if drafted else l
    q = _round(e / e.sum(-1, keepdims=True), qdtype) if drafted else l.astype(np.float32)
    draft = (q / rng.exponential(size=q.shape)).argmax(-1).astype(np.int32) if drafted else np.zeros((batch, 0), np.int32)
    u = rng.random((batch, drafted)).astype(np.float32)
    noise = rng.exponential(size=(batch, vocab)).astype(np.float32) + np.float32(1e-12)
    return draft, logits, u, noise, q, temp


def _run(gpu, dtype, qdtype, draft, logits, u, noise, q, temp, counts=None):
    """Device tokens against the host's.  Comparisons closer than 1e-9 (the device's sums carry about 1e-7 of
    32-bit weights, each random, into 64 bits) would leave the answer open: the seeds have none within 1e-6."""
    from tallax_amd import speculative
    want = R.verify(draft, logits.astype(np.float64), u, noise, None if q is None else q.astype(np.float64), temp, counts)
    assert want[2] > 1e-6, "a seed with a comparison too close to call"
    got = speculative.verify(torch.from_numpy(draft).to(gpu), _dev(logits, dtype, gpu), torch.from_numpy(u).to(gpu),
                             torch.from_numpy(noise).to(gpu), draft_probs=None if q is None else _dev(q, qdtype, gpu),
                             temperature=torch.from_numpy(temp).to(gpu),
                             counts=None if counts is None else torch.from_numpy(counts).to(gpu))
    assert got[0].dtype == torch.int32 and got[1].dtype == torch.int32
    assert np.array_equal(got[1].cpu().numpy(), want[1])
    assert np.array_equal(got[0].cpu().numpy(), want[0])
    return want


@pytest.mark.parametrize("dtype,qdtype", [("bf16", "f32"), ("f32", "bf16"), ("f32", None), ("bf16", None)])
@pytest.mark.parametrize("batch,drafted,vocab", [
    (1, 0, 1), (2, 1, 1), (3, 1, 7), (2, 2, 100), (5, 3, 1000), (4, 4, 4095), (3, 5, 4096), (3, 2, 4097),
    (2, 8, 8193), (9, 1, 32000), (2, 63, 513), (2, 3, 50257), (1, 2, 201088)])
def test_verify(gpu, dtype, qdtype, batch, drafted, vocab):
    draft, logits, u, noise, q, temp = _inputs(batch + drafted + vocab, batch, drafted, vocab, dtype, qdtype or "f32")
    if vocab > 1 and qdtype is None and drafted:
        draft[0] = logits[0, :drafted].argmax(-1)  # a draft that may be accepted
    _run(gpu, dtype, qdtype, draft, logits, u, noise, q if qdtype else None, temp)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_counts_greedy_and_bad_drafts(gpu, dtype):
    draft, logits, u, noise, q, temp = _inputs(5, 12, 4, 3001, dtype, "f32")
    temp[::3] = 0.0
    temp[4] = -1.0
    draft[0], draft[3, :2] = logits[0, :4].argmax(-1), logits[3, :2].argmax(-1)
    draft[5, 0], draft[7, 0], draft[9, 1] = -1, 3001, 2 ** 31 - 1
    logits[6, :, 17] = logits[6, :, 1200] = logits[6].max() + 1  # greedy ties go to the lowest
    logits = _round(logits, dtype)
    draft[6, :2] = [17, 1200]
    counts = np.array([4, 0, 1, 2, 4, 3, 4, 4, 0, 3, 9, -2], np.int32)
    want = _run(gpu, dtype, "f32", draft, logits, u, noise, q, temp, counts)
    assert want[1][0] == 4 and want[1][6] == 1 and want[0][6, 1] == 17


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_masks_and_strange_logits(gpu, dtype):
    draft, logits, u, noise, q, temp = _inputs(6, 10, 2, 5000, dtype, "f32")
    logits[0, :, 10:] = -np.inf            # almost everything masked
    logits[1] = -np.inf                    # nothing left
    logits[2, 0] = -np.inf
    logits[3, :, ::2] = np.nan
    logits[4, :, [3, 4000]] = np.inf       # two share the whole weight
    logits[5] = np.finfo(np.float32).min if dtype == "f32" else -3.3895314e38
    logits[6, :, 77] = 1e30
    logits[7] = np.nan
    temp[8:] = 0.0
    logits[8] = -np.inf
    logits[9, :, 4321] = np.inf
    logits = _round(logits, dtype) if dtype == "bf16" else logits
    draft[0] = [3, 4]
    want = _run(gpu, dtype, "f32", draft, logits, u, noise, q, temp)
    assert want[0][1, 0] == -1 and want[0][7, 0] == -1 and want[0][8, 0] == -1 and want[0][9, 0] == 4321


def test_residual_that_is_nowhere_positive(gpu):
    """Draft probabilities of twice the target's: half of the drafts are refused, and p - q has no positive place."""
    rng = np.random.default_rng(7)
    logits = rng.standard_normal((40, 2, 6000)).astype(np.float32)
    e = np.exp(logits[:, :1].astype(np.float64))
    q = (2 * e / e.sum(-1, keepdims=True)).astype(np.float32)
    draft = rng.integers(0, 6000, (40, 1)).astype(np.int32)
    u = rng.random((40, 1)).astype(np.float32)
    noise = rng.exponential(size=(40, 6000)).astype(np.float32) + np.float32(1e-12)
    want = _run(gpu, "f32", "f32", draft, logits, u, noise, q, np.ones(40, np.float32))
    assert 5 < want[1].sum() < 35


def test_temperatures(gpu):
    draft, logits, u, noise, q, temp = _inputs(8, 8, 2, 2000, "f32", "f32")
    temp[:] = [1e-5, 2e-5, 1e-3, 0.01, 10.0, 1e4, 1e30, 9e-6]
    _run(gpu, "f32", "f32", draft, logits, u, noise, q, temp)


def test_the_first_token_is_distributed_as_the_target(gpu):
    """Whatever the draft's distribution, token 0 has the target's: 20000 rows, 5 standard deviations."""
    from tallax_amd import speculative
    batch, vocab = 20000, 8
    gen = torch.Generator(device=gpu)
    gen.manual_seed(3)
    row = torch.randn((1, 2, vocab), generator=gen, device=gpu) * 1.5
    q = torch.softmax(torch.randn((1, 1, vocab), generator=gen, device=gpu) * 1.5, -1).expand(batch, 1, vocab).contiguous()
    draft = torch.multinomial(q[:, 0], 1, generator=gen).to(torch.int32)
    u = torch.rand((batch, 1), generator=gen, device=gpu)
    noise = torch.empty((batch, vocab), device=gpu).exponential_(1.0, generator=gen).clamp_(min=1e-12)
    tokens, accepted = speculative.verify(draft, row.expand(batch, 2, vocab).contiguous(), u, noise, draft_probs=q)
    p = torch.softmax(row[0].double(), -1)
    for at, rows in ((0, tokens), (1, tokens[accepted == 1])):
        n = rows.shape[0]
        freq = torch.bincount(rows[:, at].long(), minlength=vocab).double() / n
        assert ((freq - p[at]).abs() < 5 * (p[at] * (1 - p[at]) / n).sqrt()).all()
    keep = float(torch.minimum(p[0], q[0, 0].double()).sum())
    assert abs(float(accepted.double().mean()) - keep) < 5 * (keep * (1 - keep) / batch) ** 0.5


def test_strides_streams_and_graph(gpu):
    from tallax_amd import speculative
    gen = torch.Generator(device=gpu)
    gen.manual_seed(4)
    big = torch.randn((6, 5, 9001), generator=gen, device=gpu).to(torch.bfloat16)
    logits = big[:, 1:5, 1:]  # rows that begin off 16 bytes, and a part of a larger tensor
    args = [torch.randint(0, 9000, (6, 3), generator=gen, device=gpu, dtype=torch.int32), logits,
            torch.rand((6, 3), generator=gen, device=gpu),
            torch.empty((6, 9000), device=gpu).exponential_(1.0, generator=gen).clamp_(min=1e-12)]
    want = speculative.verify(*args, temperature=0.8)
    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream())
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)
    with torch.cuda.stream(side):
        there = speculative.verify(*args, temperature=0.8, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, there))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = speculative.verify(*args, temperature=0.8, workspace=ws)
    for rep in range(3):
        big.copy_(torch.randn(big.shape, generator=gen, device=gpu) * (rep + 1))
        args[0].copy_(logits[:, :3].float().argmax(-1) if rep == 1 else args[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured]
        want = speculative.verify(*args, temperature=0.8)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), rep


def test_refusals(gpu):
    from tallax_amd import speculative
    draft = torch.zeros((2, 3), dtype=torch.int32, device=gpu)
    logits = torch.zeros((2, 4, 100), device=gpu)
    u, noise = torch.zeros((2, 3), device=gpu), torch.ones((2, 100), device=gpu)
    speculative.verify(draft, logits, u, noise)
    for bad in (dict(draft_tokens=draft.long()), dict(draft_tokens=draft[:, :2]), dict(target_logits=logits[0]),
                dict(target_logits=logits[:, :0]), dict(uniforms=u[:1]), dict(noise=noise[:, :50]),
                dict(noise=noise.double()), dict(draft_probs=logits), dict(counts=draft[0]),
                dict(temperature=torch.ones(3)), dict(target_logits=logits.cpu())):
        args = dict(draft_tokens=draft, target_logits=logits, uniforms=u, noise=noise)
        with pytest.raises(ValueError):
            speculative.verify(**{**args, **bad})
    with pytest.raises(NotImplementedError):
        speculative.verify(draft, logits.half(), u, noise)
    with pytest.raises(NotImplementedError):
        speculative.verify(torch.zeros((1, 64), dtype=torch.int32, device=gpu), torch.zeros((1, 65, 8), device=gpu),
                           torch.zeros((1, 64), device=gpu), torch.ones((1, 8), device=gpu))
    empty = speculative.verify(draft[:0], logits[:0], u[:0], noise[:0])
    assert empty[0].shape == (0, 4) and empty[1].shape == (0,)


def test_small_probabilities_race_closely(gpu):
    """Two tokens of probability 2^-66 to 2^-148 whose noise makes them the largest, a few 1e-6 apart: a 32-bit
    exponent is rounded by as much there, and below 2^-126 a 32-bit probability by more."""
    rng = np.random.default_rng(9)
    batch, vocab = 3000, 32
    rows = np.arange(batch)
    logits = np.full((batch, 1, vocab), -np.inf, np.float32)
    at = np.stack([rng.permutation(vocab)[:3] for _ in range(batch)]).T
    a = rng.uniform(-102, -46, batch)
    logits[rows, 0, at[0]], logits[rows, 0, at[1]], logits[rows, 0, at[2]] = 0, a, a + rng.uniform(-0.7, 0.7, batch)
    p = np.exp(logits[:, 0].astype(np.float64))
    p /= p.sum(-1, keepdims=True)
    noise = rng.exponential(size=(batch, vocab)).astype(np.float32) + np.float32(1e-12)
    noise[rows, at[0]] = 2.0 ** 60
    noise[rows, at[1]] = p[rows, at[1]] * 2.0 ** 30
    apart = 1 + rng.uniform(1.2e-6, 6e-6, batch) * rng.choice([-1, 1], batch)
    s = p[rows, at[1]] / noise[rows, at[1]].astype(np.float64) * apart
    noise[rows, at[2]] = p[rows, at[2]] / s
    none = np.zeros((batch, 0), np.int32)
    want = _run(gpu, "f32", None, none, logits, none.astype(np.float32), noise, None, np.ones(batch, np.float32))
    assert 1000 < (want[0][:, 0] == at[1]).sum() < 2000 and ((want[0][:, 0] == at[1]) | (want[0][:, 0] == at[2])).all()


@pytest.mark.parametrize("dtype,qdtype", [("bf16", "f32"), ("f32", None)])
def test_many_sequences_of_long_rows(gpu, dtype, qdtype):
    """More workgroups in the race than find the accepted drafts themselves; some sequences greedy, some masked."""
    batch, vocab = 70, 33001
    draft, logits, u, noise, q, temp = _inputs(10, batch, 1, vocab, dtype, qdtype or "f32")
    temp[::7] = 0.0
    logits[3] = -np.inf
    logits[4, :, 1:] = -np.inf
    counts = np.where(np.arange(batch) % 5 == 0, 0, 1).astype(np.int32)
    _run(gpu, dtype, qdtype, draft, logits, u, noise, q if qdtype else None, temp, counts)
