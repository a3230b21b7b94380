"""GPU: speculative.verify where logits are far from 0 (finite masks, forced tokens, infinities) and where a
workgroup takes several steps of a row, against its definition in 64 bits on the host."""
import numpy as np
import pytest
import torch

from oracle import tallax_oracle as O
from tests import serving_ref as R

pytestmark = pytest.mark.gpu

# no powers of two among them: a maximum times 1 / temperature is then rounded
TEMPERATURES = np.array([0.2, 0.3, 0.45, 0.6, 0.7, 0.8, 0.9, 1.0, 1.1, 1.3, 1.5, 2.7], np.float32)
STEP = {"bf16": 8192, "f32": 4096}  # elements of a step of the rows' sums


def _near(rng, logits, temp, dtype):
    """Draft probabilities near the target's, and drafts drawn from them."""
    l = (logits[:, :-1].astype(np.float64) + 0.6 * rng.standard_normal(logits[:, :-1].shape))
    with np.errstate(over="ignore"):
        e = np.exp((l - l.max(-1, keepdims=True)) / temp[:, None, None])
    q = O.round_to_dtype((e / e.sum(-1, keepdims=True)).astype(np.float32), dtype).astype(np.float32)
    return q, (q / rng.exponential(size=q.shape)).argmax(-1).astype(np.int32)


def _check(gpu, dtype, draft, logits, u, noise, q, temp, counts=None, steps=None):
    """Device tokens against the host's; no comparison of the seeds is within 1e-6 of equality (32-bit weights are
    off by some 1e-7).  steps: of a workgroup of the sums and of the race."""
    from tallax_amd import _lib, speculative
    want = R.verify(draft, logits.astype(np.float64), u, noise, None if q is None else q.astype(np.float64), temp, counts)
    assert want[2] > 1e-6, "a seed with a comparison too close to call"
    l = torch.from_numpy(logits).to(gpu).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    d, u, noise, temp = (torch.from_numpy(x).to(gpu) for x in (draft, u, noise, temp))
    q = None if q is None else torch.from_numpy(q).to(gpu)
    c = None if counts is None else torch.from_numpy(counts).to(gpu)
    if steps is None:
        tokens, accepted = speculative.verify(d, l, u, noise, draft_probs=q, temperature=temp, counts=c)
    else:
        batch, rows, vocab = l.shape
        tokens, accepted = torch.empty_like(l[..., 0], dtype=torch.int32), torch.empty_like(l[:, 0, 0], dtype=torch.int32)
        need = _lib.LIB.tallax_verify_workspace_size(batch, rows - 1, vocab, _lib.dtype_code(l))
        ws = _lib.workspace(l.device, need)
        _lib.check(_lib.LIB.tallax_testing_verify_steps(
            _lib.ptr(d), _lib.ptr(l), _lib.dtype_code(l), batch, rows - 1, vocab, _lib.ptr(c), _lib.ptr(temp),
            _lib.ptr(q), _lib.F32, _lib.ptr(u), _lib.ptr(noise), _lib.ptr(tokens), _lib.ptr(accepted), _lib.ptr(ws),
            ws.numel(), _lib.stream_of(l), *steps), "verify_steps")
    assert np.array_equal(accepted.cpu().numpy(), want[1])
    assert np.array_equal(tokens.cpu().numpy(), want[0])
    return want


def _randoms(rng, batch, drafted, vocab):
    return (rng.random((batch, drafted)).astype(np.float32),
            rng.exponential(size=(batch, vocab)).astype(np.float32) + np.float32(1e-12))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [8192, 32000, 32003])
@pytest.mark.parametrize("mask", [-1e4, -1e8, -1e9, -2e9, -1e10, -1e30, -1.5e38, float("-inf")])
def test_masked_but_for_a_few(gpu, dtype, vocab, mask):
    """A grammar's mask: 40 tokens are left, so most threads' elements are all masked."""
    rng = np.random.default_rng(20)
    batch, drafted = len(TEMPERATURES), 2
    logits = np.full((batch, drafted + 1, vocab), mask)
    for b in range(batch):
        at = rng.permutation(vocab)[:40]
        logits[b][:, at] = 3 * rng.standard_normal((drafted + 1, 40))
    logits = O.round_to_dtype(logits.astype(np.float32), dtype).astype(np.float32)
    u, noise = _randoms(rng, batch, drafted, vocab)
    q, draft = _near(rng, logits, TEMPERATURES, "f32")
    want = _check(gpu, dtype, draft, logits, u, noise, q, TEMPERATURES)
    assert want[1].max() == 2 and want[1].min() == 0
    _check(gpu, dtype, draft, logits, u, noise, None, TEMPERATURES)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e30])
def test_padded_vocabulary(gpu, dtype, mask):
    """The last elements of every row are masked, for more than a thread's elements."""
    rng = np.random.default_rng(21)
    batch, drafted, vocab = len(TEMPERATURES), 2, 50304
    logits = 3 * rng.standard_normal((batch, drafted + 1, vocab))
    logits[..., 32000:] = mask
    logits = O.round_to_dtype(logits.astype(np.float32), dtype).astype(np.float32)
    u, noise = _randoms(rng, batch, drafted, vocab)
    q, draft = _near(rng, logits, TEMPERATURES, "f32")
    _check(gpu, dtype, draft, logits, u, noise, q, TEMPERATURES)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("forced", [1e6, 1e9, 1e10, 1e30, 2.9e38])
def test_forced_tokens(gpu, dtype, forced):
    """One logit, or two equal ones, far above all others; the rest of a row is all equally far away."""
    rng = np.random.default_rng(22)
    batch, drafted, vocab = len(TEMPERATURES), 1, 16384
    logits = 3 * rng.standard_normal((batch, drafted + 1, vocab))
    at = rng.permutation(vocab)[:2 * batch].reshape(2, batch)
    logits[np.arange(batch), :, at[0]] = forced
    logits[np.arange(batch)[::2], :, at[1][::2]] = forced
    logits[1] = forced  # a whole row: no token is ahead
    logits = O.round_to_dtype(logits.astype(np.float32), dtype).astype(np.float32)
    u, noise = _randoms(rng, batch, drafted, vocab)
    draft = at[0][:, None].astype(np.int32)
    draft[3, 0] = (at[0][3] + 1) % vocab
    want = _check(gpu, dtype, draft, logits, u, noise, None, TEMPERATURES)
    assert want[1][3] == 0 and want[1][5] == 1


# of the sums and of the race; the plan's own number at these sizes is 1
STEPS = [(2, 2), (3, 1), (5, 7), (1, 3), (65536, 65536)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("steps", STEPS, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("off", [0, 3])
def test_several_steps(gpu, dtype, steps, off):
    """Rows of five steps and some more; the maximum lies in the first, a middle and the last one."""
    rng = np.random.default_rng(23)
    batch, drafted, vocab = 12, 3, 5 * STEP[dtype] + 77 + off
    logits = 3 * rng.standard_normal((batch, drafted + 1, vocab))
    for b in range(batch):
        at = (b % 6) * STEP[dtype] + 5 if b % 6 < 5 else vocab - 3
        logits[b, :, at] += 9  # greedy rows take it, the others often
    logits = O.round_to_dtype(logits.astype(np.float32), dtype).astype(np.float32)
    temp = TEMPERATURES.copy()
    temp[6:] = 0.0
    temp[8:10] = 1.7
    u, noise = _randoms(rng, batch, drafted, vocab)
    q, draft = _near(rng, logits, np.where(temp > 0, temp, 1).astype(np.float32), "f32")
    draft[6:8] = logits[6:8, :drafted].argmax(-1)
    draft[0, 0] = -1
    counts = np.array([3, 2, 3, 1, 3, 0, 3, 2, 3, 3, 9, -1], np.int32)
    want = _check(gpu, dtype, draft, logits, u, noise, q, temp, counts, steps)
    assert want[1][6] == 3
    _check(gpu, dtype, draft, logits, u, noise, None, temp, None, steps)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("steps", STEPS, ids=lambda s: "%dx%d" % s)
def test_strange_logits_in_several_steps(gpu, dtype, steps):
    """Infinities, NaN, finite masks and the type's ends in the first, a middle and the last step of a workgroup."""
    rng = np.random.default_rng(24)
    step = STEP[dtype]
    batch, drafted, vocab = 24, 1, 5 * step
    top = float(torch.finfo(torch.bfloat16 if dtype == "bf16" else torch.float32).max)
    logits = 3 * rng.standard_normal((batch, drafted + 1, vocab))
    for i, at in enumerate((0, 2 * step + 9, 5 * step - 1)):
        logits[i, :, at] = np.inf
        logits[3 + i, :, at] = top
        logits[6 + i, :, at] = 1e9
        logits[9 + i, :, at] = np.nan
        logits[12 + i] = -1e9 if i < 2 else -1e10
        logits[12 + i, :, at // step * step:(at // step + 1) * step] = 3 * rng.standard_normal((drafted + 1, step))
        logits[15 + i, :, at // step * step:(at // step + 1) * step] = -np.inf
        logits[18 + i, :, (0, at if at else step)] = np.inf  # two share the whole weight
    logits[21] = -top
    logits[22] = -np.inf
    logits[22, :, [step + 1, 4 * step + 1]] = -top
    logits[23] = np.nan
    logits = O.round_to_dtype(logits.astype(np.float32), dtype).astype(np.float32)
    for temps in (TEMPERATURES, TEMPERATURES[::-1], np.zeros_like(TEMPERATURES)):
        temp = np.concatenate([temps, temps[::-1]]).copy()
        u, noise = _randoms(rng, batch, drafted, vocab)
        clean = np.where(np.isnan(logits), -np.inf, logits)
        draft = clean[:, :1].argmax(-1).astype(np.int32)
        draft[::5, 0] = 7
        want = _check(gpu, dtype, draft, logits, u, noise, None, temp, None, steps)
        assert want[0][23, 0] == -1 and want[1][1] == 1


def test_refuses_steps(gpu):
    from tallax_amd import _lib
    for steps in ((-1, 0), (0, -1), (65537, 1)):
        st = _lib.LIB.tallax_testing_verify_steps(4, 4, 0, 2, 3, 100, None, 4, None, 0, 4, 4, 4, 4, 256, 1 << 20, None,
                                                  *steps)
        assert st == _lib.INVALID_ARGUMENT
