"""GPU: append_rotated, decode_shared and route together, as examples/shared_prompt.py runs them; in captured graphs,
on other streams and two at a time."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from tests import serving_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "shared_prompt.py")
    spec = importlib.util.spec_from_file_location("shared_prompt", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("samples,length", [(3, 67), (40, 67), (3, 1111), (20, 1111)])
def test_a_prompt_kept_once_changes_no_token(gpu, example, samples, length):
    """In float32 and greedily, samples behind shared prompts decode what they decode with prompts of their own."""
    model = example.Model(vocab=1500, hidden=256, heads=6, kv_heads=3, dim=40, n_experts=24, dtype=torch.float32)
    gen = torch.Generator(device=gpu)
    gen.manual_seed(10)
    prompts = torch.randint(0, 1500, (2, length), generator=gen, device=gpu, dtype=torch.int32)
    own = example.generate(model, prompts, samples, 24, shared=False)
    once = example.generate(model, prompts, samples, 24)
    assert torch.equal(own, once)
    assert bool((once.reshape(2, samples, 24) == once.reshape(2, samples, 24)[:, :1]).all())


def test_samples_differ(gpu, example):
    model = example.Model(vocab=1000, hidden=128, heads=4, kv_heads=2, dim=64)
    prompts = torch.randint(0, 1000, (3, 100), device=gpu, dtype=torch.int32)
    tokens = example.generate(model, prompts, 5, 12, temperature=1.0)
    assert tokens.shape == (15, 12) and int(tokens.min()) >= 0 and int(tokens.max()) < 1000
    assert len({tuple(t) for t in tokens.tolist()}) > 10


class Step:
    """The three calls on buffers that stay where they are."""

    def __init__(self, gpu, batch, heads, kv_heads, dim, dtype, seed, prefix=300):
        rng = np.random.default_rng(seed)
        lens = [0 if i % 5 == 3 else 5 + i % 20 for i in range(batch)]
        k, v, table = R.make_cache(rng, batch + 1, kv_heads, dim, 16, -(-prefix // 16), lens + [prefix], dtype)
        self.k, self.v = k.to(gpu), v.to(gpu)
        pages = max(2, -(-(max(lens) + 1) // 16))
        self.prefix = table[batch:].contiguous().to(gpu)
        free = torch.arange(k.shape[0] - 2 * batch, k.shape[0], dtype=torch.int32)
        own = table[:batch, :pages].clone()
        own[own < 0] = free[:int((own < 0).sum())] if int((own < 0).sum()) <= free.numel() else -1
        self.table = own.to(gpu)
        i32 = dict(dtype=torch.int32, device=gpu)
        self.begins, self.lens = torch.tensor([prefix], **i32), torch.tensor(lens, **i32)
        gen = torch.Generator(device=gpu)
        gen.manual_seed(seed)
        self.qkv = torch.randn((batch, 1, heads + 2 * kv_heads, dim), generator=gen, device=gpu).to(dtype)
        self.split = [heads, kv_heads, kv_heads]
        self.f = torch.rand(dim // 2, generator=gen, device=gpu)
        self.logits = torch.randn((batch, 64), generator=gen, device=gpu)
        self.bias = torch.randn(64, generator=gen, device=gpu) * 0.05
        self.ws = torch.empty(1 << 25, dtype=torch.uint8, device=gpu)

    def fresh(self, seed):
        gen = torch.Generator(device=self.qkv.device)
        gen.manual_seed(seed)
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=gen, device=self.qkv.device))
        self.logits.copy_(torch.randn(self.logits.shape, generator=gen, device=self.qkv.device))

    def __call__(self, workspace=True):
        from tallax_amd import experts, kvcache
        q, k, v = self.qkv.split(self.split, 2)
        lens, q = kvcache.append_rotated(self.k, self.v, self.table, self.lens, q, k, v, self.f)
        out, lse = kvcache.decode_shared(q, self.k, self.v, self.prefix, self.begins, self.table, lens,
                                         workspace=self.ws if workspace else None)
        w, ids = experts.route(self.logits, 6, score="sigmoid", bias=self.bias, groups=8, top_groups=3, group_score="top2")
        return lens, q, out, lse, w, ids


SHAPES = [(3, 4, 2, 64, torch.bfloat16), (20, 8, 4, 128, torch.bfloat16), (70, 8, 4, 128, torch.bfloat16),
          (70, 4, 4, 80, torch.float32), (9, 4, 2, 256, torch.float32)]


@pytest.mark.parametrize("prefix", [300, 2500])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_captured_step(gpu, shape, prefix):
    """Captured without a run before; each replay, with new inputs and eager work between them, is the eager result."""
    step = Step(gpu, *shape, seed=1, prefix=prefix)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(5):
        step.fresh(100 + i)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        want = step(workspace=False)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True)), i


@pytest.mark.parametrize("prefix", [300, 2500])
def test_two_captured_steps_of_one_workspace(gpu, prefix):
    """Two graphs, replayed one after the other in turn, whose calls use the same workspace."""
    steps = [Step(gpu, *SHAPES[2], seed=2, prefix=prefix), Step(gpu, *SHAPES[1], seed=3, prefix=prefix)]
    steps[1].ws = steps[0].ws
    graphs, held = [], []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(s())
        graphs.append(g)
    want = [[x.clone() for x in s(workspace=False)] for s in steps]
    for i in (0, 1, 1, 0, 1):
        for x in held[i]:
            x.zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held[i], want[i], strict=True)), i


@pytest.mark.parametrize("prefix", [300, 2500])
def test_two_streams_at_once(gpu, prefix):
    steps = [Step(gpu, *SHAPES[2], seed=4, prefix=prefix), Step(gpu, *SHAPES[3], seed=5, prefix=prefix)]
    want = [[x.clone() for x in s()] for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu) for _ in steps]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(steps):
            with torch.cuda.stream(streams[i]):
                got[i].append(s())
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[i], strict=True))


def test_inputs_are_left_as_they_were(gpu):
    step = Step(gpu, *SHAPES[1], seed=6)
    kept = [x.clone() for x in (step.qkv, step.table, step.prefix, step.lens, step.begins, step.f, step.logits, step.bias)]
    step()
    now = (step.qkv, step.table, step.prefix, step.lens, step.begins, step.f, step.logits, step.bias)
    assert all(torch.equal(a, b) for a, b in zip(kept, now, strict=True))


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("batch,prefix", [(3, 300), (3, 2500), (20, 300), (20, 2500), (70, 2500)])
def test_pools_of_more_than_32_bits(gpu, batch, prefix, heads_first):
    """The last pages of pools of 6.5 GB, page after page or head after head, against a pool of their own."""
    step = Step(gpu, batch, 16, 8, 128, torch.bfloat16, seed=7, prefix=prefix)
    pages, kv_heads, page, dim = step.k.shape
    start = step.k.clone(), step.v.clone()
    want = [x.clone() for x in step()]
    kept = step.k, step.v
    many = 6_500_000_000 // (kv_heads * page * dim * 2)
    shape = (kv_heads, many, page, dim) if heads_first else (many, kv_heads, page, dim)
    far = [torch.empty(shape, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    step.k, step.v = [x.transpose(0, 1) if heads_first else x for x in far]
    for pool, first in zip((step.k, step.v), start, strict=True):
        pool[-pages:] = first
    for table in (step.table, step.prefix):
        table[table >= 0] += many - pages
    got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    assert torch.equal(step.k[-pages:], kept[0]) and torch.equal(step.v[-pages:], kept[1])


@pytest.mark.parametrize("prefix", [300, 2500])
@pytest.mark.parametrize("batch", [2, 40, 70])
def test_pools_without_a_page(gpu, batch, prefix):
    """Every token is dropped and nothing is seen."""
    step = Step(gpu, batch, 8, 4, 128, torch.bfloat16, seed=8, prefix=prefix)
    q = step()[1]
    step.k, step.v = step.k[:0], step.v[:0]
    lens, turned, out, lse, _, _ = step()
    assert torch.equal(q, turned) and torch.equal(lens, step.lens + 1)
    assert not bool(out.any()) and bool((lse == -float("inf")).all())
