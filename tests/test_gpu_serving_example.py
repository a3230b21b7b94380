"""GPU: the serving operators together, as examples/speculative_decoding.py runs them."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "speculative_decoding.py")
    spec = importlib.util.spec_from_file_location("speculative_decoding", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _text(tokens, n):
    return [[t for t in row if t >= 0][:n] for row in tokens.flatten(1).tolist()]


def test_greedy_drafts_change_no_token(gpu, example):
    """In float32, what is decoded greedily with drafts is what is decoded token by token."""
    model = example.Model(vocab=1500, hidden=256, heads=6, kv_heads=3, dim=40, dtype=torch.float32)
    prompt = torch.randint(0, 1500, (7, 33), device=gpu, dtype=torch.int32)
    plain, _, _ = example.generate(model, prompt, 40, 0)
    drafted, accepted, _ = example.generate(model, prompt, 40, 3)
    assert 0.5 < float(accepted.float().mean()) < 3
    assert _text(plain, 40) == _text(drafted, 40)


def test_cache_stays_within_its_budget(gpu, example):
    model = example.Model(vocab=1000, hidden=128, heads=4, kv_heads=2, dim=64)
    prompt = torch.randint(0, 1000, (5, 200), device=gpu, dtype=torch.int32)
    tokens, accepted, lens = example.generate(model, prompt, 24, 4, budget=64, every=8, temperature=0.8)
    assert lens.tolist() == [64] * 5
    assert bool(((tokens >= 0).sum(-1) == accepted + 1).all()) and int(tokens.max()) < 1000
