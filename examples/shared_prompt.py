"""Several samples of each of several prompts, decoded behind prompts that are kept once.

A one-layer model with rotary positions and a mixture of experts, with random
weights.  Each prompt's keys and values are written to the cache once
(kvcache.append_rotated); its samples decode together, each with a block table
for its own tokens alone: a step rotates and appends them (append_rotated),
attends to prompt and own tokens (kvcache.decode_shared), sends each token to
its experts (experts.route) and draws the next (sampling.sample).

    python examples/shared_prompt.py [--prompts 4] [--samples 16] [--length 8000] [--steps 100]
"""
from __future__ import annotations

import argparse
import os
import sys
import time
from types import SimpleNamespace

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from tallax_amd import experts, kvcache, sampling  # noqa: E402


class Model:
    """One layer: attention, then the experts that a token is sent to."""

    def __init__(self, vocab=8000, hidden=512, heads=8, kv_heads=2, dim=64, n_experts=32, chosen=4, groups=4,
                 dtype=torch.bfloat16, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)

        def weight(*shape, scale):
            return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

        self.heads, self.kv_heads, self.dim, self.vocab, self.dtype = heads, kv_heads, dim, vocab, dtype
        self.chosen, self.groups = chosen, groups
        self.embedding = weight(vocab, hidden, scale=1.0)
        self.wqkv = weight(hidden, (heads + 2 * kv_heads) * dim, scale=hidden ** -0.5)
        self.wo = weight(heads * dim, hidden, scale=0.6 * (heads * dim) ** -0.5)
        self.router = weight(hidden, n_experts, scale=hidden ** -0.5)
        self.balance = torch.randn(n_experts, generator=gen, device="cuda") * 0.05
        self.up = weight(n_experts, hidden, 2 * dim, scale=hidden ** -0.5)
        self.down = weight(n_experts, 2 * dim, hidden, scale=(2 * dim) ** -0.5)
        self.head = weight(hidden, vocab, scale=4.0 * hidden ** -0.5)
        self.frequencies = 10000.0 ** (-torch.arange(dim // 2, device="cuda") / (dim // 2))

    def queries_keys_values(self, tokens):
        qkv = (self.embedding[tokens.long()] @ self.wqkv).reshape(*tokens.shape, -1, self.dim)
        return qkv.split([self.heads, self.kv_heads, self.kv_heads], 2)

    def logits(self, tokens, attended):
        x = self.embedding[tokens.long()] + attended.flatten(2) @ self.wo
        x = x[:, -1]
        w, ids = experts.route(x @ self.router, self.chosen, score="sigmoid", bias=self.balance, groups=self.groups,
                               top_groups=self.groups // 2, group_score="top2")
        for j in range(self.chosen):
            e = ids[:, j].long()
            inner = torch.relu((x[:, None] @ self.up[e])[:, 0])
            x = x + w[:, j, None].to(self.dtype) * (inner[:, None] @ self.down[e])[:, 0]
        return x @ self.head


@torch.inference_mode()
def generate(model, prompts, samples, steps, shared=True, page=16, temperature=0.0, seed=0):
    """tokens [prompts * samples, steps].  shared: prompts are kept once, else again for each sample."""
    count, n = prompts.shape
    batch = count * samples
    front, own = -(-n // page), -(-(steps + (0 if shared else n)) // page)
    pages = batch * own + (count * front if shared else 0)
    k_pages, v_pages = (torch.empty((pages, model.kv_heads, page, model.dim), dtype=model.dtype, device="cuda")
                        for _ in range(2))
    perm = torch.randperm(pages, device="cuda").to(torch.int32)
    table, prefix = perm[:batch * own].reshape(batch, own), perm[batch * own:].reshape(count, -1)
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")

    # the prompts' keys and values, but for the last token, which is the first that each sample is fed
    fed = prompts[:, :-1] if shared else prompts[:, :-1].repeat_interleave(samples, 0)
    q, k, v = model.queries_keys_values(fed)
    written, _ = kvcache.append_rotated(k_pages, v_pages, prefix if shared else table, lens[:fed.shape[0]], q, k, v,
                                        model.frequencies)
    begins = written if shared else None
    lens = lens if shared else written

    last = prompts[:, -1:].repeat_interleave(samples, 0)
    how = SimpleNamespace(top_k=40, top_p=0.95, temperature=temperature)
    tokens = []
    for step in range(steps):
        q, k, v = model.queries_keys_values(last)
        at = (lens + (n - 1 if shared else 0))[:, None]
        lens, q = kvcache.append_rotated(k_pages, v_pages, table, lens, q, k, v, model.frequencies, token_positions=at)
        if shared:
            attended, _ = kvcache.decode_shared(q, k_pages, v_pages, prefix, begins, table, lens)
        else:
            attended, _ = kvcache.decode(q, k_pages, v_pages, table, lens)
        last = sampling.sample((seed, step), model.logits(last, attended), how)[:, None]
        tokens.append(last)
    return torch.cat(tokens, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompts", type=int, default=4)
    ap.add_argument("--samples", type=int, default=16)
    ap.add_argument("--length", type=int, default=8000)
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--temperature", type=float, default=0.7)
    a = ap.parse_args()
    model = Model()
    prompts = torch.randint(0, model.vocab, (a.prompts, a.length), device="cuda", dtype=torch.int32)
    for shared in (False, True):
        generate(model, prompts, a.samples, 4, shared, temperature=a.temperature)
        torch.cuda.synchronize()
        start = time.perf_counter()
        tokens = generate(model, prompts, a.samples, a.steps, shared, temperature=a.temperature)
        torch.cuda.synchronize()
        seconds = time.perf_counter() - start
        print(f"{'prompts kept once' if shared else 'a prompt a sample'}: {tokens.numel()} tokens in "
              f"{seconds * 1e3:.0f} ms, {tokens.numel() / seconds:.0f} tokens/s")


if __name__ == "__main__":
    main()
