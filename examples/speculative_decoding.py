"""Speculative decoding over a paged key-value cache that is kept to a budget.

A one-layer attention model with random weights decodes a batch of sequences.
Each step drafts a few tokens with a bigram table, writes their keys and values
behind the sequences (kvcache.append), attends from all of them at once
(kvcache.decode), keeps the drafts that the model agrees with and draws the next
token (speculative.verify); every few steps the cache is cut back to the slots
that attention has used most (kvcache.evict).  Nothing is copied to the host
until the tokens are read at the end.

    python examples/speculative_decoding.py [--batch 64] [--steps 200] [--drafted 4] [--budget 512]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from tallax_amd import kvcache, speculative  # noqa: E402


class Model:
    """Logits of a token from its embedding and the attention over what came before it."""

    def __init__(self, vocab=8000, hidden=512, heads=8, kv_heads=2, dim=64, dtype=torch.bfloat16, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)

        def weight(rows, cols, scale):
            return (torch.randn((rows, cols), generator=gen, device="cuda") * scale).to(dtype)

        self.heads, self.kv_heads, self.dim, self.vocab, self.dtype = heads, kv_heads, dim, vocab, dtype
        self.embedding = weight(vocab, hidden, 1.0)
        self.wq, self.wk, self.wv = (weight(hidden, h * dim, hidden ** -0.5) for h in (heads, kv_heads, kv_heads))
        self.wo = weight(heads * dim, hidden, 0.6 * (heads * dim) ** -0.5)
        self.head = weight(hidden, vocab, 4.0 * hidden ** -0.5)
        # what the embedding alone would be followed by: the draft
        self.bigram = torch.cat([(rows @ self.head).argmax(-1) for rows in self.embedding.split(1024)]).to(torch.int32)

    def keys_values(self, x):
        shape = (*x.shape[:2], self.kv_heads, self.dim)
        return (x @ self.wk).reshape(shape), (x @ self.wv).reshape(shape)

    def queries(self, x):
        return (x @ self.wq).reshape(*x.shape[:2], self.heads, self.dim)

    def logits(self, x, attended):
        return (x + attended.flatten(2) @ self.wo) @ self.head


@torch.inference_mode()
def generate(model, prompt, steps, drafted, budget=None, every=8, page=16, temperature=0.0, seed=0):
    """(tokens [batch, steps, drafted + 1] padded with -1, accepted [batch, steps], lens) after `steps` steps."""
    batch, n = prompt.shape
    most = n + steps * (drafted + 1) if budget is None else max(n, budget) + every * (drafted + 1)
    width = -(-most // page)
    shape = (batch * width, model.kv_heads, page, model.dim)
    k_pages, v_pages = (torch.empty(shape, dtype=model.dtype, device="cuda") for _ in range(2))
    table = torch.randperm(batch * width, device="cuda").reshape(batch, width).to(torch.int32)
    scores = torch.zeros((batch, model.kv_heads, width * page), device="cuda")
    positions = torch.full_like(scores, -1, dtype=torch.int32)
    lens, seen = (torch.zeros(batch, dtype=torch.int32, device="cuda") for _ in range(2))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    noise = torch.empty((batch, model.vocab), device="cuda")

    if n > 1:  # one layer: the prompt's own outputs are not needed, only its keys and values
        k, v = model.keys_values(model.embedding[prompt[:, :-1].long()])
        lens = kvcache.append(k_pages, v_pages, table, lens, k, v, scores=scores, positions=positions, seen=seen)
        seen = lens.clone()
    last = prompt[:, -1:].to(torch.int32)
    tokens, accepted = [], []
    for step in range(steps):
        draft = [last]
        for _ in range(drafted):
            draft.append(model.bigram[draft[-1].long()])
        fed = torch.cat(draft, 1)
        x = model.embedding[fed.long()]
        k, v = model.keys_values(x)
        filled = kvcache.append(k_pages, v_pages, table, lens, k, v, scores=scores, positions=positions, seen=seen)
        attended, _, _ = kvcache.decode(model.queries(x), k_pages, v_pages, table, filled, scores=scores,
                                        out_scores=scores)
        took, count = speculative.verify(fed[:, 1:], model.logits(x, attended),
                                         torch.rand((batch, drafted), generator=gen, device="cuda"),
                                         noise.exponential_(generator=gen).clamp_(min=1e-20), temperature=temperature)
        # the slots of refused drafts are written over by the next step
        lens, seen = lens + count + 1, seen + count + 1
        last = took.gather(1, count[:, None].long())
        tokens.append(took)
        accepted.append(count)
        if budget is not None and step % every == every - 1:
            lens, scores, positions = kvcache.evict(k_pages, v_pages, table, lens, scores, positions, seen,
                                                    budget=budget, recent=budget // 4, sinks=min(4, budget // 2))
    return torch.stack(tokens, 1), torch.stack(accepted, 1), lens


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--drafted", type=int, default=4)
    ap.add_argument("--budget", type=int, default=512)
    ap.add_argument("--prompt", type=int, default=1000)
    ap.add_argument("--temperature", type=float, default=0.7)
    a = ap.parse_args()
    model = Model()
    prompt = torch.randint(0, model.vocab, (a.batch, a.prompt), device="cuda", dtype=torch.int32)
    for drafted in sorted({0, a.drafted}):
        generate(model, prompt, 8, drafted, a.budget, temperature=a.temperature)
        torch.cuda.synchronize()
        start = time.perf_counter()
        tokens, accepted, lens = generate(model, prompt, a.steps, drafted, a.budget, temperature=a.temperature)
        torch.cuda.synchronize()
        seconds = time.perf_counter() - start
        made = int((tokens >= 0).sum())
        print(f"{drafted} drafted: {made} tokens in {seconds * 1e3:.0f} ms, {made / seconds:.0f} tokens/s, "
              f"{float(accepted.float().mean()) + 1:.2f} tokens a step, longest cache {int(lens.max())} slots")


if __name__ == "__main__":
    main()
