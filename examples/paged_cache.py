"""Answering from long contexts with a paged key-value cache and retrieval.

Several requests with prompts of different lengths share one cache.  Their
prompts are written and attended to in one step; then each step adds a token to
every request, which attends to the blocks of its context that score best for
it (and, for comparison, to all of them).  With a budget every request is cut to
the tokens that got most attention, after its prompt and whenever it has grown by a
page since.  One attention layer with random weights stands for the model.

    python examples/paged_cache.py [--requests 8] [--context 16384] [--steps 32]
                                   [--budget 4096]
"""

from __future__ import annotations

import argparse
import time
from pathlib import Path
import sys

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch  # noqa: E402

import mlxvs_amd as mlxvs  # noqa: E402

HEADS, KV_HEADS, DIM, PAGE, WIDTH = 32, 8, 128, 64, 1024


class Layer:
    """Queries, keys and values of a token from its features."""

    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.qkv = (torch.randn(WIDTH, (HEADS + 2 * KV_HEADS) * DIM, generator=g, device="cuda")
                    * WIDTH ** -0.5).bfloat16()
        self.out = (torch.randn(HEADS * DIM, WIDTH, generator=g, device="cuda")
                    * (HEADS * DIM) ** -0.5).bfloat16()

    def project(self, x):
        # (strided views of one product's rows: the cache takes them as they are)
        q, k, v = (x @ self.qkv).split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], dim=1)
        return q.unflatten(1, (HEADS, DIM)), k.unflatten(1, (KV_HEADS, DIM)), \
            v.unflatten(1, (KV_HEADS, DIM))


def run(requests=8, context=16384, steps=32, blocks=32, seed=0, budget=0):
    """Returns the lengths at the end, the mean cosine of the two answers' outputs
    and the mean time of a decoding step in milliseconds.  budget: tokens of a
    request that are kept, 0 for all."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = dict(dtype=torch.int32, device="cuda")
    prompts = [max(1, context * (i + 1) // requests - 7 * i) for i in range(requests)]
    columns = -(-(max(prompts) + steps) // PAGE)
    pages = sum(-(-(p + steps) // PAGE) for p in prompts)

    layer = Layer(seed)
    cache = mlxvs.PagedKVCache.empty(pages, KV_HEADS, PAGE, DIM)
    table = torch.full((requests, columns), -1, **ints)
    free = torch.randperm(pages, generator=g, device="cuda").int()
    cursor = torch.zeros(1, **ints)  # how much of the free list is taken
    lengths = torch.zeros(requests, **ints)
    rotary = mlxvs.Rotary(DIM)
    evicted = torch.zeros(requests, **ints)  # tokens of a request that the cache has lost
    longest = max(prompts) + (0 if budget else steps)  # tokens that a request holds at most
    mass = torch.zeros(requests, KV_HEADS, columns * PAGE, device="cuda") if budget else None

    def cut(q, plan, lse):
        """The step's attention counted, and the requests cut that hold a page too many."""
        nonlocal lengths, cursor, evicted, longest
        cache.weigh(q, table, plan.starts, plan.positions, lse, mass, longest=longest)
        kept = cache.keep(mass, plan.lengths, budget, first=min(4, budget // 2),
                          recent=min(2 * PAGE, budget // 2), above=budget + PAGE - 1)
        lengths, cursor = cache.compact(table, plan.lengths, kept, free, plan.cursor, mass=mass)
        evicted = evicted + plan.lengths - lengths
        longest = budget + PAGE

    # the prompts, all tokens in one step
    total = sum(prompts)
    plan = mlxvs.kv_plan(lengths, torch.tensor(prompts, **ints), table, free, cursor, PAGE, total)
    x = torch.randn(total, WIDTH, generator=g, device="cuda").bfloat16()
    q, k, v = layer.project(x)
    q, k = rotary.rotate(q, k, plan.positions)
    cache.append(k, v, plan.slots)
    out, lse = cache.attend(q, table, plan.requests, plan.positions, longest=longest, lse=True)
    last = torch.tensor(prompts, device="cuda").cumsum(0) - 1  # the prompts' last tokens
    x = torch.tanh(out[last].flatten(1) @ layer.out)
    lengths, cursor = plan.lengths, plan.cursor
    if budget:
        cut(q, plan, lse)

    one = torch.ones(requests, **ints)
    close, spent = 0.0, 0.0
    for i in range(steps):
        torch.cuda.synchronize()
        start = time.perf_counter()
        plan = mlxvs.kv_plan(lengths, one, table, free, cursor, PAGE, requests)
        q, k, v = layer.project(x)
        q, k = rotary.rotate(q, k, plan.positions, requests=plan.requests, evicted=evicted)
        cache.append(k, v, plan.slots)
        best = cache.select(q, table, plan.requests, plan.positions, blocks, last=2)
        out = cache.attend(q, table, plan.requests, plan.positions, blocks=best)
        x = torch.tanh(out.flatten(1) @ layer.out)
        lengths, cursor = plan.lengths, plan.cursor
        torch.cuda.synchronize()
        spent += time.perf_counter() - start if i else 0.0  # (the first one warms up)
        full, lse = cache.attend(q, table, plan.requests, plan.positions, longest=longest, lse=True)
        if budget:
            cut(q, plan, lse)
        close += torch.cosine_similarity(out.float().flatten(1), full.float().flatten(1)).mean() \
            .item()
    return lengths.tolist(), close / max(1, steps), 1e3 * spent / max(1, steps - 1)


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--requests", type=int, default=8)
    p.add_argument("--context", type=int, default=16384, help="tokens of the longest prompt")
    p.add_argument("--steps", type=int, default=32, help="tokens to answer with")
    p.add_argument("--blocks", type=int, default=32, help="blocks of 64 tokens to attend to")
    p.add_argument("--budget", type=int, default=0, help="tokens of a request to keep (0: all)")
    a = p.parse_args()
    lengths, close, ms = run(a.requests, a.context, a.steps, a.blocks, budget=a.budget)
    print(f"{a.requests} requests of {min(lengths)} to {max(lengths)} tokens, {a.steps} steps of "
          f"{ms:.3f} ms; {a.blocks} selected blocks against all: cosine {close:.4f}")


if __name__ == "__main__":
    main()
