"""Serving a decoder block over a paged key-value cache: several conversations
of different lengths share one pool of pages, their prompts enter together, and
each then gets a token a step.  With --budget the cache of a conversation is held
at that many tokens: after every step the token of least accumulated attention
weight leaves it.

    python burn-extended_b200/examples/paged_decode.py [--steps 64] [--budget 96]

The block is attention (append, decode, evict on mxmoe.paged) and the MXFP4
mixture of experts (mxmoe.MoeGatedSwiGLU), with random weights; the projections
are torch products.  What it prints is checked against dense attention over all
tokens in 32 bits."""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import mxmoe  # noqa: E402
from mxmoe import synth  # noqa: E402
from mxmoe.paged import PagedKvCache, RotaryConfig, RotaryTable  # noqa: E402

D, HEADS, KV_HEADS, HEAD_DIM, PAGE = 256, 16, 2, 64, 16


class Block:
    """One decoder block with random weights."""

    def __init__(self, seed=0):
        inp = synth.make_inputs(D, 256, 4, 2, 1, True, seed=seed)
        self.moe = mxmoe.MoeConfig(inp.d, inp.f, inp.E, inp.k).init(0)
        self.moe.set_router(inp.gamma, inp.gate_w, inp.gate_b)
        self.moe.set_resident(inp.host, inp.b1 * 1e-3, inp.b2 * 1e-3)
        g = torch.Generator("cuda").manual_seed(seed)

        def weight(a, b):
            return (torch.randn(a, b, device="cuda", generator=g) / a ** 0.5).bfloat16()

        self.qkv, self.out = weight(D, (HEADS + 2 * KV_HEADS) * HEAD_DIM), weight(HEADS * HEAD_DIM, D)
        self.sinks = torch.randn(HEADS, device="cuda", generator=g)

    def heads(self, x):
        h = (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-5)).bfloat16()
        n = [HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM]
        return [t.unflatten(1, (-1, HEAD_DIM)) for t in (h @ self.qkv).split(n, 1)]


class Pages:
    """The caller's book-keeping: which pages are free."""

    def __init__(self, n):
        self.free = list(range(n))

    def rows(self, counts, width):
        table = np.zeros((len(counts), width), np.int32)
        for i, n in enumerate(counts):
            table[i, :n] = [self.free.pop() for _ in range(n)]
        return torch.from_numpy(table).cuda()


def dense(q, k, v, sinks, positions, rotary):
    """The last token's attention over all tokens, in 32 bits."""
    q, k = (rotary.apply(t.contiguous(), positions[-t.shape[0]:]).float() for t in (q, k))
    k, v = (t.float().repeat_interleave(HEADS // KV_HEADS, 1) for t in (k, v))
    s = torch.einsum("hd,nhd->hn", q[-1], k) / HEAD_DIM ** 0.5
    p = torch.softmax(torch.cat([s, sinks[:, None]], 1), 1)[:, :-1]
    return torch.einsum("hn,nhd->hd", p, v)


def serve(prompts=(40, 7, 120, 1), steps=32, budget=0, seed=0):
    """-> (largest distance from dense attention over the steps, relative to its largest value; cached tokens by step)."""
    block, rows = Block(seed), len(prompts)
    rotary = RotaryTable.of(RotaryConfig(HEAD_DIM, scaling="yarn", scaling_factor=32.0), 4096)
    most = max(prompts) + steps if budget == 0 else max(max(prompts), budget) + 1
    width = -(-most // PAGE)
    pages = Pages(rows * width)
    tables = pages.rows([width] * rows, width)
    cache = PagedKvCache(rows * width, PAGE, HEADS, KV_HEADS, HEAD_DIM, torch.bfloat16, track=True)
    g = torch.Generator("cuda").manual_seed(seed + 1)

    # The prompts' tokens in one call; each attends as a row of its own to those before it.
    row = np.repeat(np.arange(rows), prompts)
    index = np.concatenate([np.arange(n) for n in prompts])
    row_t, index_t = (torch.from_numpy(a.astype(np.int32)).cuda() for a in (row, index))
    x = torch.randn(len(row), D, device="cuda", generator=g).bfloat16()
    q, k, v = block.heads(x)
    kept = [[[t[row == i]] for t in (k, v)] for i in range(rows)]  # for the check alone
    q = cache.append(q, k, v, tables, index_t, rotary, rows=row_t)
    att = cache.decode(q, tables[row_t.long()].contiguous(), index_t + 1, sinks=block.sinks)
    x = block.moe.forward(x + att.flatten(1) @ block.out)

    ends = np.cumsum(prompts) - 1
    x = x[torch.from_numpy(ends).cuda()].contiguous()
    seen = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    lens, far, sizes = seen.clone(), 0.0, []
    if budget:
        lens = cache.evict(tables, lens, seen, budget, recent=budget // 4)
    for _ in range(steps):
        q, k, v = block.heads(x)
        turned = cache.append(q, k, v, tables, lens, rotary, positions=seen)
        lens, seen = lens + 1, seen + 1
        att = cache.decode(turned, tables, lens, sinks=block.sinks, track=True)
        for i in range(rows):
            for t, new in zip(kept[i], (k, v)):
                t.append(new[i:i + 1])
            at = torch.arange(int(seen[i]), dtype=torch.int32, device="cuda")
            want = dense(q[i:i + 1], torch.cat(kept[i][0]), torch.cat(kept[i][1]), block.sinks, at, rotary)
            far = max(far, float((att[i].float() - want).abs().max() / want.abs().max()))
        x = block.moe.forward(x + att.flatten(1) @ block.out)
        x = (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-5)).bfloat16()  # keeps random weights tame
        if budget:
            lens = cache.evict(tables, lens, seen, budget, recent=budget // 4)
        sizes.append(lens.tolist())
    cache.sync_status()
    block.moe.sync_status()
    return far, sizes


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--budget", type=int, default=0, help="cached tokens of a conversation; 0: all")
    a = ap.parse_args()
    far, sizes = serve(steps=a.steps, budget=a.budget)
    print(f"cached tokens after {a.steps} steps: {sizes[-1]}; largest distance from dense attention: {far:.2e}")


if __name__ == "__main__":
    main()
