"""Decode with a bounded 8-bit key/value cache: the five cache ops as one loop uses them.

    python examples/long_context_decode.py [--steps N] [--budget TOKENS] [--fmt int8|e4m3]

A batch of sequences is filled by a prompt (KvAppend, KvAttention over all its rows), then takes one token a
step: KvAppend of the new K and V, KvAttention, KvScore of the weights.  A sequence that reaches the budget
is cut to half of it by KvEvict, into pages taken from the free list, and its old pages are given back.  The
model around the attention is a stand-in (random projections); what is shown is who owns what: the pool and
the free list are the program's, the ops only read and write pages that a table names.  At the end KvRead
shows what a sequence still holds.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from nemotron_ops_b200 import ops  # noqa: E402


class PagedCache:
    """The pool of one layer, its free pages, and the sequences' tables and lengths."""

    def __init__(self, sequences, capacity, heads, head_size, page=32, fmt=ops.KV_INT8, device="cuda"):
        self.page, self.fmt, self.width = page, fmt, -(-capacity // page)
        pages = sequences * self.width * 3 // 2 + sequences
        self.k, self.v = (torch.zeros(pages, heads, page, head_size, dtype=torch.uint8, device=device) for _ in range(2))
        self.ks, self.vs = (torch.zeros(pages, heads, device=device) for _ in range(2))
        self.free = list(range(pages))
        self.owned = [[] for _ in range(sequences)]
        self.table = torch.zeros(sequences, self.width, dtype=torch.int32, device=device)
        self.lens = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.length = [0] * sequences  # the host's copy: what pages are needed is decided without a transfer
        self.score = torch.zeros(sequences, heads, self.width * page, device=device)

    @property
    def buffers(self):
        return self.k, self.v, self.ks, self.vs

    def grow(self, rows):
        """Room for `rows` more tokens of every sequence; returns the start positions."""
        for s, pages in enumerate(self.owned):
            self.length[s] += rows
            need = -(-self.length[s] // self.page) - len(pages)
            if need > 0:
                new = [self.free.pop() for _ in range(need)]
                self.table[s, len(pages):len(pages) + need] = torch.tensor(new, dtype=torch.int32)
                pages += new
        start = self.lens.clone()
        self.lens += rows
        return start

    def evict(self, keep, sinks, recent):
        """Cut every sequence to `keep` tokens, in pages of their own; the old pages become free."""
        blocks = -(-keep // self.page)
        fresh = [[self.free.pop() for _ in range(blocks)] for _ in self.owned]
        new_table = torch.zeros_like(self.table)
        new_table[:, :blocks] = torch.tensor(fresh, dtype=torch.int32)
        kept, self.lens, score = ops.KvEvict(*self.buffers, self.table, self.lens, self.score, new_table, keep,
                                             sinks=sinks, recent=recent, fmt=self.fmt)
        self.score.zero_()
        self.score[:, :, :keep] = score
        for s, pages in enumerate(self.owned):
            self.free += pages  # later calls of this stream may write them: the moves come first
            self.length[s] = min(self.length[s], keep)
            self.owned[s] = fresh[s]
        self.table = new_table
        return kept


def attend(cache, qkv, heads, groups, head_size, start):
    """One layer's attention over rows [S, R, (groups + 2) * heads * head_size] of a fused projection."""
    q, k, v = qkv.split((groups * heads * head_size, heads * head_size, heads * head_size), -1)
    q, k, v = (x.unflatten(-1, (-1, head_size)) for x in (q, k, v))
    scale = head_size ** -0.5
    ops.KvAppend(k, v, *cache.buffers, cache.table, start, cache.lens, fmt=cache.fmt)
    o, lse = ops.KvAttention(q, *cache.buffers, cache.table, start, cache.lens, scale, fmt=cache.fmt)
    ops.KvScore(q, cache.k, cache.ks, cache.table, start, cache.lens, lse, cache.score, scale, fmt=cache.fmt)
    return o


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--sequences", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--budget", type=int, default=800)
    ap.add_argument("--fmt", choices=("int8", "e4m3"), default="int8")
    a = ap.parse_args(argv)
    heads, groups, head_size = 2, 4, 128
    width = (groups + 2) * heads * head_size
    torch.manual_seed(0)
    cache = PagedCache(a.sequences, max(a.budget, a.prompt) + 1, heads, head_size,
                       fmt=ops.KV_INT8 if a.fmt == "int8" else ops.KV_E4M3)
    out = torch.randn(groups * heads * head_size, width, device="cuda").mul_(0.05).bfloat16()
    x = torch.randn(a.sequences, a.prompt, width, device="cuda").bfloat16()
    o = attend(cache, x, heads, groups, head_size, cache.grow(a.prompt))
    evictions = 0
    for _ in range(a.steps):
        if cache.length[0] >= a.budget:
            cache.evict(a.budget // 2, sinks=4, recent=a.budget // 8)
            evictions += 1
        x = o[:, -1:].flatten(2) @ out + torch.randn(a.sequences, 1, width, device="cuda").bfloat16()
        o = attend(cache, x, heads, groups, head_size, cache.grow(1))
    zero = torch.zeros_like(cache.lens)
    k, _ = ops.KvRead(*cache.buffers, cache.table, zero, cache.lens, cache.length[0], fmt=cache.fmt)
    held = sum(map(len, cache.owned))
    print(f"{a.prompt} + {a.steps} tokens a sequence, {evictions} evictions, {cache.lens.tolist()} tokens held in "
          f"{held} pages; K of sequence 0 has norm {float(k[0].float().norm()):.1f}; device status {ops.device_status()}")
    return o, cache


if __name__ == "__main__":
    main()
