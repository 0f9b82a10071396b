#!/usr/bin/env python3
"""A serving loop over one block of a multi-stream residual model.

Each step of the loop is what a server does with a block's attention half:

  cache_update           the step's page table: rows go on, fork, end and grow
  cache_copy_pages       the private copies of partly filled pages that forks share
  mhc_pre                the block's input from its residual streams
  (projection)           a library product, queries, keys and values at once
  qk_norm_rope_append    norms, rotary positions, keys and values into the cache
  paged_attention        every new token over its row's pages
  (projection, mixing)   the output back into the streams
  cache_compact          now and then: the pages in use to the front of the pool

A prompt's chunk takes the same path: each of its tokens is a row of its own for
the attention, with the table of its sequence and the length up to itself.

    python examples/serve_block.py [--steps N] [--check]

--check recomputes every row's attention from the whole history of its inputs,
without a cache, and compares.
"""
from __future__ import annotations

import argparse
import math
import random
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import __graft_entry__  # noqa: E402


class ServedBlock:
    """A block's attention half with a paged cache of `pages` pages."""

    def __init__(self, rows=8, n=4, D=512, heads=8, kv_heads=2, d=64, page=16, pages=96, width=16, chunk=24, seed=0,
                 dtype=torch.bfloat16, device="cuda"):
        self.pkg = __graft_entry__.load_package()
        self.pkg.torch_ops()
        self.ops = torch.ops.mhcpre
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g).to(device)  # noqa: E731
        self.n, self.D, self.heads, self.kv_heads, self.d = n, D, heads, kv_heads, d
        self.page, self.pages, self.chunk, self.rows, self.device = page, pages, chunk, rows, device
        M = n * n + 2 * n
        self.phi = rand(M, n * D).div_(math.sqrt(n * D)).view(n * D, M)
        self.alpha, self.bias = torch.tensor([0.5, 0.3, 0.2], device=device), 0.1 * rand(M)
        self.w_qkv = rand(D, (heads + 2 * kv_heads) * d).div_(math.sqrt(D)).to(dtype)
        self.w_out = rand(heads * d, D).div_(math.sqrt(heads * d)).to(dtype)
        self.q_weight, self.k_weight = 1 + 0.1 * rand(d), 1 + 0.1 * rand(d)
        self.inv_freq = self.pkg.rotary_frequencies(d, kind="ramp", factor=4.0, device=device)
        # A head's slots of a page lie together, so that a wave reads whole pages.
        self.k_cache, self.v_cache = (torch.zeros(pages, kv_heads, page, d, dtype=dtype, device=device).transpose(1, 2)
                                      for _ in range(2))
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=device)

    def plan(self, parents, counts):
        """The step's pages: (slots [rows, S], granted [rows], positions [rows, S]) for S tokens a row."""
        S = max(1, max(counts))
        i32 = dict(dtype=torch.int32, device=self.device)
        self.table, self.lengths, slots, granted, src, dst = self.ops.cache_update(
            self.table, self.lengths, torch.tensor(parents, **i32), torch.tensor(counts, **i32), self.pages, self.page,
            S)
        self.ops.cache_copy_pages(self.k_cache, self.v_cache, src, dst)
        first = (self.lengths - granted)[:, None]
        return slots, granted, first + torch.arange(S, **i32)

    def forward(self, x, slots, granted, positions):
        """x [rows, S, n, D] to (x after the attention half, hIn, attention's output)."""
        rows, S = x.shape[:2]
        h_in, h_post, h_res = self.ops.mhc_pre(x, self.phi, self.alpha, self.bias)
        qkv = (h_in @ self.w_qkv).view(rows, S, self.heads + 2 * self.kv_heads, self.d)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 2)
        q = self.ops.qk_norm_rope_append(q, k, v, positions, self.inv_freq, slots, self.k_cache, self.v_cache,
                                         self.q_weight, self.k_weight)
        # A token sees its row up to itself; what is not a token of this step sees nothing.
        upto = torch.where(slots >= 0, positions + 1, 0).int()
        table = self.table if S == 1 else self.table.repeat_interleave(S, 0)
        o, _ = self.ops.paged_attention(q, self.k_cache, self.v_cache, table, upto)
        y = o.flatten(2) @ self.w_out
        mixed = (h_res[..., None] * x[:, :, None].float()).sum(3) + h_post[..., None] * y[:, :, None].float()
        return mixed.to(x.dtype), h_in, o

    def compact(self):
        """Moves the pages in use to the front; returns how many there are."""
        self.table, src, dst, used = self.ops.cache_compact(self.table, self.lengths, self.pages, self.page)
        self.ops.cache_copy_pages(self.k_cache, self.v_cache, src, dst)
        return used

    def plain_attention(self, history):
        """The last token's attention output from the inputs [t, D] of all its row's tokens, in 32 bits."""
        t = history.shape[0]
        qkv = (history @ self.w_qkv).float().view(t, -1, self.d)
        q, k, v = qkv[-1:, :self.heads], qkv[:, self.heads:self.heads + self.kv_heads], qkv[:, -self.kv_heads:]
        angle = torch.arange(t, device=self.device, dtype=torch.float64)[:, None] * self.inv_freq
        cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

        def turned(z, weight, c, s):
            z = z / torch.sqrt((z * z).mean(2, keepdim=True) + 1e-6) * weight
            a, b = z.chunk(2, 2)
            return torch.cat((a * c - b * s, a * s + b * c), 2).to(self.w_out.dtype).float()

        q, k = turned(q, self.q_weight, cos[-1:], sin[-1:]), turned(k, self.k_weight, cos, sin)
        k, v = (z.repeat_interleave(self.heads // self.kv_heads, 1) for z in (k, v))
        p = torch.softmax((q * k).sum(2) / math.sqrt(self.d), 0)
        return (p[:, :, None] * v).sum(0)


def serve(steps=24, check=False, seed=0, say=print):
    """Runs the loop; returns the largest difference from the plain attention (None without check)."""
    rng = random.Random(seed)
    block = ServedBlock(seed=seed)
    g = torch.Generator(device=block.device).manual_seed(seed)
    histories = [torch.zeros(0, block.D, dtype=torch.bfloat16, device=block.device)] * block.rows
    worst, tokens, forks = 0.0, 0, 0
    for step in range(steps):
        parents, counts = [], []
        for r in range(block.rows):
            kind = rng.random()
            if step == 0 or kind < 0.08:  # a new sequence: its prompt
                parents.append(-1)
                counts.append(rng.randint(1, block.chunk))
            else:
                parents.append(rng.randrange(block.rows) if kind < 0.2 else r)
                counts.append(1)
                forks += parents[-1] != r
        slots, granted, positions = block.plan(parents, counts)
        x = torch.randn(block.rows, slots.shape[1], block.n, block.D, generator=g, device=block.device)
        x, h_in, o = block.forward(x.to(torch.bfloat16), slots, granted, positions)
        granted = granted.tolist()
        tokens += sum(granted)
        histories = [torch.cat((histories[p][:0] if p < 0 else histories[p], h_in[r, :granted[r]]))
                     for r, p in enumerate(parents)]
        if check:
            for r, n in enumerate(granted):
                if n:
                    want = block.plain_attention(histories[r])
                    worst = max(worst, float((o[r, n - 1].float() - want).abs().max()))
        if step % 8 == 7:
            say(f"step {step + 1}: {int(block.compact())} of {block.pages} pages in use after compaction, "
                f"lengths {block.lengths.tolist()}")
    say(f"{tokens} tokens in {steps} steps, {forks} forks"
        + (f", largest difference from attention without a cache {worst:.3g}" if check else ""))
    return worst if check else None


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--check", action="store_true")
    args = ap.parse_args()
    serve(args.steps, args.check)
