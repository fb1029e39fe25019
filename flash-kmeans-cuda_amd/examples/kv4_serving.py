"""A serving loop over a 4-bit key/value cache whose levels k-means learned.

Learns sixteen levels per head from a sample of keys and values, prefills a
ragged batch of prompts and decodes a few tokens of each, every step with the
same four calls: block tables, append, attend, and the caller's own work in
between (random here).  Prints how far the attention is from that over the
unquantised keys and values.

    python flash-kmeans-cuda_amd/examples/kv4_serving.py
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from flash_kmeans_cuda import kv4  # noqa: E402

HEADS, GROUP, DIM, BLOCK = 2, 4, 128, 64  # cache heads, query heads of each


class Loop:
    """What a server keeps: the cache, the block tables and the free list."""

    def __init__(self, levels, requests: int, num_blocks: int, max_blocks: int) -> None:
        self.cache = kv4.Cache.empty(num_blocks, BLOCK, DIM, *levels, torch.bfloat16)
        self.tables = torch.full((requests, max_blocks), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(num_blocks, device="cuda").to(torch.int32)
        self.seq = torch.zeros(requests, dtype=torch.int32, device="cuda")

    def step(self, new: torch.Tensor, q, k, v) -> torch.Tensor:
        """Append the new tokens (`new` per request) and attend from them."""
        self.seq = self.seq + new
        slots, cu, taken = kv4.block_tables(self.seq, new, self.tables, self.free, BLOCK, len(k))
        kv4.append(self.cache, k, v, slots)
        # A server keeps its list on the host, where the lengths tell what is
        # taken; reading the count here waits for the GPU.
        if int(taken) > len(self.free):
            raise RuntimeError("the cache is full")
        self.free = self.free[int(taken):]
        return kv4.attend(q, self.cache, self.tables, self.seq, cu)


def plain(q, ks, vs, lens, new):
    """The same attention over the exact keys and values, request by request."""
    out, at = [], 0
    for k, v, n, m in zip(ks, vs, lens, new):
        rows = q[at:at + m].float().view(m, HEADS, GROUP, DIM)
        z = torch.einsum("mhgd,nhd->mhgn", rows, k.float()) * DIM ** -0.5
        seen = torch.arange(n, device=q.device) <= torch.arange(n - m, n, device=q.device)[:, None]
        z = z.masked_fill(~seen[:, None, None], float("-inf"))
        out.append(torch.einsum("mhgn,nhd->mhgd", z.softmax(-1), v.float()).reshape(m, -1, DIM))
        at += m
    return torch.cat(out)


def main(steps: int = 4, seed: int = 0) -> float:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def vectors(n, heads=HEADS):
        return torch.randn(n, heads, DIM, generator=g, device="cuda").to(torch.bfloat16)

    levels = kv4.learn_levels(vectors(512)), kv4.learn_levels(vectors(512))
    prompts = [200, 33, 700, 1]
    loop = Loop(levels, len(prompts), 64, 16)
    ks, vs = [[vectors(0) for _ in prompts] for _ in range(2)]
    worst = 0.0
    for step in range(steps + 1):
        new = prompts if step == 0 else [1] * len(prompts)
        k, v, q = vectors(sum(new)), vectors(sum(new)), vectors(sum(new), HEADS * GROUP)
        ks = [torch.cat(p) for p in zip(ks, k.split(new))]
        vs = [torch.cat(p) for p in zip(vs, v.split(new))]
        out = loop.step(torch.tensor(new, dtype=torch.int32, device="cuda"), q, k, v)
        want = plain(q, ks, vs, [len(x) for x in ks], new)
        err = float((out.float() - want).norm() / want.norm())
        worst = max(worst, err)
        print(f"step {step}: {sum(new)} new tokens, {int(loop.seq.sum())} cached, "
              f"4-bit attention off by {100 * err:.1f}%")
    return worst


if __name__ == "__main__":
    main()
