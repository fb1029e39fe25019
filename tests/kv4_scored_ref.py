"""Plain 64-bit reference of the 4-bit cache's attention with capped scores,
distances and masks, on the CPU, with what its errors may be."""

from __future__ import annotations

import math

import torch

import kv4_ref as ref


def seen(n, m, causal=True, window=None, starts=None, prefix=None):
    """(m, n) which tokens each of a request's m queries sees."""
    t, p = torch.arange(n)[None, :], torch.arange(n - m, n)[:, None]
    ok = torch.ones(m, n, dtype=torch.bool)
    if causal:
        ok &= (t <= p) | (t < (0 if prefix is None else prefix))
    if window is not None:
        ok &= t > p - window
    if starts is not None:
        ok &= t >= starts[:, None]
    return ok


def attend(q, cache, tables, seq, nq, causal=True, sm_scale=None, max_seq=None, softcap=None,
           slopes=None, window=None, starts=None, prefix_lens=None, pick=None):
    """-> (out, lse, and the largest errors that the kernel's arithmetic allows
    of both), float64; of the rows pick (ascending) alone where it is given.

    Errors of a token's score in fp32, as a factor of its weight e^(1 + e_t):
      D products and sums, the key's scale and the score's:  (D + 12) 2^-24 |q| |k|
      1 - 2 / (1 + e^2x) with an exponential and a reciprocal of one unit in the
      last place (2^-23) each, of sums that are rounded to 2^-24: the reciprocal,
      at most 1, is off by 2^-22 and a quarter of the exponential's error, twice
      the cap times that below                                  cap 2^-20
      and for caps above 256 at most                               |z| 2^-18:
      where tanh is below 1/3 its series, 2^-22 of it left out and five
      roundings, and above that the same 2^-20 of the cap
      the distance's product, its sum and the difference to the maximum:
                                                              |bias| 2^-22
      the score itself, rounded in powers of two                  |z| 2^-22
      and 2^-21 for the exponential of the weight.
    A weight times its scale and the result are rounded to the type (u) once
    each; fp16's smallest numbers are 2^-25 off, and 2^-20 of the weights' sum
    bounds what is lost below them."""
    k_codes, v_codes, k_scales, v_scales, k_levels, v_levels = cache
    num_blocks, heads, bs, half = k_codes.shape
    T, H, D = q.shape
    G = H // heads
    u = ref.UNIT[q.dtype]
    sm_scale = D ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    tol = torch.zeros(T, H, D, dtype=torch.float64)
    lse_tol = torch.zeros(T, H, dtype=torch.float64)
    row = 0
    for r, (n, m) in enumerate(zip(seq, nq)):
        n = max(n, 0) if max_seq is None else min(max(n, 0), max_seq)
        rows = slice(row, row + m)
        ok = seen(n, m, causal, window, None if starts is None else starts[rows].long(),
                  None if prefix_lens is None else int(prefix_lens[r]))
        pos = torch.arange(n - m, n)
        if pick is not None:
            rows = torch.tensor([i for i in pick if row <= i < row + m], dtype=torch.long)
            ok, pos = ok[rows - row], pos[rows - row]
        t = torch.arange(n)
        blk = tables[r, t // bs].long() if n else t
        ok &= ((blk >= 0) & (blk < num_blocks))[None, :]
        row += m
        if not bool(ok.any()):
            continue
        some = ok.any(0)
        t, blk, ok = t[some], blk[some], ok[:, some]
        away = (pos[:, None] - t[None, :]).abs().double()
        alive = ok.any(1)
        for h in range(heads):
            k = ref.held(k_codes, k_scales, k_levels, blk, t % bs, h)
            v = ref.held(v_codes, v_scales, v_levels, blk, t % bs, h)
            for g in range(h * G, (h + 1) * G):
                qq = q[rows, g].double()
                z = sm_scale * qq @ k.T
                e = (D + 12) * 2.0 ** -24 * abs(sm_scale) * (qq.abs() @ k.abs().T)
                if softcap is not None:
                    z = softcap * torch.tanh(z / softcap)
                    e = e + (softcap * 2.0 ** -20 if softcap <= 256 else z.abs() * 2.0 ** -18)
                if slopes is not None:
                    bias = float(slopes[g]) * away
                    z = z - bias
                    e = e + bias.abs() * 2.0 ** -22
                e = e + z.abs() * 2.0 ** -22 + 2.0 ** -21
                z = z.masked_fill(~ok, -math.inf)
                top = torch.logsumexp(z, 1, keepdim=True)
                p = torch.where(alive[:, None], torch.exp(z - top), 0.0)
                e = torch.where(ok, e, 0.0)
                mine = torch.where(alive[:, None], p @ v, 0.0)
                mag = p @ v.abs()
                mean = (p * e).sum(1, keepdim=True)
                out[rows, g] = mine
                lse[rows, g] = torch.where(alive, top[:, 0], -math.inf)
                tol[rows, g] = (u * mine.abs() * 1.01 + (u * 1.01 + mean + 2.0 ** -20) * mag
                                + (p * e) @ v.abs() + 2.0 ** -25)
                lse_tol[rows, g] = mean[:, 0] + 2.0 ** -21 + torch.where(
                    alive, top[:, 0].abs(), 0.0) * 2.0 ** -22
    return out, lse, tol, lse_tol


# Prompts whose work per workgroup is many groups of 32 tokens and several items:
# (dtype, D, heads, query heads per head, block size, tokens, queries).
LONG_PROMPTS = [
    (torch.bfloat16, 64, 7, 4, 32, [3100, 1500, 2700], [3100, 1500, 1100]),
    (torch.float16, 128, 9, 3, 16, [2900, 1300, 3300], [2900, 1300, 900]),
    (torch.bfloat16, 256, 7, 5, 48, [3000, 1100, 2300], [3000, 1100, 1000])]
LONG_OPTIONS = [("cap",), ("slopes", "prefix"), ("window",), ("docs",),
                ("cap", "slopes", "window", "docs", "prefix")]
LONG_WINDOW, LONG_DOCUMENTS = 1700, 2000


def replay(D, heads, G, seq, nq, cus, causal=True, window=None, starts=None, prefix_lens=None):
    """The shares that the form for prompts cuts its work into, as lists of
    (head, tile, first token, last token, whether the item goes on in the next
    share): csrc/kv4_attend_scored.hip's walk over tiles of 16 rows a wave."""
    cols, overhead = (192 if D == 256 else 256), (10 if D == 64 else 6)
    tiles, row = [], 0
    for r, (n, m) in enumerate(zip(seq, nq)):
        p = torch.arange(n - m, n)
        last = torch.full((m,), n) if not causal else (p + 1).clamp(
            min=0 if prefix_lens is None else int(prefix_lens[r])).clamp(0, n)
        first = torch.zeros(m, dtype=torch.long)
        if window is not None:
            first = (p - window + 1).clamp(min=0)
        if starts is not None:
            first = torch.maximum(first, starts[row:row + m].long())
        for col in range(0, m * G, cols):
            i = slice(col // G, (min(col + cols, m * G) - 1) // G + 1)
            some = first[i] < last[i]
            lo = int(first[i][some].min()) // 16 * 16 if bool(some.any()) else 0
            hi = int(last[i][some].max()) if bool(some.any()) else 0
            tiles.append((lo, hi, overhead + -(-(hi - lo) // 32) if hi > lo else 2))
        row += m
    items = [(h, t, *tile) for h in range(heads) for t, tile in enumerate(tiles)]
    total = sum(x[4] for x in items)
    share = max(-(-total // cus), 2)
    shares, at, x = [], 0, 0
    while x < len(items):
        left, mine = share, []
        while left and x < len(items):
            h, t, lo, hi, n = items[x]
            end = min(n, at + left)
            token = [hi if a == n else min(lo + max(a - overhead, 0) * 32, hi) for a in (at, end)]
            if token[0] < token[1] or (lo == hi and end == n):
                mine.append((h, t, *token, token[1] < hi))
            left -= end - at
            at = end
            if end == n:
                x, at = x + 1, 0
        shares.append(mine)
    return shares
