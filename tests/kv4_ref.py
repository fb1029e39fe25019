"""Plain 64-bit references of the 4-bit cache's operators, on the CPU."""

from __future__ import annotations

import math

import numpy as np
import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # largest rounding error


def random_levels(heads, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    lv = torch.erfinv(2 * (torch.arange(16) + 0.5) / 16 - 1) * 0.5
    lv = lv * (1 + 0.2 * torch.rand(heads, 1, generator=g))
    order = torch.rand(heads, 16, generator=g).argsort(1)
    return lv.gather(1, order).to(dtype)


def random_cache(num_blocks, heads, bs, D, dtype, seed, k_mean=2.8, v_mean=1.4):
    """The six tensors of a cache, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randint(0, 256, (num_blocks, heads, bs, D // 2), generator=g,
                           dtype=torch.uint8) for _ in range(2)]
    scales = [(m * torch.exp(0.3 * torch.randn(num_blocks, heads, bs, generator=g))).to(dtype)
              for m in (k_mean, v_mean)]
    return [*codes, *scales, random_levels(heads, dtype, seed + 1),
            random_levels(heads, dtype, seed + 2)]


def held(codes, scales, levels, blk, off, h):
    """Vectors (n, D) of head h in 64 bits."""
    c = codes[blk, h, off].long()
    both = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    return levels[h].double()[both] * scales[blk, h, off].double()[:, None]


def attend(q, cache, tables, seq, nq, causal=True, sm_scale=None, max_seq=None):
    """-> (out, lse, weight of |v|, bound of sum |q k|), all (T, H, ...) float64."""
    k_codes, v_codes, k_scales, v_scales, k_levels, v_levels = cache
    num_blocks, heads, bs, half = k_codes.shape
    T, H, D = q.shape
    G = H // heads
    sm_scale = D ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    mag = torch.zeros(T, H, D, dtype=torch.float64)
    zabs = torch.zeros(T, H, dtype=torch.float64)
    row = 0
    for r, (n, m) in enumerate(zip(seq, nq)):
        n = max(n, 0) if max_seq is None else min(max(n, 0), max_seq)
        t = torch.arange(n)
        blk = tables[r, t // bs].long() if n else t
        ok = (blk >= 0) & (blk < num_blocks)
        t, blk = t[ok], blk[ok]
        off = t % bs
        for h in range(heads):
            if not len(t):
                break
            k = held(k_codes, k_scales, k_levels, blk, off, h)
            v = held(v_codes, v_scales, v_levels, blk, off, h)
            for i in range(m):
                see = t <= (n - m + i) if causal else torch.ones_like(t, dtype=torch.bool)
                if not bool(see.any()):
                    continue
                qq = q[row + i, h * G:(h + 1) * G].double()
                z = sm_scale * qq @ k[see].T
                top = z.amax(1, keepdim=True)
                p = torch.exp(z - top)
                s = p.sum(1, keepdim=True)
                hs = slice(h * G, (h + 1) * G)
                out[row + i, hs] = p @ v[see] / s
                mag[row + i, hs] = p @ v[see].abs() / s
                lse[row + i, hs] = (top + s.log())[:, 0]
                zabs[row + i, hs] = abs(sm_scale) * (qq.abs() @ k[see].abs().T).amax(1)
        row += m
    return out, lse, mag, zabs


def attend_tolerances(ref, D, dtype):
    """Largest errors of out and lse that the kernel's arithmetic allows.

    Score: D products and sums in fp32, a few roundings more, and exp2 to
    2^-21: a weight is off by e = (D + 8) 2^-24 sum |q k| + 2^-21 relative,
    numerator and denominator each.  Weight times scale and the result are
    rounded to the type once each (u); fp16 results below its normal range
    are 2^-25 off."""
    out, lse, mag, zabs = ref
    u = UNIT[dtype]
    e = (D + 8) * 2.0 ** -24 * zabs + 2.0 ** -21
    tol = u * out.abs() * 1.01 + (u * 1.01 + 2 * e[..., None] + 2.0 ** -20) * mag + 2.0 ** -25
    return tol, e + 2.0 ** -21 + lse.abs().nan_to_num(posinf=0.0) * 2.0 ** -22


def quantise(x, levels):
    """(codes, scales as fp32, values as float64) of x (T, heads, D) by the
    definition: fp32 quotient and distances, lowest index of equal ones."""
    with np.errstate(all="ignore"):
        a = x.float().numpy()
        lv = levels.float().numpy()
        s = np.abs(a).max(-1)
        s = np.where(s < np.float32(2.0 ** -126), np.float32(0), s).astype(np.float32)
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0)).astype(np.float32)
        y = a * inv[..., None]
        best = np.abs(y - lv[:, 0][None, :, None])
        code = np.zeros(a.shape, np.int64)
        for c in range(1, 16):
            d = np.abs(y - lv[:, c][None, :, None])
            less = d < best
            code[less] = c
            best = np.where(less, d, best)
        val = lv.astype(np.float64)[np.arange(a.shape[1])[None, :, None], code] * \
            s.astype(np.float64)[..., None]
    return code, s, val


def block_tables(seq, new, tables, free, bs, num_tokens):
    """(tables, slots, cu_new, taken) by walking the requests."""
    tables = tables.copy()
    slots, cu, taken = [], [0], 0
    for r, (n, m) in enumerate(zip(seq, new)):
        n = max(n, 0)
        m = min(max(m, 0), n)
        held_blocks = -(-(n - m) // bs)
        for j in range(held_blocks, -(-n // bs)):
            if j < tables.shape[1]:
                tables[r, j] = free[taken] if taken < len(free) else -1
            taken += 1
        for p in range(n - m, n):
            b = tables[r, p // bs] if p // bs < tables.shape[1] else -1
            slots.append(b * bs + p % bs if b >= 0 else -1)
        cu.append(cu[-1] + m)
    slots = (slots + [-1] * num_tokens)[:num_tokens]
    return tables, np.array(slots, np.int32).reshape(-1), np.array(cu, np.int32), taken
