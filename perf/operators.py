"""Operators around a key/value cache held in 4 bits, measured case by case.

The cache stores each key and value vector as D 4-bit codes into 16 levels of
its head (centroids that the package's k-means learns) and one scale.  Three
kinds of work, as a serving loop meets them:

* "tables": one `kv4.block_tables` call, at the start of a step: the blocks
  and cache slots of the step's new tokens from the requests' lengths;
* "append": one `kv4.append` call with the step's keys and values, and one
  `kv4.read` of the same slots (what 4 bits hold is returned as the values
  they stand for);
* "attend": one `kv4.attend` call, the step's queries over the cache: single
  tokens, a few drafted tokens each, and prompts.

`own` chooses between the package's kernels and the same formulas in plain
torch operations.  Lengths are drawn from the case's own `lens` seed, so that
the work of a case is known without a GPU; everything else from `seed`.
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
LEVELS = 16
MIN_SCALE = 2.0 ** -126  # vectors below it are stored as zero


def _kv4():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "flash-kmeans-cuda_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from flash_kmeans_cuda import kv4
    return kv4


def _tables(name, R, seq, new, block_size, pad, lens, idle=0):
    c = {"op": "tables", "R": R, "seq_lo": seq[0], "seq_hi": seq[1], "new_lo": new[0],
         "new_hi": new[1], "block_size": block_size, "pad": pad, "lens": lens, "idle": idle}
    return c if name is None else {"name": name, **c}


def _append(name, dtype, T, Hkv, D, block_size, fused):
    c = {"op": "append", "dtype": dtype, "T": T, "Hkv": Hkv, "D": D,
         "block_size": block_size, "fused": fused}
    return c if name is None else {"name": name, **c}


def _attend(name, dtype, R, seq, q, Hkv, G, D, block_size, lens, idle=0, lse=False, fused=False):
    c = {"op": "attend", "dtype": dtype, "R": R, "seq_lo": seq[0], "seq_hi": seq[1],
         "q_lo": q[0], "q_hi": q[1], "Hkv": Hkv, "G": G, "D": D, "block_size": block_size,
         "lens": lens, "idle": idle, "lse": lse, "fused": fused}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # The step of a small batch: one new token each, a handful of launches'
        # worth of latency and nothing else.
        _tables("tables_decode", 37, (1, 4096), (1, 1), 16, 11, 1, idle=5),
        # A large mixed step: prompts of every length beside single tokens.
        _tables("tables_mixed", 2048, (1, 16384), (1, 512), 64, 1000, 2),
        # One decoding step's keys and values, sliced from the fused projection.
        _append("append_decode", "bf16", 64, 8, 128, 16, True),
        # A prompt of odd length.
        _append("append_prompt", "f16", 8191, 8, 128, 64, False),
        # The tokens of a whole prefill batch, many small heads.
        _append("append_batch", "bf16", 32768, 16, 64, 128, False),
        # The smallest answer: one request with a short context.
        _attend("decode_one", "bf16", 1, (517, 517), (1, 1), 8, 4, 128, 16, 3),
        # An ordinary decoding batch, ragged, some of its rows idle.
        _attend("decode_batch", "bf16", 64, (1024, 32768), (1, 1), 8, 4, 128, 64, 4, idle=3,
                fused=True),
        # Two very long contexts: the only parallelism is along the context.
        _attend("decode_long", "f16", 2, (100003, 131071), (1, 1), 4, 16, 128, 128, 5),
        # Heads that share nothing, of 64 columns.
        _attend("decode_mha64", "f16", 48, (200, 4096), (1, 1), 16, 1, 64, 32, 6),
        # Checking a few drafted tokens per request at once; the statistics
        # of each row are kept, to join it with attention over other keys.
        _attend("verify_drafts", "bf16", 40, (300, 8192), (2, 7), 8, 4, 128, 16, 7, lse=True),
        # Prompts from the first token on, ragged.
        _attend("prefill", "bf16", 5, (700, 4096), (700, 4096), 8, 4, 128, 64, 8),
        # A chunk of new tokens behind a long cached prefix, wide heads.
        _attend("prefill_chunk256", "f16", 2, (12000, 16000), (1000, 1500), 2, 8, 256, 64, 9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    lens = rng.randrange(1 << 30)
    op = rng.choice(["tables", "append", "attend", "attend", "attend"])
    if op == "tables":
        R = _log_int(rng, 1, 4096)
        hi = _log_int(rng, 1, 32768)
        new = 1 if rng.random() < 0.5 else min(hi, _log_int(rng, 1, max(1, (1 << 17) // R)))
        return _tables(None, R, (1, hi), (1, new), rng.choice([16, 32, 48, 64, 128]),
                       rng.randrange(0, 2000), lens, idle=rng.randrange(3) if R > 2 else 0)
    dtype = rng.choice(["f16", "bf16"])
    D = rng.choice([64, 128, 128, 256])
    if op == "append":
        Hkv = rng.choice([1, 2, 4, 5, 8, 16])
        T = _log_int(rng, 1, 65536 * 8 * 64 // (Hkv * D))
        return _append(None, dtype, T, Hkv, D, rng.choice([16, 32, 48, 64, 128]),
                       rng.random() < 0.5)
    Hkv = rng.choice([1, 2, 4, 5, 8, 16])
    G = rng.choice([1, 2, 3, 4, 7, 8, 16])
    bs = rng.choice([16, 32, 48, 64, 128])
    kind = rng.choice(["decode", "drafts", "prompt"])
    if kind == "prompt":
        # Pairs of a query and a key it may see, over all heads and columns.
        budget = 1 << 36
        hi = _log_int(rng, 1, 8192)
        R = max(1, min(8, budget // (Hkv * G * D * hi * hi)))
        hi = max(1, min(hi, math.isqrt(budget // (R * Hkv * G * D))))
        pre = _log_int(rng, 1, 8192) if rng.random() < 0.5 else 0
        pre = min(pre, max(0, budget // (R * Hkv * G * D * hi) - hi))
        return _attend(None, dtype, R, (pre + 1, pre + hi), (1, hi), Hkv, G, D, bs, lens,
                       lse=rng.random() < 0.3)
    hi = _log_int(rng, 1, 131072)
    top = (1 << 29) // (Hkv * D * hi)  # elements of keys in the cache
    R = _log_int(rng, 1, max(1, min(256, top)))
    hi = max(1, min(hi, (1 << 29) // (Hkv * D * R)))
    q = (1, 1) if kind == "decode" else (1, rng.randrange(2, 9))
    lo = 1 if rng.random() < 0.5 else hi
    return _attend(None, dtype, R, (lo, hi), q, Hkv, G, D, bs, lens,
                   idle=rng.choice([0, 0, 1]) if R > 1 else 0, lse=rng.random() < 0.3,
                   fused=rng.random() < 0.3)


def _lengths(case):
    """(tokens per request after the step, new tokens or queries of the step)."""
    rng = random.Random(case["lens"])
    a, b = ("new_lo", "new_hi") if case["op"] == "tables" else ("q_lo", "q_hi")
    seq, new = [], []
    for r in range(case["R"]):
        # A prompt from its first token on has as many queries as tokens.
        s = _log_int(rng, case["seq_lo"], case["seq_hi"])
        whole = case["op"] == "attend" and case[a] == case["seq_lo"] and case[b] == case["seq_hi"]
        n = s if whole and case[b] > 1 else min(s, _log_int(rng, case[a], case[b]))
        if r < case.get("idle", 0):
            # a decoding batch keeps its idle rows
            s, n = 0, (1 if case["op"] == "attend" and case["q_hi"] == 1 else 0)
        seq.append(s)
        new.append(n)
    return seq, new


def work(case):
    if case["op"] == "tables":
        seq, new = _lengths(case)
        bs = case["block_size"]
        fresh = sum(-(-s // bs) - -(-(s - n) // bs) for s, n in zip(seq, new))
        old = sum(1 for s, n in zip(seq, new) if (s - n) % bs)
        out = sum(new) + case["pad"] + len(seq) + 2
        return {"bytes": 4 * (2 * len(seq) + 2 * fresh + old + out), "flops": 0}
    if case["op"] == "append":
        vec, D = 2 * case["T"] * case["Hkv"], case["D"]
        # keys and values in; codes and scales, and the values they stand for, out
        return {"bytes": vec * (2 * D + D // 2 + 2 + 2 * D) + 4 * case["T"],
                "flops": vec * D * 6}
    seq, nq = _lengths(case)
    D, Hkv, H = case["D"], case["Hkv"], case["Hkv"] * case["G"]
    pairs = sum(n * (s - n) + n * (n + 1) // 2 for s, n in zip(seq, nq) if s)
    return {"bytes": sum(seq) * Hkv * (D + 4) + sum(nq) * H * (4 * D + (4 if case["lse"] else 0))
            + 4 * sum(-(-s // case["block_size"]) for s in seq),
            "flops": 4 * D * H * pairs}


def _ints(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _block_map(seq, bs, spare, g):
    """Block tables over a shuffled pool: (tables, unused blocks)."""
    n = [-(-s // bs) for s in seq]
    pool = torch.randperm(sum(n) + spare, generator=g, device="cuda").to(torch.int32)
    tables = torch.zeros(len(seq), max(max(n), 1), dtype=torch.int32, device="cuda")
    rows = torch.repeat_interleave(torch.arange(len(seq)), torch.tensor(n))
    first = torch.tensor([0] + n[:-1]).cumsum(0)
    cols = torch.arange(sum(n)) - first[rows]
    tables[rows.cuda(), cols.cuda()] = pool[:sum(n)]
    return tables, pool[sum(n):].contiguous()


def _levels(Hkv, g, dtype):
    """Sixteen levels per head as k-means finds them for normal columns over
    their vector's largest magnitude: near the normal's quantiles, a little
    different in every head, in no particular order."""
    p = (torch.arange(LEVELS, device="cuda") + 0.5) / LEVELS
    lv = torch.erfinv(2 * p - 1) * 0.5
    lv = lv * (1 + 0.1 * torch.rand(Hkv, 1, generator=g, device="cuda"))
    lv = lv + 0.01 * torch.randn(Hkv, LEVELS, generator=g, device="cuda")
    order = torch.rand(Hkv, LEVELS, generator=g, device="cuda").argsort(1)
    return lv.gather(1, order).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "tables":
        seq, new = _lengths(case)
        bs = case["block_size"]
        held = [a - b for a, b in zip(seq, new)]
        need = sum(-(-a // bs) - -(-h // bs) for a, h in zip(seq, held))
        tab, free = _block_map(held, bs, need + 64, g)
        tables = torch.full((len(seq), -(-max(seq) // bs)), -1, dtype=torch.int32, device="cuda")
        w = min(tab.shape[1], tables.shape[1])
        cols = torch.arange(w, device="cuda")
        have = (_ints(held) + bs - 1) // bs
        tables[:, :w] = torch.where(cols < have[:, None], tab[:, :w], tables[:, :w])
        s.update(seq=_ints(seq), new=_ints(new), tables=tables, free=free,
                 num_tokens=sum(new) + case["pad"])
    else:
        dtype, Hkv, D, bs = DTYPES[case["dtype"]], case["Hkv"], case["D"], case["block_size"]
        s["k_levels"], s["v_levels"] = _levels(Hkv, g, dtype), _levels(Hkv, g, dtype)
        if case["op"] == "append":
            T = case["T"]
            G = 4 if case["fused"] else 0  # query heads in front of the keys
            x = torch.randn(T, (G + 2) * Hkv, D, generator=g, device="cuda")
            x *= torch.exp(0.5 * torch.randn(T, (G + 2) * Hkv, 1, generator=g, device="cuda"))
            x = x.to(dtype)
            if not case["fused"]:
                x = x.view(T, 2, Hkv, D).transpose(0, 1).contiguous()
            s["k"], s["v"] = ((x[:, G * Hkv:(G + 1) * Hkv], x[:, (G + 1) * Hkv:])
                              if case["fused"] else (x[0], x[1]))
            nb = -(-T // bs) + 8
            # whole blocks, scattered over the pool
            order = torch.randperm(nb, generator=g, device="cuda")
            t = torch.arange(T, device="cuda")
            s["slots"] = (order[t // bs] * bs + t % bs).to(torch.int32)
            s["k_codes"], s["v_codes"] = (torch.zeros(nb, Hkv, bs, D // 2, dtype=torch.uint8,
                                                      device="cuda") for _ in range(2))
            s["k_scales"], s["v_scales"] = (torch.zeros(nb, Hkv, bs, dtype=dtype, device="cuda")
                                            for _ in range(2))
        else:
            seq, nq = _lengths(case)
            H = Hkv * case["G"]
            s["tables"], _ = _block_map(seq, bs, 8, g)
            nb = sum(-(-n // bs) for n in seq) + 8
            # every level about equally often, as k-means leaves them
            for name in ("k_codes", "v_codes"):
                s[name] = torch.randint(0, 256, (nb, Hkv, bs, D // 2), generator=g,
                                        dtype=torch.uint8, device="cuda")
            for name, mean in (("k_scales", 2.8), ("v_scales", 1.4)):
                s[name] = (mean * torch.exp(0.2 * torch.randn(nb, Hkv, bs, generator=g,
                                                              device="cuda"))).to(dtype)
            extra = 2 * Hkv if case["fused"] else 0  # the step's own keys and values behind q
            s["q"] = (2.0 * torch.randn(sum(nq), H + extra, D, generator=g,
                                        device="cuda")).to(dtype)[:, :H]
            s["seq"] = _ints(seq)
            s["seq_list"], s["nq_list"] = seq, nq
            s["cu_q"] = None
            if case["q_hi"] > 1:
                s["cu_q"] = _ints([0] + nq).cumsum(0, dtype=torch.int32)
            s["max_seq"] = max(seq)
        if own:
            s["cache"] = _kv4().Cache(*(s[n] for n in (
                "k_codes", "v_codes", "k_scales", "v_scales", "k_levels", "v_levels")))
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        kv4 = _kv4_module()
        if op == "tables":
            slots, cu_new, taken = kv4.block_tables(
                state["seq"], state["new"], state["tables"], state["free"],
                state["case"]["block_size"], state["num_tokens"])
            return {"tables": state["tables"], "slots": slots, "cu_new": cu_new, "taken": taken}
        if op == "append":
            kv4.append(state["cache"], state["k"], state["v"], state["slots"])
            k, v = kv4.read(state["cache"], state["slots"])
            return {"k": k, "v": v}
        r = kv4.attend(state["q"], state["cache"], state["tables"], state["seq"], state["cu_q"],
                       max_seq=state["max_seq"], return_lse=state["case"]["lse"])
        return {"out": r[0], "lse": r[1]} if state["case"]["lse"] else {"out": r}
    return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}[op](state)


_module = None


def _kv4_module():
    global _module
    if _module is None:
        _module = _kv4()
    return _module


# ------------------------------------------------------------ plain forms

def _plain_tables(s):
    bs = s["case"]["block_size"]
    seq, new, free, T = s["seq"], s["new"], s["free"], s["num_tokens"]
    tables, R = s["tables"], seq.numel()
    old = seq - new
    have = (old + bs - 1) // bs
    need = (seq + bs - 1) // bs - have
    end = new.cumsum(0)
    first = need.cumsum(0) - need
    i = torch.arange(T, device=seq.device)
    r = torch.searchsorted(end, i, right=True).clamp_(max=R - 1)
    live = i < end[-1]
    p = old[r] + i - (end - new)[r]
    j = torch.where(live, p // bs, 0)
    fresh = live & (j >= have[r])
    block = torch.where(fresh, free[torch.where(fresh, first[r] + j - have[r], 0)], tables[r, j])
    slots = torch.where(live, block * bs + p % bs, -1).to(torch.int32)
    # every token of a block writes the same entry, padding the spare column
    grown = torch.cat([tables, tables[:, :1]], 1)
    grown[r, torch.where(live, j, tables.shape[1])] = block
    tables = grown[:, :-1].contiguous()
    cu = torch.cat([end.new_zeros(1), end]).to(torch.int32)
    return {"tables": tables, "slots": slots, "cu_new": cu,
            "taken": need.sum().view(1).to(torch.int32)}


def _unpack(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()


def _values(codes, scales, levels):
    """fp32 values (n, Hkv, D) of packed codes (n, Hkv, D/2)."""
    Hkv = levels.shape[0]
    base = LEVELS * torch.arange(Hkv, device=codes.device)[:, None]
    return levels.float().flatten()[_unpack(codes) + base] * scales.float()[..., None]


def _plain_append(s):
    bs = s["case"]["block_size"]
    slots = s["slots"].long()
    blk, off = slots // bs, slots % bs
    out = {}
    for n in ("k", "v"):
        x = s[n].float()
        levels = s[n + "_levels"].float()
        scale = x.abs().amax(-1)
        scale = torch.where(scale < MIN_SCALE, 0.0, scale)
        inv = torch.where(scale > 0, 1.0 / scale, 0.0)
        y = x * inv[..., None]
        best = (y - levels[:, 0, None]).abs()
        code = torch.zeros_like(y, dtype=torch.uint8)
        for c in range(1, LEVELS):
            d = (y - levels[:, c, None]).abs()
            code = torch.where(d < best, c, code)
            best = torch.minimum(best, d)
        s[n + "_codes"][blk, :, off] = code[..., 0::2] | (code[..., 1::2] << 4)
        s[n + "_scales"][blk, :, off] = scale.to(s[n].dtype)
        out[n] = _values(s[n + "_codes"][blk, :, off], s[n + "_scales"][blk, :, off],
                         s[n + "_levels"]).to(s[n].dtype)
    return out


def _plain_attend(s):
    case = s["case"]
    bs, D, Hkv, G = case["block_size"], case["D"], case["Hkv"], case["G"]
    dev, dtype = s["q"].device, s["q"].dtype
    T = s["q"].shape[0]
    out = torch.zeros(T, Hkv * G, D, dtype=dtype, device=dev)
    lse = torch.full((T, Hkv * G), -math.inf, device=dev)
    row = 0
    for r, (n, nq) in enumerate(zip(s["seq_list"], s["nq_list"])):
        if n and nq:
            t = torch.arange(n, device=dev)
            blk, off = s["tables"][r, t // bs].long(), t % bs
            k, v = (_values(s[x + "_codes"][blk, :, off], s[x + "_scales"][blk, :, off],
                            s[x + "_levels"]).transpose(0, 1).contiguous() for x in ("k", "v"))
            kt = k.transpose(1, 2).contiguous()
            step = max(1, (1 << 29) // (Hkv * G * n))
            for a in range(0, nq, step):
                b = min(nq, a + step)
                q = s["q"][row + a:row + b].float().view(b - a, Hkv, G, D).transpose(0, 1)
                sc = (q.reshape(Hkv, (b - a) * G, D) @ kt) * D ** -0.5
                pos = n - nq + torch.arange(a, b, device=dev).repeat_interleave(G)
                sc = sc.masked_fill(t > pos[:, None], -math.inf)
                m = sc.amax(-1, keepdim=True)
                p = torch.exp(sc - m)
                z = p.sum(-1, keepdim=True)
                o = (p @ v) / z
                out[row + a:row + b] = o.view(Hkv, b - a, G, D).transpose(0, 1).reshape(
                    b - a, Hkv * G, D).to(dtype)
                lse[row + a:row + b] = (m + z.log()).view(Hkv, b - a, G).transpose(0, 1).reshape(
                    b - a, Hkv * G)
        row += nq
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


# ------------------------------------------------------------ 64 bits

def exact(case, seed):
    """The operators from their definitions, in 64 bits.  Block numbers and
    slots by walking the requests; the stored levels by the definition's
    32-bit quotients and distances (a choice, not a computed number), the
    values they stand for in 64."""
    if case["op"] == "attend" and work(case)["flops"] > 4e12:
        return None
    if case["op"] == "append" and case["T"] * case["Hkv"] * case["D"] > 1 << 26:
        return None
    if case["op"] == "tables":
        if sum(_lengths(case)[1]) > 1 << 20:
            return None
        return _exact_tables(case, seed)
    return (_exact_append if case["op"] == "append" else _exact_attend)(case, seed)


def _exact_tables(case, seed):
    s = prepare(case, seed)
    bs = case["block_size"]
    seq, new = _lengths(case)
    tables = s["tables"].cpu().numpy().copy()
    free = s["free"].cpu().numpy()
    slots = np.full(s["num_tokens"], -1, np.int32)
    at, taken, cu = 0, 0, [0]
    for r, (n, fresh) in enumerate(zip(seq, new)):
        held = n - fresh
        for j in range(-(-held // bs), -(-n // bs)):
            tables[r, j] = free[taken]
            taken += 1
        pos = np.arange(held, n)
        slots[at:at + fresh] = tables[r, pos // bs] * bs + pos % bs
        at += fresh
        cu.append(at)
    return {"tables": torch.from_numpy(tables), "slots": torch.from_numpy(slots),
            "cu_new": torch.tensor(cu, dtype=torch.int32),
            "taken": torch.tensor([taken], dtype=torch.int32)}


def _exact_append(case, seed):
    s = prepare(case, seed)
    out = {}
    for n in ("k", "v"):
        x = s[n].float().cpu().numpy()
        levels = s[n + "_levels"].float().cpu().numpy()
        scale = np.abs(x).max(-1, keepdims=True)
        scale[scale < np.float32(MIN_SCALE)] = 0
        inv = np.divide(np.float32(1), scale, out=np.zeros_like(scale), where=scale > 0)
        y = x * inv
        held = np.empty(x.shape, np.float64)
        for h in range(x.shape[1]):
            dist = np.abs(y[:, h, :, None] - levels[h]) if y.shape[0] <= 4096 else None
            if dist is not None:
                held[:, h] = levels[h][dist.argmin(-1)]
            else:
                for a in range(0, y.shape[0], 4096):
                    d = np.abs(y[a:a + 4096, h, :, None] - levels[h])
                    held[a:a + 4096, h] = levels[h][d.argmin(-1)]
        out[n] = torch.from_numpy(held * scale.astype(np.float64))
    return out


def _exact_attend(case, seed):
    s = prepare(case, seed)
    bs, D, G = case["block_size"], case["D"], case["G"]
    T, H = s["q"].shape[0], s["q"].shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device="cuda")
    row = 0
    for r, (n, nq) in enumerate(zip(s["seq_list"], s["nq_list"])):
        if n == 0 or nq == 0:
            row += nq
            continue
        slot = torch.tensor([int(b) * bs for b in s["tables"][r].tolist()], device="cuda")
        slot = (slot[:, None] + torch.arange(bs, device="cuda")).flatten()[:n]
        hidden = (torch.arange(n, device="cuda")[None, :]
                  - torch.arange(nq, device="cuda")[:, None]) > n - nq
        for h in range(H):
            kv = []
            for x in ("k", "v"):
                byte = s[x + "_codes"][:, h // G].reshape(-1, D // 2)[slot].int()
                lv = s[x + "_levels"][h // G].double()
                val = torch.empty(n, D, dtype=torch.float64, device="cuda")
                val[:, 0::2], val[:, 1::2] = lv[byte % 16], lv[byte // 16]
                kv.append(val * s[x + "_scales"][:, h // G].reshape(-1)[slot].double()[:, None])
            z = s["q"][row:row + nq, h].double() @ kv[0].t().contiguous() / math.sqrt(D)
            z[hidden] = -math.inf
            top = torch.logsumexp(z, 1)
            lse[row:row + nq, h] = top
            out[row:row + nq, h] = torch.exp(z - top[:, None]) @ kv[1]
        row += nq
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
