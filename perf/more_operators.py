"""More operators around the key/value cache held in 4 bits, case by case.

Two kinds of work beside the plain serving step:

* "attend": one `kv4.attend` call whose scores are capped (cap * tanh(z / cap)),
  lowered with the distance between query and key, or masked: a window of the
  last tokens, documents packed into one request, a prefix that every query
  sees.  Single tokens, drafts and prompts.
* pages of the cache: "fork" (rows that go on from others' tokens, sharing
  their whole blocks), "free" (the blocks that no row holds), "compact" (the
  held blocks moved into another cache) and "copy" (blocks named one by one).

`own` chooses between the package's kernels and the same formulas in plain
torch operations.  Lengths, documents, prefixes and parents are drawn from the
case's own `lens` seed, so that the work of a case is known without a GPU;
everything else from `seed`.
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
TENSORS = ("k_codes", "v_codes", "k_scales", "v_scales")

_module = None


def _kv4():
    global _module
    if _module is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "flash-kmeans-cuda_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from flash_kmeans_cuda import kv4
        _module = kv4
    return _module


def _named(name, c):
    return c if name is None else {"name": name, **c}


def _attend(name, dtype, R, seq, q, Hkv, G, D, block_size, lens, cap=0.0, slopes=False, window=0,
            docs=0, prefix=False, idle=0, lse=False):
    return _named(name, {
        "op": "attend", "dtype": dtype, "R": R, "seq_lo": seq[0], "seq_hi": seq[1], "q_lo": q[0],
        "q_hi": q[1], "Hkv": Hkv, "G": G, "D": D, "block_size": block_size, "lens": lens,
        "cap": cap, "slopes": slopes, "window": window, "docs": docs, "prefix": prefix,
        "idle": idle, "lse": lse})


def _pages(name, op, dtype, R, seq, Hkv, D, block_size, lens, spare=64, group=1, children=0):
    """group: rows that go on from the same tokens and share their whole blocks
    (with different lengths behind them); children: rows after a fork."""
    return _named(name, {
        "op": op, "dtype": dtype, "R": R, "seq_lo": seq[0], "seq_hi": seq[1], "Hkv": Hkv, "D": D,
        "block_size": block_size, "lens": lens, "spare": spare, "group": group,
        "children": children})


def listed():
    return [
        # The smallest answer: one new token over a short context, capped scores.
        _attend("decode_one_capped", "bf16", 1, (777, 777), (1, 1), 8, 4, 128, 16, 1, cap=50.0),
        # An ordinary decoding batch of a layer that looks back over a window,
        # wide heads, some rows idle: most contexts are longer than the window.
        _attend("decode_window", "bf16", 64, (1024, 32768), (1, 1), 8, 2, 256, 64, 2, cap=50.0,
                window=4096, idle=3),
        # A few drafted tokens per request over long contexts, scores lowered
        # with the distance; the statistics are kept for joining.
        _attend("drafts_distance", "f16", 24, (300, 65536), (2, 7), 4, 8, 128, 32, 3, slopes=True,
                lse=True),
        # Ragged prompts from the first token on, capped scores, every token.
        _attend("prompt_capped", "bf16", 4, (900, 6000), (900, 6000), 8, 4, 128, 64, 15, cap=30.0),
        # Two long prompts, each many documents that do not see one another.
        _attend("prompt_documents", "f16", 2, (9000, 16000), (9000, 16000), 16, 1, 64, 64, 5,
                docs=700),
        # Prompts whose first part every token sees, wide heads, distances.
        _attend("prompt_prefix", "bf16", 3, (2000, 5000), (2000, 5000), 2, 8, 256, 48, 6,
                slopes=True, prefix=True, lse=True),
        # Several samples from each of a few prompts.
        _pages("fork_samples", "fork", "bf16", 8, (500, 4000), 8, 128, 64, 7, children=64),
        # A step of a beam search: beams of a group go on from one another.
        _pages("fork_beams", "fork", "f16", 512, (100, 3000), 4, 128, 16, 8, group=4,
               spare=1024, children=512),
        # The free list of a small server, a step like any other.
        _pages("free_small", "free", "bf16", 64, (1, 8192), 1, 64, 64, 9, spare=1500),
        # That of a large pool of small blocks, with shared beginnings.
        _pages("free_large", "free", "bf16", 2048, (1, 16384), 1, 64, 16, 10, spare=100000,
               group=3),
        # Moving a server's requests into a smaller cache.
        _pages("compact_pool", "compact", "bf16", 96, (1024, 16384), 8, 128, 64, 11, spare=3000,
               group=2),
        # One request's blocks handed to another cache.
        _pages("copy_request", "copy", "f16", 1, (30001, 30001), 8, 128, 64, 12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    lens = rng.randrange(1 << 30)
    op = rng.choice(["attend", "attend", "attend", "fork", "free", "compact", "copy"])
    dtype = rng.choice(["f16", "bf16"])
    bs = rng.choice([16, 32, 48, 64, 128])
    Hkv = rng.choice([1, 2, 4, 5, 8, 16])
    D = rng.choice([64, 128, 128, 256])
    if op != "attend":
        if op == "free":
            Hkv, D = 1, 64  # the tables alone are read
        hi = _log_int(rng, 1, 32768)
        # what the cache holds: 448 MiB at most, and 2^21 blocks
        most = min((7 << 26) // (Hkv * (D + 4) * (hi + bs)), (1 << 21) // (hi // bs + 1))
        R = _log_int(rng, 1, max(1, min(2048, most)))
        lo = 1 if rng.random() < 0.5 else hi
        group = rng.choice([1, 1, 2, 4])
        children = _log_int(rng, 1, 2048) if op == "fork" else 0
        return _pages(None, op, dtype, R, (lo, hi), Hkv, D, bs, lens, group=group,
                      spare=children + _log_int(rng, 1, 4096), children=children)
    G = rng.choice([1, 2, 3, 4, 7, 8, 16])
    cap = rng.choice([0.0, 20.0, 30.0, 50.0])
    slopes = rng.random() < 0.3
    window = _log_int(rng, 1, 8192) if rng.random() < 0.4 else 0
    docs = _log_int(rng, 16, 4096) if rng.random() < 0.3 else 0
    kind = rng.choice(["decode", "drafts", "prompt"])
    prefix = kind != "decode" and rng.random() < 0.3
    idle = 0
    if kind == "prompt":
        # Pairs of a query and a key it may see, over all heads and columns.
        budget = 1 << 36
        hi = _log_int(rng, 1, 8192)
        R = max(1, min(8, budget // (Hkv * G * D * hi * hi)))
        hi = max(1, min(hi, math.isqrt(budget // (R * Hkv * G * D))))
        pre = _log_int(rng, 1, 8192) if rng.random() < 0.5 else 0
        pre = min(pre, max(0, budget // (R * Hkv * G * D * hi) - hi))
        seq, q = (pre + 1, pre + hi), (1, hi)
    else:
        hi = _log_int(rng, 1, 131072)
        R = _log_int(rng, 1, max(1, min(256, (1 << 29) // (Hkv * D * hi))))
        hi = max(1, min(hi, (1 << 29) // (Hkv * D * R)))
        seq = (1 if rng.random() < 0.5 else hi, hi)
        q = (1, 1) if kind == "decode" else (1, rng.randrange(2, 9))
        idle = rng.choice([0, 0, 1]) if R > 1 else 0
    return _attend(None, dtype, R, seq, q, Hkv, G, D, bs, lens, cap=cap, slopes=slopes,
                   window=window, docs=docs, prefix=prefix, idle=idle, lse=rng.random() < 0.3)


# ------------------------------------------------------------ what a case is

def _queries(case):
    """(tokens, queries, prefixes) per request and each query row's first
    token by its document."""
    rng = random.Random(case["lens"])
    seq, nq, prefix, starts = [], [], [], []
    whole = case["q_lo"] == case["seq_lo"] and case["q_hi"] == case["seq_hi"]
    for r in range(case["R"]):
        s = _log_int(rng, case["seq_lo"], case["seq_hi"])
        # a prompt from its first token on has as many queries as tokens
        n = s if whole and case["q_hi"] > 1 else min(s, _log_int(rng, case["q_lo"], case["q_hi"]))
        if r < case["idle"]:
            # a decoding batch keeps its idle rows
            s, n = 0, (1 if case["q_hi"] == 1 else 0)
        seq.append(s)
        nq.append(n)
        prefix.append(int(s * rng.uniform(0.2, 0.9)) if case["prefix"] else 0)
        first = np.zeros(max(s, n), np.int64)
        if case["docs"]:
            at = 0
            while at < s:
                end = at + _log_int(rng, max(1, case["docs"] // 4), 2 * case["docs"])
                first[at:end] = at
                at = end
        starts.append(first[len(first) - n:])
    return seq, nq, prefix, starts


def _seen(case, n, m, prefix, starts):
    """The tokens [first, last) that each of a request's m queries sees."""
    p = np.arange(n - m, n)
    last = np.minimum(np.maximum(p + 1, prefix), n)
    first = np.maximum(starts, p - case["window"] + 1 if case["window"] else 0)
    return first, last


def _rows(case):
    """Tokens per row, and the row whose whole blocks it shares (or itself),
    up to which token."""
    rng = random.Random(case["lens"])
    seq, of, upto = [], [], []
    for r in range(case["R"]):
        seq.append(_log_int(rng, case["seq_lo"], case["seq_hi"]))
        lead = r - r % case["group"]
        of.append(lead)
        bs = case["block_size"]
        upto.append(0 if lead == r else
                    int(min(seq[r], seq[lead]) * rng.uniform(0, 1)) // bs * bs)
    return seq, of, upto


def _parents(case):
    """The row that each child goes on from: of its group, in no order."""
    rng = random.Random(case["lens"] + 1)
    g, F = max(case["group"], 1), case["children"]
    got = []
    for j in range(F):
        lead = j * case["R"] // F // g * g
        got.append(min(lead + rng.randrange(g), case["R"] - 1))
    return got


def _blocks(case):
    """(entries of each row as numbers from 0 on, how many there are)."""
    seq, of, upto = _rows(case)
    bs, rows, at = case["block_size"], [], 0
    for s, o, u in zip(seq, of, upto):
        own_blocks = -(-s // bs) - u // bs
        rows.append(np.concatenate([rows[o][:u // bs], np.arange(at, at + own_blocks)])
                    if u else np.arange(at, at + own_blocks))
        at += own_blocks
    return seq, rows, at


def _fork_copies(case, seq, rows):
    """Children whose last block has to be copied."""
    bs, parents = case["block_size"], _parents(case)
    whole = set()
    for p in set(parents):
        whole.update(rows[p][:seq[p] // bs].tolist())
    first, copies = set(whole), []
    for j, p in enumerate(parents):
        if seq[p] % bs:
            b = int(rows[p][-1])
            if b in first:
                copies.append(j)
            first.add(b)
    return copies


def work(case):
    bs, D, Hkv = case["block_size"], case["D"], case["Hkv"]
    if case["op"] == "attend":
        H = Hkv * case["G"]
        pairs = tokens = blocks = 0
        seq, nq, prefix, starts = _queries(case)
        for n, m, f, st in zip(seq, nq, prefix, starts):
            first, last = _seen(case, n, m, f, st)
            ok = last > first
            pairs += int((last - first)[ok].sum())
            edge = np.zeros(n + 1, np.int64)
            np.add.at(edge, first[ok], 1)
            np.add.at(edge, last[ok], -1)
            some = np.cumsum(edge)[:n] > 0
            tokens += int(some.sum())
            blocks += len(set((np.flatnonzero(some) // bs).tolist()))
        rows = sum(nq)
        small = 4 * (2 * case["R"] + blocks + (rows if case["docs"] else 0))
        return {"bytes": tokens * Hkv * (D + 4) + rows * H * (4 * D + (4 if case["lse"] else 0))
                + small, "flops": 4 * D * H * pairs}
    seq, rows, held = _blocks(case)
    entries = sum(len(r) for r in rows)
    block = bs * Hkv * (D + 4)
    if case["op"] == "free":
        return {"bytes": 4 * (case["R"] + entries + held + case["spare"] + 1), "flops": 0}
    if case["op"] == "copy":
        return {"bytes": 2 * held * block + 8 * held, "flops": 0}
    if case["op"] == "compact":
        width = max(len(r) for r in rows)
        return {"bytes": 2 * held * block + 4 * (entries + case["R"] * (width + 1) + 1),
                "flops": 0}
    width = max(len(r) for r in rows)
    parents, copies = _parents(case), _fork_copies(case, seq, rows)
    used = sum(len(rows[p]) for p in set(parents))
    # of a block that is not full the tokens in it
    moved = sum(seq[parents[j]] % bs for j in copies) * Hkv * (D + 4)
    return {"bytes": 2 * moved + 4 * (used + len(copies) + len(parents) * (width + 2) + 1),
            "flops": 0}


# ------------------------------------------------------------ inputs

def _ints(v, dev="cuda"):
    return torch.as_tensor(np.asarray(v, dtype=np.int32)).to(dev)


def _table(rows, number, width):
    """Rows of block numbers, -1 behind them."""
    t = np.full((len(rows), max(width, 1)), -1, np.int64)
    for r, b in enumerate(rows):
        t[r, :len(b)] = b
    t = torch.from_numpy(t).cuda()
    return torch.where(t >= 0, number[t.clamp(min=0)], -1).to(torch.int32)


def _levels(Hkv, g, dtype):
    """Sixteen levels per head near the quantiles of a normal column over its
    vector's largest magnitude, in no particular order."""
    p = (torch.arange(LEVELS, device="cuda") + 0.5) / LEVELS
    lv = torch.erfinv(2 * p - 1) * 0.5
    lv = lv * (1 + 0.1 * torch.rand(Hkv, 1, generator=g, device="cuda"))
    lv = lv + 0.01 * torch.randn(Hkv, LEVELS, generator=g, device="cuda")
    order = torch.rand(Hkv, LEVELS, generator=g, device="cuda").argsort(1)
    return lv.gather(1, order).to(dtype)


def _fill(s, case, nb, g):
    """A cache of nb blocks: every level about equally often, as k-means
    leaves them, and scales as vectors of normal columns have."""
    dtype, Hkv, D, bs = DTYPES[case["dtype"]], case["Hkv"], case["D"], case["block_size"]
    s["k_levels"], s["v_levels"] = _levels(Hkv, g, dtype), _levels(Hkv, g, dtype)
    for name in ("k_codes", "v_codes"):
        s[name] = torch.randint(0, 256, (nb, Hkv, bs, D // 2), generator=g, dtype=torch.uint8,
                                device="cuda")
    for name, mean in (("k_scales", 2.8), ("v_scales", 1.4)):
        s[name] = (mean * torch.exp(0.2 * torch.randn(nb, Hkv, bs, generator=g,
                                                      device="cuda"))).to(dtype)


def _slopes(H):
    return torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda") / H).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s, bs = {"case": case}, case["block_size"]
    if case["op"] == "attend":
        seq, nq, prefix, starts = _queries(case)
        H, D, dtype = case["Hkv"] * case["G"], case["D"], DTYPES[case["dtype"]]
        n = [-(-x // bs) for x in seq]
        nb = sum(n) + 8
        _fill(s, case, nb, g)
        first = np.cumsum([0] + n)
        s["tables"] = _table([np.arange(a, a + b) for a, b in zip(first, n)],
                             torch.randperm(nb, generator=g, device="cuda"), max(n))
        # capped scores are the larger ones: a cap changes what they give
        s["q"] = ((6.0 if case["cap"] else 2.0) * torch.randn(
            sum(nq), H, D, generator=g, device="cuda")).to(dtype)
        s["seq"], s["seq_list"], s["nq_list"] = _ints(seq), seq, nq
        s["cu_q"] = _ints(np.cumsum([0] + nq)) if case["q_hi"] > 1 else None
        s["max_seq"] = max(seq)
        s["slopes"] = _slopes(H) if case["slopes"] else None
        s["starts"] = _ints(np.concatenate(starts)) if case["docs"] else None
        s["prefix"], s["prefix_list"] = (_ints(prefix) if case["prefix"] else None), prefix
    else:
        seq, rows, held = _blocks(case)
        nb = held + case["spare"]
        number = torch.randperm(nb, generator=g, device="cuda")
        s["num_blocks"] = nb
        if case["op"] != "free":
            _fill(s, case, nb, g)
        if case["op"] == "copy":
            s["src"] = number[:held].to(torch.int32)
            s["dst"] = torch.randperm(held + 8, generator=g, device="cuda")[:held].to(torch.int32)
        else:
            s["tables"] = _table(rows, number, max(len(r) for r in rows))
            s["seq"] = _ints(seq)
        if case["op"] == "fork":
            s["parents"] = _ints(_parents(case))
            # (a free list may be shorter than what is asked of it, but this one is not)
            s["free"] = number[held:].to(torch.int32)
        if case["op"] in ("copy", "compact"):
            s["into"] = {n: torch.zeros((held + 8, *s[n].shape[1:]), dtype=s[n].dtype,
                                        device="cuda") for n in TENSORS}
    if own and "k_codes" in s:
        levels = s["k_levels"], s["v_levels"]
        s["cache"] = _kv4().Cache(*(s[n] for n in TENSORS), *levels)
        if "into" in s:
            s["into_cache"] = _kv4().Cache(*(s["into"][n] for n in TENSORS), *levels)
    return s


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        return {"attend": _plain_attend, "fork": _plain_fork, "free": _plain_free,
                "compact": _plain_compact, "copy": _plain_copy}[op](s)
    kv4 = _kv4()
    if op == "attend":
        r = kv4.attend(s["q"], s["cache"], s["tables"], s["seq"], s["cu_q"],
                       max_seq=s["max_seq"], return_lse=case["lse"],
                       softcap=case["cap"] or None, slopes=s["slopes"],
                       window=case["window"] or None, starts=s["starts"],
                       prefix_lens=s["prefix"])
        return {"out": r[0], "lse": r[1]} if case["lse"] else {"out": r}
    if op == "fork":
        tables, seq, taken = kv4.fork(s["cache"], s["tables"], s["seq"], s["parents"], s["free"])
        return {"tables": tables, "seq": seq, "taken": taken, **_held(s)}
    if op == "free":
        free, count = kv4.free_blocks(s["tables"], s["seq"], case["block_size"], s["num_blocks"])
        return {"free": free, "count": count}
    if op == "compact":
        tables, used = kv4.compact(s["cache"], s["tables"], s["seq"], s["into_cache"])
        return {"tables": tables, "used": used, **_held(s["into"])}
    kv4.copy_blocks(s["cache"], s["src"], s["into_cache"], s["dst"])
    return _held(s["into"])


def _held(s):
    """What the pages hold: bytes that were copied have to be equal, so they
    are given as they are."""
    return {n: s[n] for n in TENSORS}


# ------------------------------------------------------------ plain forms

def _values(codes, scales, levels):
    """fp32 values (n, Hkv, D) of packed codes (n, Hkv, D/2)."""
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    base = LEVELS * torch.arange(levels.shape[0], device=codes.device)[:, None]
    return levels.float().flatten()[both + base] * scales.float()[..., None]


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
            step = max(1, (1 << 28) // (Hkv * G * n))
            for a in range(0, nq, step):
                b = min(nq, a + step)
                rows = slice(row + a, row + b)
                q = s["q"][rows].float().view(b - a, Hkv, G, D).transpose(0, 1)
                z = (q.reshape(Hkv, (b - a) * G, D) @ kt) * D ** -0.5
                if case["cap"]:
                    z = torch.tanh(z / case["cap"]) * case["cap"]
                p = n - nq + torch.arange(a, b, device=dev)
                if case["slopes"]:
                    away = (p[:, None] - t).abs().float()
                    z = z.view(Hkv, b - a, G, n) - (s["slopes"].view(Hkv, 1, G, 1)
                                                    * away[:, None, :])
                    z = z.view(Hkv, (b - a) * G, n)
                seen = (t <= p[:, None]) | (t < s["prefix_list"][r])
                if case["window"]:
                    seen &= t > p[:, None] - case["window"]
                if case["docs"]:
                    seen &= t >= s["starts"][rows, None]
                z = z.masked_fill(~seen.repeat_interleave(G, 0), -math.inf)
                m = z.amax(-1, keepdim=True)
                some = m > -math.inf
                e = torch.exp(z - torch.where(some, m, 0.0))
                total = e.sum(-1, keepdim=True)
                o = (e @ v) / torch.where(some, total, 1.0)
                out[rows] = o.view(Hkv, b - a, G, D).transpose(0, 1).reshape(
                    b - a, Hkv * G, D).to(dtype)
                lse[rows] = (m + total.log()).view(Hkv, b - a, G).transpose(0, 1).reshape(
                    b - a, Hkv * G)
        row += nq
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _in_rows(s, tables, seq):
    """Which entries of the tables are held, and how many there are a row."""
    n = (seq + s["case"]["block_size"] - 1) // s["case"]["block_size"]
    return torch.arange(tables.shape[1], device=tables.device) < n[:, None], n


def _plain_fork(s):
    bs, nb = s["case"]["block_size"], s["num_blocks"]
    parents = s["parents"].long()
    F = parents.numel()
    tables, seq = s["tables"][parents], s["seq"][parents]
    held, n = _in_rows(s, tables, seq)
    tables = torch.where(held, tables, -1)
    part = seq % bs > 0
    at = (n - 1).clamp(min=0).long()
    last = tables.gather(1, at[:, None])[:, 0].long()
    whole = torch.arange(tables.shape[1], device=tables.device) < (seq // bs)[:, None]
    j = torch.arange(F, device=tables.device)
    first = torch.full((nb + 1,), F, device=tables.device)
    first.scatter_reduce_(0, torch.where(part, last, nb), j, "amin")
    first[torch.where(whole, tables, nb).flatten().long()] = -1
    copy = part & (first[last.clamp(min=0)] != j)
    order = copy.cumsum(0)
    fresh = s["free"][torch.where(copy, order - 1, 0)].long()
    source = torch.where(part, last, 0)
    target = torch.where(copy, fresh, source)
    for name in TENSORS:
        s[name][target] = s[name][source]
    tables.scatter_(1, at[:, None], torch.where(part, target, tables.gather(
        1, at[:, None])[:, 0].long())[:, None].to(torch.int32))
    return {"tables": tables, "seq": seq, "taken": order[-1:].to(torch.int32), **_held(s)}


def _named_blocks(s):
    """Which blocks some row holds."""
    held, _ = _in_rows(s, s["tables"], s["seq"])
    named = torch.zeros(s["num_blocks"] + 1, dtype=torch.bool, device=held.device)
    named[torch.where(held, s["tables"], s["num_blocks"]).flatten().long()] = True
    return named[:-1], held


def _plain_free(s):
    named, _ = _named_blocks(s)
    place = torch.where(named, s["num_blocks"], (~named).cumsum(0) - 1)
    free = torch.full((s["num_blocks"] + 1,), -1, dtype=torch.int32, device=named.device)
    free[place] = torch.arange(s["num_blocks"], dtype=torch.int32, device=named.device)
    return {"free": free[:-1].contiguous(), "count": (~named).sum().view(1).to(torch.int32)}


def _plain_compact(s):
    named, held = _named_blocks(s)
    number = named.cumsum(0) - 1
    tables = torch.where(held, number[s["tables"].clamp(min=0).long()], -1).to(torch.int32)
    source = named.nonzero()[:, 0]
    for name in TENSORS:
        s["into"][name][:source.numel()] = s[name][source]
    return {"tables": tables, "used": named.sum().view(1).to(torch.int32), **_held(s["into"])}


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for name in TENSORS:
        s["into"][name][dst] = s[name][src]
    return _held(s["into"])


# ------------------------------------------------------------ 64 bits

def exact(case, seed):
    """The operators from their definitions: attention head by head in 64 bits,
    pages by walking the rows."""
    if case["op"] == "attend":
        seq, nq, _, _ = _queries(case)
        if sum(n * m for n, m in zip(seq, nq)) * case["Hkv"] * case["G"] * case["D"] > 2e12:
            return None
        return _exact_attend(case, seed)
    if case["op"] != "free" and _blocks(case)[2] * case["block_size"] * case["Hkv"] * (
            case["D"] + 4) > 1 << 28:
        return None
    if sum(len(r) for r in _blocks(case)[1]) > 1 << 20:
        return None
    return _exact_pages(case, seed)


def _exact_attend(case, seed):
    s = prepare(case, seed)
    seq, nq, prefix, starts = _queries(case)
    bs, D, G = case["block_size"], case["D"], case["G"]
    T, H = s["q"].shape[0], s["q"].shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device="cuda")
    row = 0
    for r, (n, m) in enumerate(zip(seq, nq)):
        if n == 0 or m == 0:
            row += m
            continue
        slot = torch.tensor([int(b) * bs for b in s["tables"][r].tolist()], device="cuda")
        slot = (slot[:, None] + torch.arange(bs, device="cuda")).flatten()[:n]
        first, last = _seen(case, n, m, prefix[r], starts[r])
        # a row that sees nothing keeps its 0 and -inf
        rows = torch.from_numpy(np.flatnonzero(last > first)).cuda()
        if rows.numel() == 0:
            row += m
            continue
        lo = torch.from_numpy(first).cuda()[rows, None]
        hi = torch.from_numpy(last).cuda()[rows, None]
        token = torch.arange(n, device="cuda")
        hidden = (token < lo) | (token >= hi)
        apart = (token - (rows[:, None] + (n - m))).abs().double()
        for h in range(H):
            kv = []
            for x in ("k", "v"):
                byte = s[x + "_codes"][:, h // G].reshape(-1, D // 2)[slot].int()
                lv = s[x + "_levels"][h // G].double()
                val = torch.empty(n, D, dtype=torch.float64, device="cuda")
                val[:, 0::2], val[:, 1::2] = lv[byte % 16], lv[byte // 16]
                kv.append(val * s[x + "_scales"][:, h // G].reshape(-1)[slot].double()[:, None])
            z = s["q"][row:row + m, h].double()[rows] @ kv[0].t().contiguous() / math.sqrt(D)
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            if case["slopes"]:
                z -= s["slopes"][h].double() * apart
            z[hidden] = -math.inf
            top = torch.logsumexp(z, 1)
            lse[row + rows, h] = top
            out[row + rows, h] = torch.exp(z - top[:, None]) @ kv[1]
        row += m
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _exact_pages(case, seed):
    s = prepare(case, seed)
    bs = case["block_size"]
    if case["op"] == "copy":
        src, dst = s["src"].tolist(), s["dst"].tolist()
        got = {n: s["into"][n].cpu() for n in TENSORS}
        for n in TENSORS:
            have = s[n].cpu()
            for a, b in zip(src, dst):
                got[n][b] = have[a]
        return got
    seq, rows = _blocks(case)[:2]
    tables = s["tables"].cpu().numpy()
    mine = [tables[r, :len(b)].tolist() for r, b in enumerate(rows)]
    if case["op"] != "fork":
        held = sorted({b for r in mine for b in r})
    if case["op"] == "free":
        out = np.full(s["num_blocks"], -1, np.int32)
        unused = sorted(set(range(s["num_blocks"])) - set(held))
        out[:len(unused)] = unused
        return {"free": torch.from_numpy(out),
                "count": torch.tensor([len(unused)], dtype=torch.int32)}
    if case["op"] == "compact":
        number = {b: i for i, b in enumerate(held)}
        new = np.full_like(tables, -1)
        for r, b in enumerate(mine):
            new[r, :len(b)] = [number[x] for x in b]
        got = {n: s["into"][n].cpu() for n in TENSORS}
        for n in TENSORS:
            got[n][:len(held)] = s[n].cpu()[held]
        return {"tables": torch.from_numpy(new),
                "used": torch.tensor([len(held)], dtype=torch.int32), **got}
    parents, free = _parents(case), s["free"].tolist()
    copies = set(_fork_copies(case, seq, rows))
    new = np.full((len(parents), tables.shape[1]), -1, np.int32)
    got, taken = {n: s[n].cpu() for n in TENSORS}, 0
    for j, p in enumerate(parents):
        new[j, :len(mine[p])] = mine[p]
        if j in copies:
            for n in TENSORS:
                got[n][free[taken]] = got[n][mine[p][-1]]
            new[j, len(mine[p]) - 1] = free[taken]
            taken += 1
    return {"tables": torch.from_numpy(new), "seq": torch.tensor(
        [seq[p] for p in parents], dtype=torch.int32),
        "taken": torch.tensor([taken], dtype=torch.int32), **got}
