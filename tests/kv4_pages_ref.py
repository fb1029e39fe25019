"""Plain references of the 4-bit cache's page operators, on the CPU: by walking
the rows."""

from __future__ import annotations

import numpy as np


def held(tables, seq, bs, num_blocks):
    """Per row the entries it holds, None for those that name no block."""
    rows = []
    for t, n in zip(tables, seq):
        n = min(-(-max(int(n), 0) // bs), len(t))
        rows.append([int(b) if 0 <= b < num_blocks else None for b in t[:n]])
    return rows


def free_blocks(tables, seq, bs, num_blocks):
    used = {b for row in held(tables, seq, bs, num_blocks) for b in row}
    free = [b for b in range(num_blocks) if b not in used]
    return np.array(free + [-1] * (num_blocks - len(free)), np.int32), len(free)


def fork(tables, seq, parents, free, bs, num_blocks):
    """(tables, lengths, taken, copies as (block, its copy))."""
    rows = held(tables, seq, bs, num_blocks)
    width = tables.shape[1]
    new = np.full((len(parents), width), -1, np.int32)
    out_seq, ends, whole = [], [], set()
    for j, p in enumerate(parents):
        ok = 0 <= p < len(rows)
        n = max(int(seq[p]), 0) if ok else 0
        out_seq.append(n)
        row = rows[p] if ok else []
        new[j, :len(row)] = [-1 if b is None else b for b in row]
        full = min(n // bs, width)
        whole.update(row[:full])
        ends.append(row[full] if n % bs and full < len(row) else None)
    taken, copies, owned = 0, [], set(whole)
    for j, b in enumerate(ends):
        if b is None:
            continue
        if b in owned:
            f = free[taken] if taken < len(free) else -1
            f = int(f) if 0 <= f < num_blocks else -1
            new[j, out_seq[j] // bs] = f
            if f >= 0:
                copies.append((b, f))
            taken += 1
        owned.add(b)
    return new, np.array(out_seq, np.int32), taken, copies


def compact(tables, seq, bs, num_blocks, into_blocks):
    """(tables, held blocks in order)."""
    rows = held(tables, seq, bs, num_blocks)
    used = sorted({b for row in rows for b in row if b is not None})
    number = {b: i if i < into_blocks else -1 for i, b in enumerate(used)}
    new = np.full(tables.shape, -1, np.int32)
    for r, row in enumerate(rows):
        new[r, :len(row)] = [-1 if b is None else number[b] for b in row]
    return new, used
