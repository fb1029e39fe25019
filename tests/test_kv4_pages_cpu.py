"""The page operators of the 4-bit cache refuse what their kernels could not
index, before anything reaches a device; and their reference is itself checked
against counts."""

from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest

import kv4_pages_ref as pages
from test_kv4_cpu import FAKE, _cache


def _call(fn, ok, at, value):
    from flash_kmeans_cuda import _lib
    args = list(ok)
    args[at] = value
    return getattr(_lib.lib, fn)(*args), _lib.last_error()


def test_free_blocks_refusals():
    from flash_kmeans_cuda import _lib
    need = _lib.lib.fkc_free_blocks_workspace_bytes(40)
    assert need > 0
    ok = [FAKE, 8, 8, FAKE, 3, 16, 40, FAKE, FAKE, FAKE, need, None]
    for at, value, code, word in (
            (0, None, 1, "null"), (1, 7, 1, "overlap"), (2, -1, 1, "range"), (3, None, 1, "null"),
            (4, -1, 1, "range"), (4, 1 << 31, 1, "range"), (4, 1 << 29, 4, "2^32"),
            (5, 0, 1, "range"),
            (5, (1 << 20) + 1, 1, "range"), (6, -1, 1, "range"), (6, 1 << 31, 1, "range"),
            (7, None, 1, "null"), (8, None, 1, "null"), (9, None, 2, "workspace"),
            (9, FAKE + 16, 2, "aligned"), (10, need - 1, 2, "workspace")):
        rc, msg = _call("fkc_free_blocks", ok, at, value)
        assert rc == code and word in msg, (at, value)
    assert _lib.lib.fkc_free_blocks_workspace_bytes(-1) == 0 and "range" in _lib.last_error()


def test_fork_refusals():
    from flash_kmeans_cuda import _lib
    c = _cache()
    ref = ctypes.addressof(c)
    need = _lib.lib.fkc_kv4_fork_workspace_bytes(ref, 5)
    ok = [ref, FAKE, 8, 8, FAKE, 3, FAKE, 5, FAKE, 6, FAKE, FAKE, FAKE, FAKE, need, None]
    for at, value, code, word in (
            (0, None, 1, "null cache"), (1, None, 1, "null"), (2, 7, 1, "overlap"),
            (3, -1, 1, "range"), (4, None, 1, "null"), (5, -1, 1, "range"), (6, None, 1, "null"),
            (5, 1 << 29, 4, "2^32"), (7, 1 << 29, 4, "2^32"), (7, 1 << 24, 4, "2^24"),
            (7, -1, 1, "range"), (8, None, 1, "null"), (9, -1, 1, "range"), (10, None, 1, "null"),
            (11, None, 1, "null"), (12, None, 1, "null"), (13, None, 2, "workspace"),
            (13, FAKE + 8, 2, "aligned"), (14, need - 1, 2, "workspace")):
        rc, msg = _call("fkc_kv4_fork", ok, at, value)
        assert rc == code and word in msg, (at, value)
    assert _lib.lib.fkc_kv4_fork_workspace_bytes(ref, -1) == 0 and "range" in _lib.last_error()


def test_compact_and_copy_refusals():
    from flash_kmeans_cuda import _lib
    far = 1 << 40
    c, d = _cache(), _cache(**{n: far + (i << 30) for i, n in enumerate(
        ("k_codes", "v_codes", "k_scales", "v_scales"))})
    a, b = ctypes.addressof(c), ctypes.addressof(d)
    need = _lib.lib.fkc_kv4_compact_workspace_bytes(a)
    ok = [a, FAKE, 8, 8, FAKE, 3, b, FAKE, FAKE, FAKE, need, None]
    size = 8 * 2 * 16 * 32  # bytes of codes
    near = _cache(k_codes=far, v_codes=far + (1 << 30), k_scales=far + (2 << 30),
                  v_scales=FAKE + size - 16)
    for at, value, code, word in (
            (0, None, 1, "null cache"), (6, None, 1, "null cache"), (6, a, 1, "share memory"),
            (6, ctypes.addressof(near), 1, "share memory"), (1, None, 1, "null"),
            (2, 7, 1, "overlap"), (5, -1, 1, "range"), (7, None, 1, "null"), (8, None, 1, "null"),
            (9, None, 2, "workspace"), (10, need - 1, 2, "workspace")):
        rc, msg = _call("fkc_kv4_compact", ok, at, value)
        assert rc == code and word in msg, (at, value)
    for kw in (dict(heads=4), dict(block_size=32), dict(D=128), dict(dtype=2)):
        e = _cache(**kw)
        rc, msg = _call("fkc_kv4_compact", ok, 6, ctypes.addressof(e))
        assert rc == 1 and "differ" in msg
        rc, msg = _call("fkc_kv4_copy_blocks", [a, FAKE, b, FAKE, 3, None], 2,
                        ctypes.addressof(e))
        assert rc == 1 and "differ" in msg
    ok = [a, FAKE, b, FAKE, 3, None]
    for at, value, word in ((0, None, "null cache"), (1, None, "null"), (2, None, "null cache"),
                            (3, None, "null"), (4, -1, "range"), (4, 1 << 31, "range")):
        rc, msg = _call("fkc_kv4_copy_blocks", ok, at, value)
        assert rc == 1 and word in msg
    assert _call("fkc_kv4_copy_blocks", ok, 4, 0)[0] == 0  # nothing to do
    huge = _cache(num_blocks=1, heads=16384, block_size=1 << 12, D=64)
    h = ctypes.addressof(huge)
    assert _call("fkc_kv4_copy_blocks", [h, FAKE, h, FAKE, 3, None], 4, 1)[0] == 4


def test_forks_of_blocks_past_31_bits_are_refused_by_name():
    """Blocks whose 16-byte units 32 bits do not count: the workspace's size is 0
    and says why, as the call itself does."""
    from flash_kmeans_cuda import _lib
    for kw in (dict(num_blocks=1, heads=16384, block_size=1 << 12, D=64),
               dict(num_blocks=1, heads=16384, block_size=1 << 20, D=256),
               dict(num_blocks=0, heads=8192, block_size=1 << 20, D=256)):
        c = _cache(**kw)
        ref = ctypes.addressof(c)
        assert _lib.lib.fkc_kv4_fork_workspace_bytes(ref, 5) == 0
        assert "2^31" in _lib.last_error()
        ok = [ref, FAKE, 8, 8, FAKE, 3, FAKE, 5, FAKE, 6, FAKE, FAKE, FAKE, FAKE, 1 << 40, None]
        assert _call("fkc_kv4_fork", ok, 7, 5)[0] == 4


@pytest.mark.parametrize("seed", range(40))
def test_reference_forks_leave_every_row_its_own_last_block(seed):
    """After a fork no row ends in a block that another row holds, and every
    row's blocks are its parent's or copies of them."""
    rng = random.Random(seed)
    bs, nb, width, R = 16, 60, 4, 6
    tables = np.array([[rng.randrange(12) for _ in range(width)] for _ in range(R)], np.int32)
    seq = np.array([rng.randrange(width * bs + 1) for _ in range(R)], np.int32)
    parents = [rng.randrange(-1, R) for _ in range(rng.randrange(12))]
    free = list(range(12, nb))
    new, out_seq, taken, copies = pages.fork(tables, seq, parents, free, bs, nb)
    rows = pages.held(new, out_seq, bs, nb)
    origin = dict((b, a) for a, b in copies)
    assert len(copies) == taken <= len(parents)
    for j, row in enumerate(rows):
        p = parents[j]
        if p < 0:
            assert row == []
            continue
        assert [origin.get(b, b) for b in row] == tables[p, :len(row)].tolist()
        if out_seq[j] % bs:
            others = [b for i, o in enumerate(rows) if i != j for b in o]
            whole = row[:-1]
            assert row[-1] not in others and row[-1] not in whole
