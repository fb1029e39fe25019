"""The 4-bit cache's C entry points refuse what their kernels could not index,
before anything reaches a device; host tensors are refused in Python."""

from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 0x10000  # never dereferenced: validation fails first


def _cache(**kw):
    from flash_kmeans_cuda.kv4 import _CCache
    f = dict(k_codes=FAKE, v_codes=FAKE, k_scales=FAKE, v_scales=FAKE, k_levels=FAKE,
             v_levels=FAKE, num_blocks=8, heads=2, block_size=16, D=64, dtype=1)
    f.update(kw)
    return _CCache(*f.values())


def _attend(c, q=FAKE, ts=256, hs=64, H=4, T=3, tables=FAKE, stride=8, width=8, seq=FAKE, cu=None,
            R=3, max_seq=128, out=FAKE, ws=None, nbytes=0):
    from flash_kmeans_cuda import _lib
    rc = _lib.lib.fkc_kv4_attend(ctypes.addressof(c), q, ts, hs, H, T, tables, stride, width, seq,
                                 cu, R, max_seq, 1, 0.1, out, None, ws, nbytes, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=0), 4, "dtype"), (dict(dtype=9), 1, "dtype"), (dict(D=96), 4, "D = 96"),
    (dict(D=0), 1, "D = 0"), (dict(block_size=24), 1, "block_size"),
    (dict(block_size=0), 1, "block_size"), (dict(heads=0), 1, "heads"),
    (dict(num_blocks=-1), 1, "num_blocks"), (dict(num_blocks=1 << 28), 1, "2^31"),
    (dict(num_blocks=1 << 26, heads=64), 4, "2^35"), (dict(k_codes=None), 1, "null"),
    (dict(k_levels=None, num_blocks=0), 1, "levels"), (dict(v_scales=FAKE + 8), 1, "aligned")])
def test_cache_is_checked_by_every_entry(kw, code, word):
    from flash_kmeans_cuda import _lib
    c = _cache(**kw)
    ref = ctypes.addressof(c)
    for call in (lambda: _lib.lib.fkc_kv4_append(ref, FAKE, 128, 64, FAKE, 128, 64, FAKE, 3, None),
                 lambda: _lib.lib.fkc_kv4_read(ref, FAKE, 3, FAKE, FAKE, None),
                 lambda: _attend(c, H=4 * max(kw.get("heads", 1), 1))[0]):
        assert call() == code and word in _lib.last_error()
    assert _lib.lib.fkc_kv4_attend_workspace_bytes(ref, 4, 3, 3, 128) == 0
    assert word in _lib.last_error()


def test_null_cache():
    from flash_kmeans_cuda import _lib
    assert _lib.lib.fkc_kv4_read(None, FAKE, 3, FAKE, FAKE, None) == 1
    assert "null cache" in _lib.last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(H=3), "multiple"), (dict(H=0), "multiple"), (dict(T=-1), "range"),
    (dict(T=1 << 30), "range"), (dict(max_seq=129), "longer"), (dict(max_seq=-1), "range"),
    (dict(T=4), "T == R"), (dict(stride=7), "overlap"), (dict(q=None), "null"),
    (dict(q=FAKE + 2), "aligned"), (dict(ts=252), "aligned"), (dict(hs=63), "aligned"),
    (dict(out=None), "null"), (dict(seq=None), "null"), (dict(tables=None), "null"),
    (dict(out=FAKE + 8), "aligned")])
def test_attend_refusals(kw, word):
    rc, msg = _attend(_cache(), **kw)
    assert rc == 1 and word in msg


def test_attend_workspace():
    """Long contexts of few rows are split: their workspace is asked for."""
    from flash_kmeans_cuda import _lib
    c = _cache(num_blocks=1 << 16)
    need = _lib.lib.fkc_kv4_attend_workspace_bytes(ctypes.addressof(c), 4, 1, 1, 100000)
    if need == 0:
        pytest.skip("this plan does not split")
    kw = dict(T=1, R=1, max_seq=100000, width=6250, stride=6250)
    assert _attend(c, **kw)[0] == 2
    rc, msg = _attend(c, ws=FAKE, nbytes=need - 1, **kw)
    assert rc == 2 and "workspace" in msg
    rc, msg = _attend(c, ws=FAKE + 16, nbytes=need, **kw)
    assert rc == 2 and "aligned" in msg


def test_append_and_read_refusals():
    from flash_kmeans_cuda import _lib
    L, c = _lib.lib, _cache()
    ref = ctypes.addressof(c)
    ok = [ref, FAKE, 128, 64, FAKE, 128, 64, FAKE, 3, None]
    for at, value, word in ((1, None, "null"), (4, None, "null"), (7, None, "null"),
                            (8, -1, "range"), (2, 100, "aligned"), (6, 60, "aligned"),
                            (4, FAKE + 4, "aligned")):
        args = list(ok)
        args[at] = value
        assert L.fkc_kv4_append(*args) == 1 and word in _lib.last_error()
    ok[8] = 0
    assert L.fkc_kv4_append(*ok) == 0  # nothing to do
    assert L.fkc_kv4_read(ref, FAKE, 3, FAKE + 8, None, None) == 1
    assert L.fkc_kv4_read(ref, None, 3, FAKE, None, None) == 1
    assert L.fkc_kv4_read(ref, None, 3, None, None, None) == 0  # nothing asked


def test_block_tables_refusals():
    from flash_kmeans_cuda import _lib
    ok = [FAKE, FAKE, 3, FAKE, 4, 4, FAKE, 5, 16, 9, FAKE, FAKE, FAKE, None]
    for at, value, word in ((2, -1, "range"), (7, -1, "range"), (8, 0, "range"),
                            (9, -1, "range"), (4, 3, "overlap"), (0, None, "null"),
                            (1, None, "null"), (3, None, "null"), (6, None, "null"),
                            (10, None, "null"), (11, None, "null"), (12, None, "null")):
        args = list(ok)
        args[at] = value
        assert _lib.lib.fkc_block_tables(*args) == 1 and word in _lib.last_error()


def test_host_tensors_are_refused():
    from flash_kmeans_cuda import kv4
    z = torch.zeros(2, 1, 16, 32, dtype=torch.uint8)
    s = torch.zeros(2, 1, 16, dtype=torch.float16)
    lv = torch.zeros(1, 16, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        kv4.Cache(z, z, s, s, lv, lv)
    with pytest.raises(ValueError):
        kv4.learn_levels(torch.zeros(4, 1, 64))
    with pytest.raises(ValueError):
        kv4.block_tables(i, i, i.view(2, 1), i, 16, 2)
