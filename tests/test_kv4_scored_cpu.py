"""Attention with capped, biased or masked scores: its C entry points refuse
what their kernels could not index, before anything reaches a device; and the
reference's masks are checked one by one."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import kv4_scored_ref as sref
from test_kv4_cpu import FAKE, _cache


def _scores(softcap=0.0, slopes=None, window=0, starts=None, prefix=None):
    from flash_kmeans_cuda.kv4 import _CScores
    return _CScores(softcap, slopes, window, starts, prefix)


def _attend(scores, q=FAKE, ts=256, hs=64, H=4, T=3, tables=FAKE, stride=8, width=8, seq=FAKE,
            cu=None, R=3, max_seq=128, out=FAKE, ws=None, nbytes=0, cache=None):
    from flash_kmeans_cuda import _lib
    c = cache or _cache()
    rc = _lib.lib.fkc_kv4_attend_scored(
        ctypes.addressof(c), q, ts, hs, H, T, tables, stride, width, seq, cu, R, max_seq, 1, 0.1,
        ctypes.addressof(scores) if scores is not None else None, out, None, ws, nbytes, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(softcap=-1.0), "softcap"), (dict(softcap=math.inf), "softcap"),
    (dict(softcap=math.nan), "softcap"), (dict(softcap=1e-31), "softcap"),
    (dict(softcap=1e31), "softcap"), (dict(window=-1), "window"),
    (dict(window=1 << 31), "window")])
def test_options_are_checked(kw, word):
    from flash_kmeans_cuda import _lib
    x, c = _scores(**kw), _cache()
    rc, msg = _attend(x)
    assert rc == 1 and word in msg
    assert _lib.lib.fkc_kv4_attend_scored_workspace_bytes(
        ctypes.addressof(c), 4, 3, 3, 128, 1, ctypes.addressof(x)) == 0
    assert word in _lib.last_error()


def test_null_options():
    rc, msg = _attend(None)
    assert rc == 1 and "null scores" in msg


@pytest.mark.parametrize("scores", [dict(), dict(softcap=30.0), dict(window=5), dict(slopes=FAKE),
                                    dict(starts=FAKE), dict(prefix=FAKE)])
@pytest.mark.parametrize("kw,word", [
    (dict(H=3), "multiple"), (dict(T=-1), "range"), (dict(max_seq=129), "longer"),
    (dict(T=4), "T == R"), (dict(stride=7), "overlap"), (dict(q=None), "null"),
    (dict(q=FAKE + 2), "aligned"), (dict(hs=63), "aligned"), (dict(out=None), "null"),
    (dict(seq=None), "null"), (dict(tables=None), "null"), (dict(out=FAKE + 8), "aligned")])
def test_refusals(scores, kw, word):
    rc, msg = _attend(_scores(**scores), **kw)
    assert rc == 1 and word in msg


@pytest.mark.parametrize("scores", [dict(), dict(softcap=30.0), dict(slopes=FAKE, window=90000)])
def test_workspace(scores):
    from flash_kmeans_cuda import _lib
    c, x = _cache(num_blocks=1 << 16), _scores(**scores)
    need = _lib.lib.fkc_kv4_attend_scored_workspace_bytes(
        ctypes.addressof(c), 4, 1, 1, 100000, 1, ctypes.addressof(x))
    assert need > 0
    kw = dict(T=1, R=1, max_seq=100000, width=6250, stride=6250, cache=c)
    assert _attend(x, **kw)[0] == 2
    rc, msg = _attend(x, ws=FAKE, nbytes=need - 1, **kw)
    assert rc == 2 and "workspace" in msg
    rc, msg = _attend(x, ws=FAKE + 16, nbytes=need, **kw)
    assert rc == 2 and "aligned" in msg


@pytest.mark.parametrize("scores", [dict(), dict(softcap=30.0), dict(slopes=FAKE, window=7)])
@pytest.mark.parametrize("D,waves", [(64, 8), (128, 8), (256, 4)])
def test_no_launch_of_2_32_threads(scores, D, waves):
    """Short contexts go to a workgroup each while their threads are below 2^32,
    and to equal shares (which need a workspace) from there on."""
    from flash_kmeans_cuda import _lib
    heads = 128
    c, x = _cache(num_blocks=8, heads=heads, D=D), _scores(**scores)

    def need(rows):
        if scores:
            return _lib.lib.fkc_kv4_attend_scored_workspace_bytes(
                ctypes.addressof(c), heads, rows, rows, 16, 1, ctypes.addressof(x))
        return _lib.lib.fkc_kv4_attend_workspace_bytes(ctypes.addressof(c), heads, rows, rows, 16)

    # tiles of offsets that are not known yet: one per request and one per 16 rows
    most = (2 ** 32 // (64 * waves * heads)) * 16 // 17 - 2
    assert need(most) == 0 and need(most * 17 // 16 + 8) > 0


@pytest.mark.parametrize("D,columns", [(64, 352), (128, 448), (256, 288)])
def test_the_forms_border(D, columns):
    """Up to so many columns of an average request the form for few of them is
    taken, whose parts are narrower: what the measurements beside the plan say."""
    from flash_kmeans_cuda import _lib
    c, x = _cache(num_blocks=1 << 12, D=D, heads=1), _scores(softcap=30.0)

    def parts(m):
        return _lib.lib.fkc_kv4_attend_scored_workspace_bytes(
            ctypes.addressof(c), 4, 8 * m, 8, 40000, 1, ctypes.addressof(x))

    # (the list of tiles grows with them, by less than a hundredth)
    assert parts(columns // 4) < 1.01 * parts(columns // 5)
    assert parts(columns // 4 + 1) > 3 * parts(columns // 4)
    assert parts(columns // 2) < 1.01 * parts(columns // 4 + 1)


@pytest.mark.parametrize("requests", [(1 << 26) - 4, (1 << 27) - 1])
def test_a_launch_that_weighs_tiles_has_a_wave_for_each(requests):
    """Of 64 threads, four to a workgroup: 2^26 - 4 tiles fill 2^24 workgroups of
    256, one launch too many."""
    c = _cache(num_blocks=8, heads=1)
    for scores in dict(softcap=30.0), dict(window=5):
        rc, msg = _attend(_scores(**scores), H=1, T=requests * 0, R=requests, cu=FAKE, max_seq=16,
                          cache=c, ws=FAKE, nbytes=1 << 50)
        assert rc == 0  # nothing to do
        rc, msg = _attend(_scores(**scores), H=1, T=1, R=requests, cu=FAKE, max_seq=16,
                          cache=c, ws=FAKE, nbytes=1 << 50)
        assert rc == 4 and "too many rows" in msg


def test_too_many_tiles():
    c = _cache(num_blocks=8, heads=1)
    for scores in dict(softcap=30.0), dict(window=5):
        rc, msg = _attend(_scores(**scores), H=1, T=1 << 27, R=1 << 27, max_seq=16, cache=c,
                          ws=FAKE, nbytes=1 << 50)
        assert rc == 4 and "too many rows" in msg


def test_reference_masks():
    """Written out by hand: four queries at positions 2 .. 5 of six tokens."""
    def rows(**kw):
        return ["".join("x" if v else "." for v in r) for r in sref.seen(6, 4, **kw).tolist()]
    assert rows() == ["xxx...", "xxxx..", "xxxxx.", "xxxxxx"]
    assert rows(window=2) == [".xx...", "..xx..", "...xx.", "....xx"]
    assert rows(window=2, causal=False) == [".xxxxx", "..xxxx", "...xxx", "....xx"]
    assert rows(prefix=4) == ["xxxx..", "xxxx..", "xxxxx.", "xxxxxx"]
    assert rows(prefix=4, window=3) == ["xxxx..", ".xxx..", "..xxx.", "...xxx"]
    assert rows(starts=torch.tensor([0, 3, 3, 9])) == ["xxx...", "...x..", "...xx.", "......"]
    assert sref.seen(1, 3).tolist() == [[False], [False], [True]]
    assert sref.seen(1, 3, prefix=7).tolist() == [[True], [True], [True]]


def test_reference_is_plain_attention_with_nothing_set():
    import kv4_ref as ref
    cache = ref.random_cache(4, 1, 16, 64, torch.float16, 1)
    tables = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32)
    q = torch.randn(6, 2, 64, generator=torch.Generator().manual_seed(1)).half()
    a = ref.attend(q, cache, tables, [20, 31], [2, 4])
    b = sref.attend(q, cache, tables, [20, 31], [2, 4])
    assert torch.allclose(a[0], b[0], atol=1e-12) and torch.allclose(a[1], b[1], atol=1e-12)


@pytest.mark.parametrize("shape", sref.LONG_PROMPTS, ids=lambda s: str(s[1]))
@pytest.mark.parametrize("names", sref.LONG_OPTIONS, ids="+".join)
def test_long_prompts_fill_their_shares(shape, names):
    """What the test of long shares is for: at 256 compute units shares hold more
    than one item, of two heads too, items of more than 1024 tokens, and cut
    items behind whole ones."""
    from test_gpu_kv4_scored import _options
    dtype, D, heads, G, bs, seq, nq = shape
    kw = _options(names, seq, nq, heads * G, D, window=sref.LONG_WINDOW, mean=sref.LONG_DOCUMENTS)
    for unused in "softcap", "slopes":
        kw.pop(unused, None)
    shares = sref.replay(D, heads, G, seq, nq, 256, **kw)
    with_tokens = [[x for x in s if x[2] < x[3]] for s in shares]
    assert sum(len(s) > 1 for s in with_tokens) > 100
    assert sum(len({x[0] for x in s}) > 1 for s in with_tokens) >= min(heads - 1, 5)
    assert sum(any(x[3] - x[2] > 1024 for x in s) for s in with_tokens) > 20
    assert sum(len(s) > 1 and s[-1][4] for s in with_tokens) > 50
    # every item's tokens once
    for h in range(heads):
        covered = {}
        for s in shares:
            for head, tile, a, b, more in s:
                if head == h:
                    assert covered.get(tile, a) == a
                    covered[tile] = b
