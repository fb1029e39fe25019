"""Attention over the 4-bit cache with capped scores, distances and masks on the
GPU against a plain 64-bit reference, within bounds derived from its arithmetic
(tests/kv4_scored_ref.py)."""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

import kv4_scored_ref as sref
from test_gpu_kv4 import BF16, F16, _setup, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv4():
    from flash_kmeans_cuda import kv4
    return kv4


def _slopes(H):
    return torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)])


def _documents(seq, nq, mean, seed):
    """Rows' first tokens, where every request is packed with documents."""
    rng = random.Random(seed)
    got = []
    for n, m in zip(seq, nq):
        first = np.zeros(max(n, m, 0), np.int64)
        at = 0
        while at < n:
            end = at + rng.randrange(1, 2 * mean)
            first[at:end] = at
            at = end
        got.append(first[len(first) - m:])
    return torch.from_numpy(np.concatenate(got)).to(torch.int32)


def _gpu(kw):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}


def _check(kv4, cache, tables, q, seq, nq, decode=False, **kw):
    want, want_lse, tol, lse_tol = sref.attend(q, cache, tables, seq, nq, **kw)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    cu = None if decode else i32(np.concatenate([[0], np.cumsum(nq)]).tolist())
    args = q.cuda(), dev, tables.cuda(), i32(seq), cu
    out, lse = kv4.attend(*args, return_lse=True, **_gpu(kw))
    got = out.cpu().double()
    err = (got - want).abs()
    assert bool((err <= tol).all()), f"out off by {float((err / tol.clamp(min=1e-30)).max()):.3g}"
    alive = want_lse > -math.inf
    assert torch.equal(lse.cpu() > -math.inf, alive)
    err = (lse.cpu().double() - want_lse).abs()[alive]
    assert bool((err <= lse_tol[alive]).all()), \
        f"lse off by {float((err / lse_tol[alive]).max()):.3g}"
    assert bool((got[~alive] == 0).all())
    # bit for bit again, and without lse
    assert torch.equal(out, kv4.attend(*args, **_gpu(kw)))
    return out


def _options(names, seq, nq, H, seed, window=37, mean=20):
    rng = random.Random(seed)
    n = len(nq)
    rows = sum(nq)
    kw = {}
    if "cap" in names:
        kw["softcap"] = 5.0
    if "slopes" in names:
        kw["slopes"] = _slopes(H)
    if "window" in names:
        kw["window"] = window
    if "docs" in names:
        kw["starts"] = _documents(seq, nq, mean, seed)
    if "prefix" in names:
        kw["prefix_lens"] = torch.tensor([rng.choice([0, 1, -3, max(s, 0) // 2, s, s + 9, 2 ** 31 - 1])
                                          for s in seq], dtype=torch.int32)
    assert n and rows >= 0
    return kw


OPTIONS = [("cap",), ("slopes",), ("window",), ("docs",), ("prefix",), ("cap", "window"),
           ("cap", "slopes"), ("slopes", "prefix"), ("window", "docs", "prefix"),
           ("cap", "slopes", "window", "docs", "prefix")]


def _id(o):
    return "+".join(o) if isinstance(o, tuple) else None


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,heads,G", [(64, 2, 4), (128, 3, 5), (256, 1, 16), (128, 1, 24),
                                       (64, 1, 1)])
@pytest.mark.parametrize("names", OPTIONS, ids=_id)
def test_single_tokens(kv4, dtype, D, heads, G, names):
    """Lengths around every tile and page border, idle rows."""
    seq = [1, 0, 15, 16, 17, 31, 32, 33, 64, 65, 127, 129, 500, 1]
    nq = [1] * len(seq)
    cache, tables, g = _setup(seq, 16, heads, D, dtype, 10 * D + G)
    q = (2 * torch.randn(len(seq), heads * G, D, generator=g)).to(dtype)
    _check(kv4, cache, tables, q, seq, nq, decode=True,
           **_options(names, seq, nq, heads * G, D))


@pytest.mark.parametrize("dtype,D,heads,G,bs", [
    (BF16, 128, 2, 4, 16), (F16, 64, 3, 1, 32), (F16, 256, 1, 8, 48), (BF16, 64, 1, 16, 128),
    (BF16, 128, 1, 7, 64), (BF16, 256, 2, 2, 16), (F16, 128, 2, 33, 32)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("names", OPTIONS, ids=_id)
def test_several_queries(kv4, dtype, D, heads, G, bs, causal, names):
    """Ragged: none, one, a few and many queries, more queries than tokens (the
    first ones see nothing, or the prefix), rows past the last request."""
    seq = [70, 3, 0, 200, 33, 130, 40, 0]
    nq = [3, 3, 0, 1, 33, 90, 45, 2]
    cache, tables, g = _setup(seq, bs, heads, D, dtype, D + G)
    q = (1.5 * torch.randn(sum(nq) + 4, heads * G, D, generator=g)).to(dtype)
    kw = _options(names, seq, nq, heads * G, D)
    if "starts" in kw:  # (one entry per row, those past the last request too)
        kw["starts"] = torch.cat([kw["starts"], torch.tensor([0, -1, 5, 2 ** 31 - 1],
                                                             dtype=torch.int32)])
    _check(kv4, cache, tables, q, seq, nq, causal=causal, **kw)


@pytest.mark.parametrize("D,columns", [(64, 352), (128, 448), (256, 288)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("names", [("cap",), ("slopes", "window"), ("docs", "prefix")], ids=_id)
def test_either_side_of_the_forms_border(kv4, dtype, D, columns, names):
    """The most columns of the form for few of them, and the fewest of the one
    for prompts; whole and in shares."""
    for seq in [400, 500], [3000, 1500]:
        for m in columns // 4, columns // 4 + 1:
            cache, tables, g = _setup(seq, 32, 1, D, dtype, D + m)
            q = torch.randn(2 * m, 4, D, generator=g).to(dtype)
            _check(kv4, cache, tables, q, seq, [m, m],
                   **_options(names, seq, [m, m], 4, D, window=200, mean=150))


@pytest.mark.parametrize("dtype,D,heads,G,bs", [
    (BF16, 128, 1, 4, 32), (F16, 64, 2, 2, 48), (F16, 256, 1, 2, 64), (BF16, 256, 1, 3, 16)])
@pytest.mark.parametrize("names", OPTIONS, ids=_id)
def test_prompts_in_shares(kv4, dtype, D, heads, G, bs, names):
    """Prompts and chunks behind a prefix, long enough to be cut."""
    seq, nq = [1300, 20, 2100, 0], [1300, 20, 300, 3]
    cache, tables, g = _setup(seq, bs, heads, D, dtype, 5)
    q = (1.5 * torch.randn(sum(nq), heads * G, D, generator=g)).to(dtype)
    kw = _options(names, seq, nq, heads * G, D, window=400, mean=150)
    _check(kv4, cache, tables, q, seq, nq, **kw)


@pytest.mark.parametrize("shape", sref.LONG_PROMPTS, ids=lambda s: str(s[1]))
@pytest.mark.parametrize("names", sref.LONG_OPTIONS, ids=_id)
def test_long_shares_of_prompts(kv4, shape, names):
    """Workgroups whose shares are several items, of one head and of two, cut at
    either end, and items of more than 1024 tokens; blocks missing all over them.
    A sample of the rows, every head."""
    dtype, D, heads, G, bs, seq, nq = shape
    cache, tables, g = _setup(seq, bs, heads, D, dtype, D)
    tables[0, 3] = -1
    tables[0, 1100 // bs:1200 // bs] = -1
    tables[0, 2100 // bs] = 2 ** 31 - 1
    tables[2, 2000 // bs:2064 // bs] = cache[0].shape[0]
    q = (1.5 * torch.randn(sum(nq), heads * G, D, generator=g)).to(dtype)
    kw = _options(names, seq, nq, heads * G, D, window=sref.LONG_WINDOW,
                  mean=sref.LONG_DOCUMENTS)
    rng = random.Random(D)
    first = np.concatenate([[0], np.cumsum(nq)]).tolist()
    pick = sorted({x for a, b in zip(first, first[1:]) for x in (
        a, a + 15, a + 16, b - 17, b - 1, *rng.sample(range(a, b), 25))})
    want, want_lse, tol, lse_tol = (x[pick] for x in sref.attend(q, cache, tables, seq, nq,
                                                                 pick=pick, **kw))
    dev = kv4.Cache(*(t.cuda() for t in cache))
    args = q.cuda(), dev, tables.cuda(), i32(seq), i32(first)
    out = torch.full_like(args[0], math.nan)
    _, lse = kv4.attend(*args, out=out, return_lse=True, **_gpu(kw))
    assert bool(torch.isfinite(out).all())
    err = (out.cpu().double()[pick] - want).abs()
    assert bool((err <= tol).all()), f"out off by {float((err / tol.clamp(min=1e-30)).max()):.3g}"
    err = (lse.cpu().double()[pick] - want_lse).abs()
    assert bool((err <= lse_tol).all()), f"lse off by {float((err / lse_tol).max()):.3g}"
    assert torch.equal(out, kv4.attend(*args, **_gpu(kw)))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bs", [16, 48, 256])
@pytest.mark.parametrize("names", OPTIONS, ids=_id)
def test_long_contexts(kv4, dtype, bs, names):
    """Contexts that are split over workgroups, beside short ones; and cut to
    max_seq."""
    seq = [5000, 1, 9001, 0, 700]
    cache, tables, g = _setup(seq, bs, 2, 128, dtype, bs)
    q = torch.randn(len(seq), 8, 128, generator=g).to(dtype)
    kw = _options(names, seq, [1] * 5, 8, bs, window=3333, mean=2000)
    _check(kv4, cache, tables, q, seq, [1] * 5, decode=True, **kw)
    _check(kv4, cache, tables, q, seq, [1] * 5, decode=True, max_seq=4999, **kw)
    nq = [3, 1, 2, 0, 5]
    q = torch.randn(sum(nq), 8, 128, generator=g).to(dtype)
    _check(kv4, cache, tables, q, seq, nq, **_options(names, seq, nq, 8, bs, 3333, 2000))


@pytest.mark.parametrize("nq", [1, 60, 240])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 32, 33, 100, 2 ** 31 - 1])
def test_windows(kv4, nq, window):
    seq = [250, 400, 33]
    cache, tables, g = _setup(seq, 16, 1, 64, BF16, window % 1000)
    q = torch.randn(3 * nq, 4, 64, generator=g).to(BF16)
    _check(kv4, cache, tables, q, seq, [nq] * 3, window=window)
    _check(kv4, cache, tables, q, seq, [nq] * 3, window=window, causal=False)


@pytest.mark.parametrize("nq", [1, 40, 300])
def test_starts_of_any_value(kv4, nq):
    """Unordered, negative, past the query, past everything: rows that see
    nothing beside rows that do, whole tiles of them too."""
    seq = [700, 300, 90]
    rng = random.Random(nq)
    cache, tables, g = _setup(seq, 32, 2, 128, F16, 8)
    q = torch.randn(3 * nq, 6, 128, generator=g).to(F16)
    starts = torch.tensor([rng.choice([0, -5, -2 ** 31, 2 ** 31 - 1, 299, 300, rng.randrange(700)])
                           for _ in range(3 * nq)], dtype=torch.int32)
    starts[nq:nq + nq // 2] = 5000
    for causal in True, False:
        _check(kv4, cache, tables, q, seq, [nq] * 3, starts=starts, causal=causal)
        _check(kv4, cache, tables, q, seq, [nq] * 3, starts=starts, causal=causal, softcap=20.0,
               slopes=_slopes(6), window=90)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq", [1, 70, 260])
@pytest.mark.parametrize("softcap", [0.5, 50.0, 1000.0])
def test_caps_of_small_and_large_scores(kv4, dtype, nq, softcap):
    """Scores far inside the cap, about it, and far beyond in both directions;
    a key of all zeros, one that dominates."""
    seq = [400, 300, 257, 100]
    cache, tables, g = _setup(seq, 32, 1, 128, dtype, 9)
    s = cache[2]
    s[tables[0, :13].long()] *= 30
    s[tables[1, :10].long()] *= 0.01
    s[tables[2, 3], 0, 7] = 500.0
    s[tables[3, :4].long()] = 0
    q = (2 * torch.randn(4 * nq, 4, 128, generator=g)).to(dtype)
    for scale in None, -0.3, 3.0, 0.0:
        _check(kv4, cache, tables, q, seq, [nq] * 4, sm_scale=scale, softcap=softcap)
    _check(kv4, cache, tables, q, seq, [nq] * 4, softcap=softcap, slopes=_slopes(4))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq", [1, 70, 260])
def test_slopes_of_any_size(kv4, dtype, nq):
    """Slopes of 0, so large that only the nearest token counts, negative, and
    different in every head; values from the smallest to the largest scales."""
    seq = [400, 300]
    cache, tables, g = _setup(seq, 32, 2, 64, dtype, 9)
    cache[3][tables[0, :13].long()] = (2.0 ** torch.randint(
        -14, 15, (13, 2, 32), generator=g).float()).to(dtype)
    q = (2 * torch.randn(2 * nq, 8, 64, generator=g)).to(dtype)
    slopes = torch.tensor([0.0, 1e-3, 0.1, 7.0, 1e4, -0.05, 1e-30, 0.7])
    _check(kv4, cache, tables, q, seq, [nq] * 2, slopes=slopes)
    _check(kv4, cache, tables, q, seq, [nq] * 2, slopes=slopes, causal=False)


@pytest.mark.parametrize("nq", [1, 60, 240])
@pytest.mark.parametrize("names", OPTIONS, ids=_id)
def test_missing_blocks_are_not_seen(kv4, nq, names):
    seq = [100, 60, 48]
    cache, tables, g = _setup(seq, 16, 2, 64, BF16, 4)
    tables[0, 2] = -1
    tables[0, 5] = cache[0].shape[0]
    tables[1, 0] = 2 ** 31 - 1
    tables[2] = -1  # nothing left
    q = torch.randn(3 * nq, 4, 64, generator=g).to(BF16)
    out = _check(kv4, cache, tables, q, seq, [nq] * 3,
                 **_options(names, seq, [nq] * 3, 4, nq))
    assert bool((out[2 * nq:] == 0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq", [1, 60, 240])
def test_what_a_mask_hides_is_anything(kv4, dtype, nq):
    """Pages before a window or a document may have been given back: their
    codes and scales, NaN and infinities, change nothing; where one is seen it
    shows."""
    seq = [600, 600]
    cache, tables, g = _setup(seq, 16, 1, 64, dtype, 12)
    q = torch.randn(2 * nq, 2, 64, generator=g).to(dtype)
    kw = [dict(window=40), dict(starts=torch.tensor([330] * (2 * nq), dtype=torch.int32)),
          dict(window=40, softcap=30.0, slopes=_slopes(2))]
    clean = [_check(kv4, cache, tables, q, seq, [nq] * 2, **k) for k in kw]
    for name in 2, 3:
        cache[name][tables[0, :8].long()] = math.nan
        cache[name][tables[0, 8:20].long()] = math.inf
    cache[0][tables[0, :20].long()] = 0xA5
    dev = kv4.Cache(*(t.cuda() for t in cache))
    cu = i32([0, nq, 2 * nq])
    for k, want in zip(kw, clean):
        sees = torch.zeros(2 * nq, dtype=torch.bool)
        if "window" in k:
            sees[:nq] = torch.arange(600 - nq, 600) - 40 < 319
        got = kv4.attend(q.cuda(), dev, tables.cuda(), i32(seq), cu, **_gpu(k))
        assert torch.equal(got.cpu()[~sees], want.cpu()[~sees])
        assert bool((~torch.isfinite(got.cpu()[sees])).flatten(1).any(1).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq", [1, 240])
def test_scores_that_are_not_numbers_show(kv4, dtype, nq):
    """A NaN among what a row sees makes that row NaN, and no other."""
    seq = [90, 90]
    cache, tables, g = _setup(seq, 16, 1, 64, dtype, 13)
    q = torch.randn(2 * nq, 2, 64, generator=g).to(dtype)
    for kw in dict(softcap=9.0), dict(slopes=_slopes(2)), dict(window=20):
        clean = _check(kv4, cache, tables, q, seq, [nq] * 2, **kw).cpu()
        bad = q.clone()
        bad[nq - 1, 1, 7] = math.nan
        dev = kv4.Cache(*(t.cuda() for t in cache))
        out, lse = kv4.attend(bad.cuda(), dev, tables.cuda(), i32(seq), i32([0, nq, 2 * nq]),
                              return_lse=True, **_gpu(kw))
        sees = torch.zeros(2 * nq, 2, dtype=torch.bool)
        sees[nq - 1, 1] = True
        assert torch.equal(torch.isnan(out.cpu()).all(-1), sees)
        assert torch.equal(torch.isnan(lse.cpu()), sees)
        assert torch.equal(out.cpu()[~sees], clean[~sees])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq", [1, 240])
def test_rows_that_see_nothing_ignore_their_query(kv4, dtype, nq):
    """Padding may hold NaN and infinities: such rows are 0 and -inf, and their
    neighbours what they are without them."""
    seq = [300, 80]
    cache, tables, g = _setup(seq, 16, 2, 64, dtype, 14)
    q = torch.randn(2 * nq, 4, 64, generator=g).to(dtype)
    starts = torch.zeros(2 * nq, dtype=torch.int32)
    starts[::3] = 301
    dev = kv4.Cache(*(t.cuda() for t in cache))
    for kw in dict(), dict(softcap=20.0), dict(slopes=_slopes(4), window=60):
        clean = _check(kv4, cache, tables, q, seq, [nq] * 2, starts=starts, **kw)
        bad = q.clone()
        bad[::3, :, ::2] = math.nan
        bad[::3, :, 1::2] = math.inf
        out, lse = kv4.attend(bad.cuda(), dev, tables.cuda(), i32(seq), i32([0, nq, 2 * nq]),
                              return_lse=True, starts=starts.cuda(), **_gpu(kw))
        assert torch.equal(out, clean)
        assert bool((lse[::3] == -math.inf).all())


def test_blocks_past_32_bits(kv4):
    """Codes beyond 4 GiB into the cache give what they give near its start, bit
    for bit, in both forms."""
    H, D, bs, nb = 16, 256, 128, 18000
    host, tables, g = _setup([2 * bs] * 2, bs, H, D, F16, 3, spare=0)
    far = kv4.Cache.empty(nb, bs, D, host[4].cuda(), host[5].cuda(), F16)
    assert far.k_codes.numel() > 2 ** 32
    near = kv4.Cache(*(t.cuda() for t in host))
    at = i32([nb - 1, 5, nb - 3, nb - 2])
    kv4.copy_blocks(near, i32([0, 1, 2, 3]), far, at)
    moved = at[tables.long().cuda()]
    for nq in 1, 20:
        q = torch.randn(2 * nq, 2 * H, D, generator=g).to(F16).cuda()
        q = q if nq == 1 else q.repeat(8, 1, 1)  # (enough columns for the form of prompts)
        m = q.shape[0] // 2
        for kw in (dict(softcap=20.0), dict(slopes=_slopes(2 * H).cuda(), window=100),
                   dict(prefix_lens=i32([50, 256]))):
            args = i32([250, 2 * bs]), i32([0, m, 2 * m])
            assert torch.equal(kv4.attend(q, far, moved, *args, **kw),
                               kv4.attend(q, near, tables.cuda(), *args, **kw))


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("long", [40, 2600])
def test_many_requests(kv4, ragged, long):
    """More tiles than a workgroup has threads, with and without cuts."""
    rng = random.Random(long)
    R = 1100
    seq = [rng.choice([0, 1, 17, rng.randrange(40)]) for _ in range(R)]
    seq[0] = seq[700] = seq[-1] = long
    nq = [rng.choice([0, 1, 2, 3]) for _ in range(R)] if ragged else [1] * R
    nq[700] = 1
    cache, tables, g = _setup(seq, 16, 1, 64, BF16, 6)
    q = torch.randn(sum(nq), 2, 64, generator=g).to(BF16)
    _check(kv4, cache, tables, q, seq, nq, decode=not ragged, softcap=3.0)
    _check(kv4, cache, tables, q, seq, nq, decode=not ragged, slopes=_slopes(2), window=1500)


@pytest.mark.parametrize("kw", [dict(), dict(softcap=20.0), dict(window=7)], ids=str)
def test_more_short_contexts_than_a_launch_has_workgroups(kv4, kw):
    """65600 requests of 128 heads: a workgroup of 512 threads each would be 2^32
    threads, so they go in shares.  An item's few tokens are one granule, which
    no share cuts: the answer is that of fewer requests, bit for bit."""
    H, D, R, few = 128, 64, 65600, 8
    seq = [1, 16, 7, 0, 9, 16, 3, 12]
    cache, tables, g = _setup(seq, 16, H, D, BF16, 3)
    q = torch.randn(few, H, D, generator=g).to(BF16)
    want = (_check(kv4, cache, tables, q, seq, [1] * few, decode=True, **kw) if kw else
            kv4.attend(q.cuda(), kv4.Cache(*(t.cuda() for t in cache)), tables.cuda(), i32(seq)))
    dev = kv4.Cache(*(t.cuda() for t in cache))
    many = R // few
    args = q.cuda().repeat(many, 1, 1), dev, tables.cuda().repeat(many, 1), i32(seq * many)
    for cu in None, i32(list(range(R + 1))):
        out = kv4.attend(*args, cu, **kw)
        assert torch.equal(out.view(many, few, H, D), want.expand(many, few, H, D))


@pytest.mark.parametrize("dtype,D,G", [(BF16, 128, 4), (F16, 64, 1), (F16, 256, 2)])
def test_rows_of_no_request_beside_cut_ones(kv4, dtype, D, G):
    """Steps padded to many times their queries: those rows are 0."""
    seq, nq = [1300, 40, 0, 5], [300, 900, 500, 1]
    cache, tables, g = _setup(seq, 64, 2, D, dtype, 3)
    q = (1.5 * torch.randn(9000, 2 * G, D, generator=g)).to(dtype)
    starts = torch.zeros(9000, dtype=torch.int32)
    starts[:300] = 200
    out = _check(kv4, cache, tables, q, seq, nq, softcap=30.0, starts=starts)
    assert bool((out[sum(nq):] == 0).all())


def test_the_options_of_nothing_are_none(kv4):
    """A cap far above every score, slopes of 0, a window of everything, no
    documents and no prefix: the answer without options.  Not its bits: a weight
    is rounded to the type relative to a maximum, which may lag here and does not
    there, and w 2^-a rounded times 2^a is w rounded only for whole a.  Both are
    within the bound of one rounding of each weight and of the result, which is
    what the reference's tolerance counts, so they are within twice that of each
    other."""
    seq, nq = [300, 700], [300, 5]
    cache, tables, g = _setup(seq, 16, 2, 128, BF16, 3)
    q = torch.randn(sum(nq), 8, 128, generator=g).to(BF16)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    args = q.cuda(), dev, tables.cuda(), i32(seq), i32([0, 300, 305])
    want = kv4.attend(*args).cpu().double()
    tol = sref.attend(q, cache, tables, seq, nq)[2]
    zero = torch.zeros(305, dtype=torch.int32, device="cuda")
    for kw in (dict(window=10 ** 6), dict(starts=zero), dict(prefix_lens=zero[:2])):
        assert bool(((kv4.attend(*args, **kw).cpu().double() - want).abs() <= 2 * tol).all())
    for kw in (dict(softcap=1e6), dict(slopes=torch.zeros(8, device="cuda"))):
        _check(kv4, cache, tables, q, seq, nq, **{k: v.cpu() if isinstance(v, torch.Tensor) else v
                                                  for k, v in kw.items()})


@pytest.mark.parametrize("nq", [[300, 5], [1, 1], [40, 40]])
def test_the_options_of_nothing_give_the_bits_of_none(kv4, nq):
    """bf16, where both kernels make weights relative to the largest score: a
    window of everything, no documents, no prefix leave the same operations in
    the same order."""
    seq = [300, 700]
    cache, tables, g = _setup(seq, 16, 2, 128, BF16, 3)
    q = torch.randn(sum(nq), 8, 128, generator=g).to(BF16)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    args = q.cuda(), dev, tables.cuda(), i32(seq), i32([0, nq[0], sum(nq)])
    want, want_lse = kv4.attend(*args, return_lse=True)
    zero = torch.zeros(sum(nq), dtype=torch.int32, device="cuda")
    for kw in (dict(window=10 ** 6), dict(starts=zero), dict(prefix_lens=zero[:2])):
        out, lse = kv4.attend(*args, return_lse=True, **kw)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nq", [1, 128])
@pytest.mark.parametrize("kw", [dict(window=10 ** 6), dict(softcap=50.0), dict(softcap=1000.0),
                                dict(slopes=None)], ids=str)
def test_the_largest_weight_is_not_rounded(kv4, dtype, D, nq, kw):
    """One token, late, scores up to 6 powers of two above all others, and only
    it has a value.  Weights are relative to the largest, whose weight is 1 to
    2^-20 whatever came before it: times its scale, a number of the type, it is
    exact, and what is left of the reference's bound is the result's one rounding
    and the scores' errors.  (fp16: relative to the largest weight times scale,
    which is 2^14 then.  A token whose score is D lower and whose scale is more
    than e^D times as large has the larger one; the late token's is 2^14 times
    any number below 1 then, and rounded like every other: such rows keep the
    reference's bound.)"""
    n, late, H, G = 400, 300, 2, 4
    cache, tables, g = _setup([n], 16, H, D, dtype, D + nq)
    k_codes, v_codes, k_scales, v_scales, k_levels, v_levels = cache
    k_codes[:] = k_codes[:1, :, :1]
    v_levels[:, 0] = 0
    at = tables[0, late // 16], slice(None), late % 16
    value = v_codes[at].clone()
    v_codes[:] = 0  # of level 0
    v_codes[at] = value
    k_scales[:] = 1.0
    k_scales[at] = 1.5
    both = torch.stack((k_codes[0, :, 0] & 15, k_codes[0, :, 0] >> 4), -1).flatten(-2).long()
    key = k_levels.float().gather(1, both)  # the same for all tokens of a head
    score = 0.5 + 7.5 * torch.rand(nq, H, G, 1, generator=g)  # of every other token
    q = (score * (key * D ** 0.5 / key.square().sum(-1, keepdim=True))[:, None])
    q = q.reshape(nq, H * G, D).to(dtype)
    if "slopes" in kw:
        kw = dict(slopes=torch.full((H * G,), 1e-4))
    want, want_lse, tol, lse_tol = sref.attend(q, cache, tables, [n], [nq], causal=False, **kw)
    exact = torch.ones(nq, H, G, 1, dtype=torch.bool)
    if dtype is F16:
        cap = kw.get("softcap", math.inf)
        above = [cap * torch.tanh(z / cap) if cap < math.inf else z for z in (1.5 * score, score)]
        scale = v_scales[tables[0, :n // 16].long()].float()  # (blocks, heads, slots)
        lead = scale.amax((0, 2)).log() - v_scales[at].float().log()
        exact = above[0] - above[1] > lead.view(H, 1, 1) + 0.05  # (0.05: q is rounded)
        assert nq == 1 or exact.float().mean() > 0.5
    tol = tol - 1.01 * sref.ref.UNIT[dtype] * want.abs() * exact.reshape(nq, H * G, 1)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    got, lse = kv4.attend(q.cuda(), dev, tables.cuda(), i32([n]), i32([0, nq]), causal=False,
                          return_lse=True, **_gpu(kw))
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"out off by {float((err / tol).max()):.3g}"
    assert bool(((lse.cpu().double() - want_lse).abs() <= lse_tol).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq", [1, 6, 260])
@pytest.mark.parametrize("softcap", [1e-30, 1e-9, 256.0, 257.0, 3e4, 1e9, 1e30])
def test_caps_of_any_size(kv4, dtype, nq, softcap):
    """Caps far below every score, where all weights are alike, to far above,
    where they are those without a cap."""
    seq = [400, 257]
    cache, tables, g = _setup(seq, 32, 2, 64, dtype, 11)
    cache[2][tables[0, :5].long()] *= 20
    q = (3 * torch.randn(2 * nq, 8, 64, generator=g)).to(dtype)
    for scale in None, -2.0:
        _check(kv4, cache, tables, q, seq, [nq] * 2, sm_scale=scale, softcap=softcap)
    _check(kv4, cache, tables, q, seq, [nq] * 2, softcap=softcap, slopes=_slopes(8), window=300)


def test_rows_of_nothing(kv4):
    """Queries of no request, requests of no tokens, tables without entries, no
    query at all; slopes in steps."""
    seq = [40, 60]
    cache, tables, g = _setup(seq, 16, 2, 64, F16, 7)
    dev, t = kv4.Cache(*(x.cuda() for x in cache)), tables.cuda()
    q = torch.randn(5, 8, 64, generator=g).to(F16).cuda()
    none = i32([])
    slopes = torch.zeros(8, 3, device="cuda")
    slopes[:, 1] = _slopes(8).cuda()
    strided = slopes[:, 1]
    for kw in dict(softcap=9.0), dict(slopes=strided), dict(window=20), dict(softcap=1e4):
        for args in ((t[:0], none, i32([0])), (t[:0, :0], none, i32([0])),
                     (t[:, :0], i32(seq), i32([0, 2, 5])), (t, i32([0, -3]), i32([0, 2, 5]))):
            out, lse = kv4.attend(q, dev, *args, return_lse=True, **kw)
            assert not bool(out.any()) and bool((lse == -math.inf).all())
        out = kv4.attend(q, dev, t, i32(seq), i32([0, 2, 5]), max_seq=0, **kw)
        assert not bool(out.any())
        out, lse = kv4.attend(q[:0], dev, t, i32(seq), i32([0, 0, 0]), return_lse=True, **kw)
        assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
    args = q, dev, t, i32(seq), i32([0, 2, 5])
    assert torch.equal(kv4.attend(*args, slopes=strided),
                       kv4.attend(*args, slopes=strided.contiguous()))


def test_offsets_that_do_not_ascend_end(kv4):
    """Nonsense offsets stay in range, and what they do not name is written as
    it is without them."""
    seq = [3000, 40, 900]
    cache, tables, g = _setup(seq, 16, 1, 64, BF16, 4)
    q = torch.randn(600, 4, 64, generator=g).to(BF16).cuda()
    dev = kv4.Cache(*(t.cuda() for t in cache))
    for cu in ([0, 500, 100, 600], [0, -5, 2 ** 31 - 1, 600], [600, 0, 600, 0], [7, 7, 7, 7]):
        for kw in (dict(softcap=9.0), dict(window=50, starts=i32([3] * 600))):
            out = kv4.attend(q, dev, tables.cuda(), i32(seq), i32(cu), **kw)
            torch.cuda.synchronize()
            assert out.shape == q.shape


@pytest.mark.parametrize("kw", [dict(), dict(softcap=9.0), dict(window=50)], ids=str)
def test_rows_that_one_request_names_are_its_own(kv4, kw):
    """Offsets that do not ascend: rows that a single request names are its
    answer, rows past the last offset are 0, and what nothing else is named by
    is not left as it was."""
    seq = [3000, 40, 900]
    cache, tables, g = _setup(seq, 16, 1, 64, BF16, 4)
    q = torch.randn(600, 4, 64, generator=g).to(BF16)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    # rows 100 .. 499 belong to the first and the last request
    want, want_lse, tol, lse_tol = sref.attend(q, cache, tables, seq, [500, 0, 100], **kw)
    own = [*range(100), *range(500, 600)]
    out = torch.full((600, 4, 64), math.nan, dtype=BF16, device="cuda")
    _, lse = kv4.attend(q.cuda(), dev, tables.cuda(), i32(seq), i32([0, 500, 100, 600]), out=out,
                        return_lse=True, **kw)
    assert bool(((out.cpu().double() - want).abs() <= tol)[own].all())
    assert bool(((lse.cpu().double() - want_lse).abs() <= lse_tol)[own].all())
    assert bool(torch.isfinite(out).all())
    out.fill_(math.nan)
    _, lse = kv4.attend(q.cuda(), dev, tables.cuda(), i32(seq), i32([7, 7, 7, 7]), out=out,
                        return_lse=True, **kw)
    assert not bool(out[7:].any()) and bool((lse[7:] == -math.inf).all())


def test_strided_queries_and_another_stream(kv4):
    seq, nq = [300, 90], [70, 90]
    cache, tables, g = _setup(seq, 16, 2, 64, F16, 7)
    wide = torch.randn(160, 12, 64, generator=g).to(F16)
    kw = _options(("cap", "slopes", "docs"), seq, nq, 8, 3)
    want = _check(kv4, cache, tables, wide[:, 2:10], seq, nq, **kw)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    args = wide.cuda()[:, 2:10], dev, tables.cuda(), i32(seq), i32([0, 70, 160])
    more = _gpu(kw)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = kv4.attend(*args, **more)
    side.synchronize()
    assert torch.equal(got, want)


def test_captured(kv4):
    """Captured with cuts, replayed on other inputs beside eager calls and a
    second graph of the same pool."""
    seq0 = [5000, 300, 2500]
    cache, tables, g = _setup(seq0, 16, 2, 128, BF16, 7)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    q = torch.zeros(12, 8, 128, dtype=BF16, device="cuda")
    seq, starts = i32(seq0), i32([0] * 12)
    cu, slopes = i32([0, 4, 5, 12]), _slopes(8).cuda()

    def work():
        return (kv4.attend(q, dev, gpu_tables, seq, cu, softcap=20.0,
                           starts=starts),
                kv4.attend(q, dev, gpu_tables, seq, cu, slopes=slopes, window=900))

    gpu_tables = tables.cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(work())
        graphs.append(graph)
    for i in range(4):
        q.copy_(torch.randn(12, 8, 128, generator=g).to(BF16))
        seq.copy_(i32([5000 - 900 * i, 300 - i, 2500 - 7 * i]))
        starts.copy_(i32([100 * i + j for j in range(12)]))
        eager = work()
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, eager):
                assert torch.equal(a, b)


def test_gradients_raise(kv4):
    seq = [40, 60]
    cache, tables, g = _setup(seq, 16, 1, 64, F16, 7)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    q = torch.randn(2, 4, 64, generator=g).to(F16).cuda()
    s = _slopes(4).cuda()
    for a, b in ((q.clone().requires_grad_(), s), (q, s.clone().requires_grad_())):
        out = kv4.attend(a, dev, tables.cuda(), i32(seq), slopes=b)
        assert out.requires_grad
        with pytest.raises(RuntimeError, match="no gradient"):
            out.sum().backward()
        with torch.no_grad():
            assert not kv4.attend(a, dev, tables.cuda(), i32(seq), slopes=b).requires_grad


@pytest.mark.parametrize("kw,word", [
    (dict(softcap=0.0), "softcap"), (dict(softcap=-1.0), "softcap"),
    (dict(softcap=math.inf), "softcap"), (dict(softcap=math.nan), "softcap"),
    (dict(softcap=1e-50), "softcap"), (dict(softcap=9e-31), "softcap"),
    (dict(softcap=2e30), "softcap"),
    (dict(window=0), "window"), (dict(window=-1), "window"), (dict(window=1 << 31), "window"),
    (dict(slopes=torch.zeros(4)), None), (dict(slopes="half"), "float32"),
    (dict(slopes="short"), "float32"), (dict(starts="long"), "int32"),
    (dict(starts="short"), "one entry"), (dict(prefix_lens="short"), "as long"),
    (dict(prefix_lens="wide"), "dimension")])
def test_refusals(kv4, kw, word):
    seq = [40, 60]
    cache, tables, g = _setup(seq, 16, 1, 64, F16, 7)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    q = torch.zeros(2, 4, 64, dtype=F16, device="cuda")
    made = {("slopes", "half"): torch.zeros(4, dtype=F16, device="cuda"),
            ("slopes", "short"): torch.zeros(3, device="cuda"),
            ("starts", "long"): torch.zeros(2, dtype=torch.int64, device="cuda"),
            ("starts", "short"): i32([1]), ("prefix_lens", "short"): i32([1]),
            ("prefix_lens", "wide"): i32([[1, 2]])}
    kw = {k: made[k, v] if isinstance(v, str) else v for k, v in kw.items()}
    with pytest.raises(ValueError if word is None else RuntimeError, match=word):
        kv4.attend(q, dev, tables.cuda(), i32(seq), **kw)
