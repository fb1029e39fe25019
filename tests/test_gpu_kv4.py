"""The 4-bit key/value cache on the GPU against plain 64-bit references:
block tables, storing and reading back bit for bit, attention within bounds
derived from its arithmetic (tests/kv4_ref.py)."""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def kv4():
    from flash_kmeans_cuda import kv4
    return kv4


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------ block tables

def _lens(R, hi, new_hi, seed):
    rng = random.Random(seed)
    seq = [rng.choice([0, 1, hi, rng.randrange(hi + 1)]) for _ in range(R)]
    return seq, [min(s, rng.choice([0, 1, new_hi, rng.randrange(new_hi + 1)])) for s in seq]


@pytest.mark.parametrize("R,hi,new_hi,bs,pad", [
    (1, 1, 1, 16, 0), (1, 5000, 5000, 16, 3), (7, 100, 1, 16, 2), (33, 70, 70, 48, 0),
    (300, 900, 40, 32, 17), (2047, 64, 9, 16, 0), (2048, 64, 9, 64, 1), (2049, 200, 3, 16, 900),
    (5000, 40, 2, 128, 5), (3, 9000, 9000, 1, 4)])
def test_block_tables(kv4, R, hi, new_hi, bs, pad):
    seq, new = _lens(R, hi, new_hi, R + bs)
    width = -(-max(max(seq), 1) // bs) + 1
    rng = np.random.default_rng(R)
    pool = rng.permutation(R * width + 7).astype(np.int32)
    tables = np.full((R, width), -7, np.int32)
    at = 0
    for r in range(R):
        n = -(-(seq[r] - new[r]) // bs)
        tables[r, :n] = pool[at:at + n]
        at += n
    free, num = pool[at:], sum(new) + pad
    want = ref.block_tables(seq, new, tables, free, bs, num)
    got = torch.from_numpy(tables).cuda()
    for _ in range(2):  # the entries that a call writes are not what it reads
        slots, cu, taken = kv4.block_tables(i32(seq), i32(new), got,
                                            torch.from_numpy(free).cuda(), bs, num)
        assert np.array_equal(got.cpu().numpy(), want[0])
        assert np.array_equal(slots.cpu().numpy(), want[1])
        assert np.array_equal(cu.cpu().numpy(), want[2])
        assert taken.tolist() == [want[3]]


def test_block_tables_shortages(kv4):
    """Too few free blocks, rows too short, room for fewer slots than tokens,
    lengths that make no sense: -1 where there is no block, nothing out of
    range, everything else as usual."""
    seq, new = [40, 5, 100, -3, 33, 16], [40, 9, 30, 4, 1, -2]
    tables = np.full((6, 3), -1, np.int32)
    tables[2, :3] = [9, 8, 7]
    tables[4, :2] = [5, -1]
    tables[5, 0] = 3
    for free, num in ([], 90), ([11, 12], 90), ([11, 12, 13, 14, 15, 16, 17], 30):
        free = np.array(free, np.int32)
        want = ref.block_tables(seq, new, tables, free, 16, num)
        wide = torch.full((6, 8), 77, dtype=torch.int32, device="cuda")  # rows with a stride
        wide[:, :3] = torch.from_numpy(tables)
        slots, cu, taken = kv4.block_tables(i32(seq), i32(new), wide[:, :3],
                                            torch.from_numpy(free).cuda(), 16, num)
        assert np.array_equal(wide[:, :3].cpu().numpy(), want[0])
        assert bool((wide[:, 3:] == 77).all())
        assert np.array_equal(slots.cpu().numpy(), want[1])
        assert np.array_equal(cu.cpu().numpy(), want[2]) and taken.tolist() == [want[3]]


def test_block_tables_nothing(kv4):
    slots, cu, taken = kv4.block_tables(i32([]), i32([]), i32([]).view(0, 4), i32([]), 16, 5)
    assert slots.tolist() == [-1] * 5 and cu.tolist() == [0] and taken.tolist() == [0]
    slots, cu, taken = kv4.block_tables(i32([3]), i32([0]), i32([[2]]), i32([]), 16, 0)
    assert slots.numel() == 0 and cu.tolist() == [0, 0] and taken.tolist() == [0]


# ------------------------------------------------------------ append, read

def _store(kv4, x, levels, bs, slots, nb, dtype):
    """Append x as keys and reversed x as values; -> cache."""
    heads, D = x[0].shape[1:]
    cache = kv4.Cache.empty(nb, bs, D, levels[0].cuda(), levels[1].cuda(), dtype)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(0xEE)
    for t in (cache.k_scales, cache.v_scales):
        t.fill_(-5.0)
    kv4.append(cache, x[0].cuda(), x[1].cuda(), slots.cuda())
    return cache


def _check_store(kv4, x, levels, bs, slots, nb, dtype):
    cache = _store(kv4, x, levels, bs, slots, nb, dtype)
    T, heads, D = x[0].shape
    ok = (slots >= 0) & (slots < nb * bs)
    got = [t.cpu() for t in kv4.read(cache, slots.cuda())]
    for i, (codes, scales) in enumerate(((cache.k_codes, cache.k_scales),
                                         (cache.v_codes, cache.v_scales))):
        code, s, val = ref.quantise(x[i], levels[i])
        blk, off = (slots[ok] // bs).long(), (slots[ok] % bs).long()
        byte = codes.cpu()[blk, :, off]
        assert np.array_equal((byte & 15).numpy(), code[ok.numpy()][..., 0::2])
        assert np.array_equal((byte >> 4).numpy(), code[ok.numpy()][..., 1::2])
        assert np.array_equal(scales.cpu()[blk, :, off].float().numpy(), s[ok.numpy()],
                              equal_nan=True)
        # a product of two 16-bit floats is exact in 64 bits: rounded once
        want = torch.from_numpy(val).to(dtype)
        want[~ok] = 0
        assert torch.equal(torch.nan_to_num(got[i], nan=7.0), torch.nan_to_num(want, nan=7.0))
        # the other slots are as they were
        free = torch.ones(nb, bs, dtype=torch.bool)
        free[blk, off] = False
        assert bool((codes.cpu().permute(0, 2, 1, 3)[free] == 0xEE).all())
        assert bool((scales.cpu().permute(0, 2, 1)[free] == -5.0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,heads,D,bs", [
    (1, 1, 64, 16), (1, 3, 128, 16), (5, 2, 256, 48), (63, 5, 128, 64), (257, 1, 64, 32),
    (1000, 2, 128, 16), (130, 17, 256, 16), (4099, 1, 64, 80)])
def test_store_and_read_back(kv4, dtype, T, heads, D, bs):
    g = torch.Generator().manual_seed(T + D)
    x = [(torch.randn(T, heads, D, generator=g)
          * torch.exp(2 * torch.randn(T, heads, 1, generator=g))).to(dtype) for _ in range(2)]
    levels = [ref.random_levels(heads, dtype, T + i) for i in (1, 2)]
    nb = -(-T // bs) + 2
    slots = torch.randperm(nb * bs, generator=g)[:T].to(torch.int32)
    slots[::7] = torch.where(torch.arange(T)[::7] % 2 == 0, -1, nb * bs)  # outside
    if T == 1:
        slots[0] = nb * bs - 1
    _check_store(kv4, x, levels, bs, slots, nb, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_store_ties_and_odd_values(kv4, dtype):
    """Elements on and next to the middle between two levels, repeated levels,
    levels closer than the rounding of a distance, zeros, subnormals,
    infinities and NaN: the definition's codes, bit for bit."""
    D = 64
    levels = torch.stack([
        torch.linspace(-1, 1, 16).flip(0), torch.arange(16) / 8 - 1,
        torch.tensor([0.5, -0.5] * 8), torch.zeros(16),
        torch.tensor([0.0, 1e-7, -1e-7, 2e-7, 1, -1, 0.25, 0.25, -0.25, 3e-8, -0.0, 0.75, 0.5,
                      -0.75, 100.0, -100.0]),
        torch.tensor([2.0 ** -i for i in range(8)] + [-(2.0 ** -i) for i in range(8)])]).to(dtype)
    H = levels.shape[0]
    g = torch.Generator().manual_seed(5)
    # a vector whose scale is exactly 1 holds y = x: all middles are hit
    grid = torch.arange(-256, 257) / 256.0
    pick = grid[torch.randint(0, 513, (700, H, D), generator=g)]
    pick[..., 0] = 1.0
    tiny = torch.randn(40, H, D, generator=g) * 2.0 ** -24
    tiny[:20] *= 2.0 ** -115  # below 2^-126 in bf16, 0 in fp16
    odd = torch.randn(30, H, D, generator=g)
    odd[0] = 0
    odd[1, :, 3] = math.inf
    odd[2, :, 5] = -math.inf
    odd[3, :, 7] = math.nan
    odd[4, :, 7], odd[4, :, 9] = math.nan, math.inf
    odd[5] = -0.0
    x = torch.cat([pick, tiny, odd]).to(dtype)
    slots = torch.randperm(1024, generator=g)[:x.shape[0]].to(torch.int32)
    _check_store(kv4, [x, x.flip(0)], [levels, levels.flip(0)], 32, slots, 32, dtype)


def test_store_strided_rows(kv4):
    """Keys and values sliced from a fused projection, heads before tokens,
    rows that are not 16-byte aligned, and what lies at skipped tokens."""
    T, H, D = 50, 3, 64
    g = torch.Generator().manual_seed(1)
    x = torch.randn(T, 4 * H, D, generator=g).to(BF16)
    levels = [ref.random_levels(H, BF16, i) for i in (1, 2)]
    slots = torch.randperm(96, generator=g)[:T].to(torch.int32)
    want = _store(kv4, [x[:, H:2 * H].contiguous(), x[:, 2 * H:3 * H].contiguous()], levels, 16,
                  slots, 6, BF16)
    dev = x.cuda()
    odd = torch.zeros(T * H * D + 1, dtype=BF16, device="cuda")[1:].view(T, H, D)
    odd.copy_(dev[:, 2 * H:3 * H])
    by_head = dev[:, H:2 * H].transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(T, H, 2 * D, dtype=BF16, device="cuda")
    wide[..., ::2] = dev[:, H:2 * H]
    for k, v in ((dev[:, H:2 * H], dev[:, 2 * H:3 * H]), (by_head, odd), (wide[..., ::2], odd)):
        got = kv4.Cache.empty(6, 16, D, levels[0].cuda(), levels[1].cuda(), BF16)
        kv4.append(got, k, v, slots.cuda())
        a, b = kv4.read(got, slots.cuda()), kv4.read(want, slots.cuda())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    kv4.append(got, dev[:0, :H], dev[:0, :H], slots[:0].cuda())
    assert kv4.read(got, slots[:0].cuda())[0].shape == (0, H, D)


def test_store_past_32_bits(kv4):
    """Codes beyond 4 GiB and rows beyond 2^31 elements into the cache."""
    H, D, bs, nb = 16, 256, 128, 18000
    lv = [ref.random_levels(H, F16, i) for i in (1, 2)]
    cache = kv4.Cache.empty(nb, bs, D, lv[0].cuda(), lv[1].cuda(), F16)
    assert cache.k_codes.numel() > 2 ** 32
    g = torch.Generator().manual_seed(2)
    x = torch.randn(40, H, D, generator=g).to(F16)
    blocks = [nb - 1, 3, nb - 2]
    slots = torch.tensor([blocks[t // 16] * bs + t % 16 for t in range(40)], dtype=torch.int32)
    kv4.append(cache, x.cuda(), x.flip(0).cuda(), slots.cuda())
    k, v = kv4.read(cache, slots.cuda())
    for got, src, l in ((k, x, lv[0]), (v, x.flip(0), lv[1])):
        assert torch.equal(got.cpu(), torch.from_numpy(ref.quantise(src, l)[2]).to(F16))
    # the same vectors in a small cache: the same attention, bit for bit
    small = kv4.Cache.empty(3, bs, D, lv[0].cuda(), lv[1].cuda(), F16)
    near = torch.tensor([t // 16 * bs + t % 16 for t in range(40)], dtype=torch.int32)
    kv4.append(small, x.cuda(), x.flip(0).cuda(), near.cuda())
    q = torch.randn(3, 2 * H, D, generator=g).to(F16).cuda()
    far = kv4.attend(q, cache, i32([[b] for b in blocks]), i32([16, 16, 8]))
    assert torch.equal(far, kv4.attend(q, small, i32([[0], [1], [2]]), i32([16, 16, 8])))


# ------------------------------------------------------------ attention

def _setup(seq, bs, heads, D, dtype, seed, spare=3, **kw):
    g = torch.Generator().manual_seed(seed)
    n = [-(-max(s, 0) // bs) for s in seq]
    cache = ref.random_cache(sum(n) + spare, heads, bs, D, dtype, seed, **kw)
    pool = torch.randperm(sum(n) + spare, generator=g).to(torch.int32)
    tables = torch.full((len(seq), max(n + [1])), 2 ** 31 - 1, dtype=torch.int32)
    at = 0
    for r in range(len(seq)):
        tables[r, :n[r]] = pool[at:at + n[r]]
        at += n[r]
    # what no request reaches holds anything
    used = torch.zeros(sum(n) + spare, bs, dtype=torch.bool)
    for r, s in enumerate(seq):
        for j in range(n[r]):
            used[tables[r, j], :min(bs, s - j * bs)] = True
    for t in cache[2:4]:
        junk = torch.tensor([math.nan, math.inf, -math.inf, 6e4])[
            torch.randint(0, 4, t.shape, generator=g)].to(dtype)
        t.copy_(torch.where(used[:, None, :], t, junk))
    return cache, tables, g


def _check_attend(kv4, cache, tables, q, seq, nq, decode=False, **kw):
    dtype, D = q.dtype, q.shape[2]
    want = ref.attend(q, cache, tables, seq, nq, causal=kw.get("causal", True),
                      sm_scale=kw.get("sm_scale"), max_seq=kw.get("max_seq"))
    dev = kv4.Cache(*(t.cuda() for t in cache))
    cu = None if decode else i32(np.concatenate([[0], np.cumsum(nq)]).tolist())
    out, lse = kv4.attend(q.cuda(), dev, tables.cuda(), i32(seq), cu, return_lse=True, **kw)
    tol, lse_tol = ref.attend_tolerances(want, D, dtype)
    err = (out.cpu().double() - want[0]).abs()
    assert bool((err <= tol).all()), f"out off by {float((err / tol).max()):.3g} of its bound"
    seen = want[1] > -math.inf
    assert torch.equal(lse.cpu() > -math.inf, seen)
    assert bool(((lse.cpu().double() - want[1]).abs()[seen] <= lse_tol[seen]).all())
    assert bool((out.cpu()[~seen] == 0).all())
    # bit for bit again, and without lse
    assert torch.equal(out, kv4.attend(q.cuda(), dev, tables.cuda(), i32(seq), cu, **kw))
    return out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads,G", [(1, 1), (2, 4), (3, 5), (1, 16), (2, 24)])
def test_decode(kv4, dtype, D, heads, G):
    """Single tokens: lengths around every tile and page border, idle rows."""
    seq = [1, 0, 15, 16, 17, 31, 32, 33, 64, 65, 127, 129, 500, 1]
    cache, tables, g = _setup(seq, 16, heads, D, dtype, 10 * D + G)
    q = (2 * torch.randn(len(seq), heads * G, D, generator=g)).to(dtype)
    _check_attend(kv4, cache, tables, q, seq, [1] * len(seq), decode=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bs", [16, 48, 64, 256])
def test_decode_long(kv4, dtype, bs):
    """Contexts that are split over workgroups, beside short ones."""
    seq = [5000, 1, 9001, 0, 700]
    cache, tables, g = _setup(seq, bs, 2, 128, dtype, bs)
    q = torch.randn(len(seq), 8, 128, generator=g).to(dtype)
    _check_attend(kv4, cache, tables, q, seq, [1] * len(seq), decode=True)
    _check_attend(kv4, cache, tables, q, seq, [1] * len(seq), decode=True, max_seq=4999)


@pytest.mark.parametrize("dtype,D,heads,G,bs", [
    (BF16, 128, 2, 4, 16), (F16, 64, 3, 1, 32), (F16, 256, 1, 8, 48), (BF16, 64, 1, 16, 128),
    (BF16, 128, 1, 7, 64), (BF16, 256, 2, 2, 16), (BF16, 128, 1, 32, 16), (F16, 64, 2, 24, 48),
    (F16, 256, 1, 16, 64), (F16, 128, 2, 33, 32), (BF16, 256, 1, 24, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_several_queries(kv4, dtype, D, heads, G, bs, causal):
    """Drafted tokens and prompts, ragged: none, one, a few and many queries,
    more queries than tokens (the first ones see nothing), rows past the
    last request."""
    seq = [70, 3, 0, 200, 33, 130, 40, 0]
    nq = [3, 3, 0, 1, 33, 90, 45, 2]
    cache, tables, g = _setup(seq, bs, heads, D, dtype, D + G)
    q = (1.5 * torch.randn(sum(nq) + 4, heads * G, D, generator=g)).to(dtype)
    _check_attend(kv4, cache, tables, q, seq, nq, causal=causal)


@pytest.mark.parametrize("dtype,D,heads,G", [(BF16, 128, 2, 4), (F16, 64, 1, 3),
                                             (F16, 256, 1, 2), (F16, 128, 1, 1)])
def test_prompts(kv4, dtype, D, heads, G):
    """Longer prompts from the first token on, and a chunk behind a prefix."""
    seq, nq = [333, 900, 64], [333, 150, 64]
    cache, tables, g = _setup(seq, 64, heads, D, dtype, 3)
    q = (1.5 * torch.randn(sum(nq), heads * G, D, generator=g)).to(dtype)
    _check_attend(kv4, cache, tables, q, seq, nq)


@pytest.mark.parametrize("dtype,D,heads,G,n", [(BF16, 128, 1, 4, 1500), (F16, 64, 2, 2, 1300),
                                              (F16, 256, 1, 2, 1200)])
def test_long_prompts(kv4, dtype, D, heads, G, n):
    """Prompts and prefixes that are cut into shares."""
    seq, nq = [n, 20, 2100], [n, 20, 300]
    cache, tables, g = _setup(seq, 32, heads, D, dtype, 5)
    q = (1.5 * torch.randn(sum(nq), heads * G, D, generator=g)).to(dtype)
    _check_attend(kv4, cache, tables, q, seq, nq)
    _check_attend(kv4, cache, tables, q, seq, nq, causal=False)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("long", [40, 2600])
def test_many_requests(kv4, ragged, long):
    """More requests than a workgroup has threads, with and without cuts."""
    rng = random.Random(long)
    R = 1100
    seq = [rng.choice([0, 1, 17, rng.randrange(40)]) for _ in range(R)]
    seq[0] = seq[700] = seq[-1] = long
    nq = [rng.choice([0, 1, 2, 3]) for _ in range(R)] if ragged else [1] * R
    nq[700] = 1
    cache, tables, g = _setup(seq, 16, 1, 64, BF16, 6)
    q = torch.randn(sum(nq), 2, 64, generator=g).to(BF16)
    _check_attend(kv4, cache, tables, q, seq, nq, decode=not ragged)


@pytest.mark.parametrize("nq", [1, 40, 300])
def test_missing_blocks_are_not_seen(kv4, nq):
    seq = [100, 60, 48]
    cache, tables, g = _setup(seq, 16, 2, 64, BF16, 4)
    tables[0, 2] = -1
    tables[0, 5] = cache[0].shape[0]
    tables[1, 0] = 2 ** 31 - 1
    tables[2] = -1  # nothing left
    q = torch.randn(3 * nq, 4, 64, generator=g).to(BF16)
    out = _check_attend(kv4, cache, tables, q, seq, [nq] * 3)
    assert bool((out[2 * nq:] == 0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq", [1, 70, 130])
def test_extreme_scores_and_scales(kv4, dtype, nq):
    """Scores far apart in both directions, scales over the type's range,
    one dominating token, all scores equal."""
    seq = [400, 300, 257, 100]
    cache, tables, g = _setup(seq, 32, 1, 128, dtype, 9)
    for name in (2, 3):
        s = cache[name]
        if name == 3:  # values from the smallest to the largest scales
            s[tables[0, :13].long()] = (2.0 ** torch.randint(
                -14, 15, (13, 1, 32), generator=g).float()).to(dtype)
        else:
            s[tables[1, :10].long()] *= 30
            s[tables[2, 3], 0, 7] = 500.0
            s[tables[3, :4].long()] = 0
    cache[3][tables[0, 12], :, 16:] = math.nan  # past the request's end
    q = (2 * torch.randn(4 * nq, 4, 128, generator=g)).to(dtype)
    _check_attend(kv4, cache, tables, q, seq, [nq] * 4)
    _check_attend(kv4, cache, tables, q, seq, [nq] * 4, sm_scale=-0.3)
    _check_attend(kv4, cache, tables, q, seq, [nq] * 4, sm_scale=0.0)


@pytest.mark.parametrize("nq", [1, 70, 240])
def test_values_that_are_not_finite_stay_where_they_are_seen(kv4, nq):
    seq = [90, 90]
    cache, tables, g = _setup(seq, 16, 1, 64, F16, 12)
    q = torch.randn(2 * nq, 2, 64, generator=g).to(F16)
    clean = _check_attend(kv4, cache, tables, q, seq, [nq] * 2)
    cache[3][tables[0, 5], 0, 4] = math.inf  # token 84
    dev = kv4.Cache(*(t.cuda() for t in cache))
    out = kv4.attend(q.cuda(), dev, tables.cuda(), i32(seq), i32([0, nq, 2 * nq]))
    sees = torch.arange(90 - nq, 90) >= 84
    assert bool((~torch.isfinite(out[:nq].cpu()[sees])).flatten(1).any(1).all())
    assert torch.equal(out[:nq].cpu()[~sees], clean[:nq].cpu()[~sees])
    assert torch.equal(out[nq:], clean[nq:])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq", [1, 240])
@pytest.mark.parametrize("where", ["key", "query"])
def test_scores_that_are_not_numbers_show(kv4, dtype, nq, where):
    """A NaN among what a row sees makes that row NaN, not 0, and no other."""
    seq = [90, 90]
    cache, tables, g = _setup(seq, 16, 1, 64, dtype, 13)
    q = torch.randn(2 * nq, 2, 64, generator=g).to(dtype)
    clean = _check_attend(kv4, cache, tables, q, seq, [nq] * 2).cpu()
    sees = torch.zeros(2 * nq, 2, dtype=torch.bool)
    if where == "key":
        cache[2][tables[0, 5], 0, 4] = math.nan  # token 84
        sees[:nq] = (torch.arange(90 - nq, 90) >= 84)[:, None]
    else:
        q[nq - 1, 1, 7] = math.nan
        sees[nq - 1, 1] = True
    dev = kv4.Cache(*(t.cuda() for t in cache))
    out, lse = kv4.attend(q.cuda(), dev, tables.cuda(), i32(seq), i32([0, nq, 2 * nq]),
                          return_lse=True)
    assert torch.equal(torch.isnan(out.cpu()).all(-1), sees)
    assert torch.equal(torch.isnan(lse.cpu()), sees)
    assert torch.equal(out.cpu()[~sees], clean[~sees])


def test_strides_streams_and_out(kv4):
    seq = [130, 77, 300]
    cache, tables, g = _setup(seq, 16, 2, 128, BF16, 6)
    dev = kv4.Cache(*(t.cuda() for t in cache))
    fused = torch.randn(3, 12, 128, generator=g).to(BF16).cuda()
    q, tb, sl = fused[:, 2:10], tables.cuda(), i32(seq)
    want = kv4.attend(q.contiguous(), dev, tb, sl)
    wide = torch.zeros(3, 64, dtype=torch.int32, device="cuda")
    wide[:, :tb.shape[1]] = tb
    assert torch.equal(want, kv4.attend(q, dev, wide[:, :tb.shape[1]], sl))
    assert torch.equal(want, kv4.attend(
        q.transpose(0, 1).contiguous().transpose(0, 1), dev, tb, sl))
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert kv4.attend(q, dev, tb, sl, out=out) is out
    side.synchronize()
    assert torch.equal(want, out)
    assert kv4.attend(q[:0], dev, tb[:0], sl[:0]).shape == (0, 8, 128)
    assert bool((kv4.attend(q, dev, tb, sl, max_seq=0) == 0).all())
    none = kv4.attend(q, dev, tb[:0], sl[:0], i32([0]))  # rows of no request
    assert bool((none == 0).all())


@pytest.mark.parametrize("nq,seq", [(1, [3000, 40]), (100, [300, 120]), (250, [300, 270]),
                                    (1, [120, 700])])
def test_a_step_in_a_graph(kv4, nq, seq):
    """Tables, append, read and attention captured together and replayed with
    other lengths and inputs."""
    H, D, bs, R = 2, 64, 16, 2
    lv = [ref.random_levels(H, BF16, i).cuda() for i in (1, 2)]
    num = nq * R
    width = -(-max(seq) // bs)
    g = torch.Generator().manual_seed(0)

    def inputs(cut):
        s = [n - cut for n in seq]
        held = [-(-(n - nq) // bs) for n in s]
        tb = torch.full((R, width), -1, dtype=torch.int32)
        order = torch.randperm(R * width, generator=g).to(torch.int32)
        at = 0
        for r in range(R):
            tb[r, :held[r]] = order[at:at + held[r]]
            at += held[r]
        free = torch.full((R * width,), -1, dtype=torch.int32)
        free[:R * width - at] = order[at:]
        return [torch.tensor(s, dtype=torch.int32).cuda(), tb.cuda(), free.cuda(),
                *(torch.randn(num, n, D, generator=g).to(BF16).cuda() for n in (4 * H, H, H))]

    def step(cache, s, tb, free, q, k, v):
        slots, cu, taken = kv4.block_tables(s, new, tb, free, bs, num)
        kv4.append(cache, k, v, slots)
        return (slots, cu, taken, *kv4.read(cache, slots), kv4.attend(q, cache, tb, s, cu))

    def fresh():
        codes = [c.cuda() for c in ref.random_cache(R * width, H, bs, D, BF16, 7)[:4]]
        return kv4.Cache(*codes, *lv)

    new = i32([nq] * R)
    static = inputs(0)
    cache = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, *static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(cache, *static)
    for cut in (0, 3, 17):
        cur = inputs(cut)
        want = step(fresh(), *[t.clone() for t in cur])
        for a, b in zip(static, cur):
            a.copy_(b)
        base = fresh()
        for n in ("k_codes", "v_codes", "k_scales", "v_scales"):
            getattr(cache, n).copy_(getattr(base, n))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


# ------------------------------------------------------------ levels

def test_learned_levels(kv4):
    """The levels are the loop's centroids, and better than even steps."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(400, 3, 64, generator=g)
    lv = kv4.learn_levels(x.to(BF16).cuda())
    assert lv.shape == (3, 16) and lv.dtype == torch.float32
    assert bool((lv.diff(dim=1) > 0).all()) and bool((lv.abs() <= 1).all())
    even = torch.linspace(-1, 1, 16).expand(3, 16)
    err = [np.mean((ref.quantise(x.to(BF16), l.to(BF16))[2] - x.double().numpy()) ** 2)
           for l in (lv.cpu(), even)]
    assert err[0] < 0.8 * err[1]


# ------------------------------------------------------------ refusals

def test_refusals(kv4):
    lv = ref.random_levels(2, BF16, 0).cuda()
    c = kv4.Cache.empty(4, 16, 64, lv, lv, BF16)
    x = torch.zeros(3, 2, 64, dtype=BF16, device="cuda")
    s, tb = i32([1, 2, 3]), i32([[0], [1], [2]])
    bad = [
        lambda: kv4.append(c, x.half(), x, s), lambda: kv4.append(c, x[:, :1], x, s),
        lambda: kv4.append(c, x, x[:2], s), lambda: kv4.append(c, x, x, s.long()),
        lambda: kv4.append(c, x[..., :32], x, s), lambda: kv4.read(c, s.view(1, 3)),
        lambda: kv4.attend(x[:, :1], c, tb, s), lambda: kv4.attend(x, c, tb[:2], s),
        lambda: kv4.attend(x, c, tb, s[:2]), lambda: kv4.attend(x, c, tb, s, i32([0, 3])),
        lambda: kv4.attend(x, c, tb, s, max_seq=17), lambda: kv4.attend(x, c, tb.long(), s),
        lambda: kv4.attend(x, c, tb, s, out=x.half()),
        lambda: kv4.attend(x, c, tb, s, out=torch.empty_like(x)[:, :, :32]),
        lambda: kv4.block_tables(s, s[:2], tb, s, 16, 3),
        lambda: kv4.block_tables(s, s, tb, s, 0, 3),
        lambda: kv4.block_tables(s, s, tb, s, 16, -1),
        lambda: kv4.block_tables(s, s, tb.t(), s, 16, 3),
        lambda: kv4.Cache.empty(4, 16, 96, lv, lv, BF16),
        lambda: kv4.Cache.empty(4, 24, 64, lv, lv, BF16),
        lambda: kv4.Cache.empty(4, 16, 64, lv, lv, torch.float32),
        lambda: kv4.Cache.empty(4, 16, 64, lv, lv[:1], BF16),
        lambda: kv4.Cache(c.k_codes, c.v_codes, c.k_scales, c.v_scales.half(), lv, lv),
        lambda: kv4.Cache(c.k_codes, c.v_codes[:, :, ::2], c.k_scales, c.v_scales, lv, lv),
        lambda: kv4.learn_levels(x[0]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was accepted")
    for call in (lambda: kv4.append(c, x.cpu(), x, s), lambda: kv4.read(c, s.cpu()),
                 lambda: kv4.attend(x, c, tb.cpu(), s), lambda: kv4.attend(x, c, tb, s.cpu()),
                 lambda: kv4.block_tables(s.cpu(), s, tb, s, 16, 3)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------ together

def test_serving_example():
    """Learned levels, tables, append and attention in a loop.  Sixteen levels
    leave a normal vector's elements about a tenth off (their quantisation
    error is 1% of the variance), and attention averages it."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "flash-kmeans-cuda_amd", "examples", "kv4_serving.py")
    spec = importlib.util.spec_from_file_location("kv4_serving", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(steps=3) < 0.2
