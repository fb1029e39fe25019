"""Pages of the 4-bit cache on the GPU against references that walk the rows:
free lists, forks, compaction, copies, all bit for bit, and a run of them with
append and attend."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

import kv4_pages_ref as pages
import kv4_ref as ref
from test_gpu_kv4 import BF16, F16, i32

pytestmark = pytest.mark.gpu

NAMES = ("k_codes", "v_codes", "k_scales", "v_scales")


@pytest.fixture(scope="module")
def kv4():
    from flash_kmeans_cuda import kv4
    return kv4


def _rows(R, width, bs, num_blocks, seed, odd=0.1):
    """Tables that share blocks, with lengths of every kind and, for a share
    `odd` of the entries, no block at all."""
    rng = random.Random(seed)
    tables = np.array([[rng.randrange(num_blocks) if num_blocks and rng.random() >= odd else
                        rng.choice([-1, -7, num_blocks, 2 ** 31 - 1, -2 ** 31])
                        for _ in range(width)] for _ in range(R)], np.int64)
    tables = tables.reshape(R, width).astype(np.int32)
    cap = width * bs
    seq = [rng.choice([0, 1, bs, bs + 1, cap, cap + 5, 2 ** 31 - 1, -4, rng.randrange(cap + 1),
                       rng.randrange(cap + 1), rng.randrange(cap + 1)]) for _ in range(R)]
    return tables, np.array(seq, np.int32).reshape(R)


def _strided(tables):
    """The same tables as a slice of wider rows."""
    wide = torch.full((tables.shape[0], tables.shape[1] + 5), 3, dtype=torch.int32, device="cuda")
    wide[:, :tables.shape[1]] = torch.from_numpy(tables)
    return wide[:, :tables.shape[1]]


SIZES = [(1, 1, 16, 1), (1, 1, 16, 0), (3, 0, 16, 9), (0, 4, 16, 9), (5, 7, 16, 40),
         (64, 33, 32, 4096), (7, 1025, 16, 4097), (300, 70, 48, 9001), (2, 3000, 128, 70000),
         (900, 3, 16, 1 << 20), (17, 129, 64, 262143), (1500, 128, 1, 300000)]


@pytest.mark.parametrize("R,width,bs,num_blocks", SIZES)
def test_free_blocks(kv4, R, width, bs, num_blocks):
    tables, seq = _rows(R, width, bs, num_blocks, R + width)
    want, count = pages.free_blocks(tables, seq, bs, num_blocks)
    for t in torch.from_numpy(tables).cuda(), _strided(tables):
        free, n = kv4.free_blocks(t, i32(seq.tolist()), bs, num_blocks)
        assert n.tolist() == [count]
        assert np.array_equal(free.cpu().numpy(), want)


def _cache(kv4, nb, heads, bs, D, dtype, seed):
    host = ref.random_cache(nb, heads, bs, D, dtype, seed)
    return host, kv4.Cache(*(t.cuda() for t in host))


def _same(cache, host):
    for name, t in zip(NAMES, host):
        got = getattr(cache, name).cpu()
        assert torch.equal(got.view(torch.uint8), t.view(torch.uint8)), name


def _check_fork(kv4, R, width, bs, nb, F, seed, free=None, heads=2, D=64, dtype=F16, odd=0.1,
                parents=None, tables=None, seq=None):
    rng = random.Random(seed)
    if tables is None:
        tables, seq = _rows(R, width, bs, nb - F, seed, odd)
    if parents is None:
        parents = [rng.choice([rng.randrange(R), 0, rng.randrange(-2, R + 2)]) for _ in range(F)]
    if free is None:
        free = list(range(nb - F, nb))
        rng.shuffle(free)
    host, cache = _cache(kv4, nb, heads, bs, D, dtype, seed)
    want, want_seq, taken, copies = pages.fork(tables, seq, parents, free, bs, nb)
    t = _strided(tables)
    new, new_seq, n = kv4.fork(cache, t, i32(seq.tolist()), i32(parents), i32(free))
    assert n.tolist() == [taken]
    assert np.array_equal(new_seq.cpu().numpy(), want_seq)
    assert np.array_equal(new.cpu().numpy(), want)
    assert np.array_equal(t.cpu().numpy(), tables)
    for a, b in copies:
        for x in host[:4]:
            x[b] = x[a]
    _same(cache, host)
    return new, new_seq


@pytest.mark.parametrize("R,width,bs,nb,F", [
    (1, 1, 16, 4, 2), (1, 5, 16, 40, 7), (8, 9, 32, 200, 64), (40, 3, 48, 300, 41),
    (3, 300, 16, 900, 30), (600, 4, 16, 4000, 1500), (5, 2, 128, 1100, 1025)])
def test_fork(kv4, R, width, bs, nb, F):
    _check_fork(kv4, R, width, bs, nb, F, F)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,D,bs", [(1, 64, 16), (3, 128, 48), (17, 256, 128), (5, 64, 1024)])
def test_fork_of_every_block_size(kv4, dtype, heads, D, bs):
    """Copies of blocks that are smaller and larger than what a workgroup
    moves at a time."""
    _check_fork(kv4, 4, 3, bs, 30, 9, D + bs, heads=heads, D=D, dtype=dtype)


def test_forks_of_huge_blocks(kv4):
    """More pieces of blocks than a launch has workgroups of them."""
    bs, nb, F = 1 << 18, 4, 1000
    codes = [torch.randint(0, 256, (nb, 8, bs, 32), dtype=torch.uint8, device="cuda")
             for _ in range(2)]
    scales = [torch.rand(nb, 8, bs, device="cuda").to(F16) for _ in range(2)]
    levels = [torch.rand(8, 16, device="cuda").to(F16) for _ in range(2)]
    cache = kv4.Cache(*codes, *scales, *levels)
    before = [t.clone() for t in codes + scales]
    tables, seq = np.array([[1, 0]], np.int32), np.array([bs + 5], np.int32)
    want, want_seq, taken, copies = pages.fork(tables, seq, [0] * F, [3], bs, nb)
    new, new_seq, n = kv4.fork(cache, i32(tables.tolist()), i32(seq.tolist()), i32([0] * F),
                               i32([3]))
    assert n.tolist() == [taken] and copies == [(0, 3)]
    assert np.array_equal(new.cpu().numpy(), want)
    assert np.array_equal(new_seq.cpu().numpy(), want_seq)
    for t, old in zip(codes + scales, before):
        assert torch.equal(t[:3], old[:3]) and torch.equal(t[3], old[0])


def test_pages_of_nothing(kv4):
    """Tables without rows or without entries, an empty cache, parents that are
    no rows."""
    for nb in 0, 20:
        _, cache = _cache(kv4, nb, 2, 16, 64, F16, 3)
        _, into = _cache(kv4, 5, 2, 16, 64, F16, 4)
        for tables, seq in (([], []), ([[]] * 3, [40, 0, 5]), ([[1, 2], [3, -1]], [0, -9])):
            width = 2 if len(tables) == 2 else 0
            t = torch.tensor(tables, dtype=torch.int32, device="cuda").reshape(len(seq), width)
            free, count = kv4.free_blocks(t, i32(seq), 16, nb)
            assert free.tolist() == list(range(nb)) and count.tolist() == [nb]
            new, new_seq, taken = kv4.fork(cache, t, i32(seq), i32([-1, 5, 0]), i32([9]))
            assert new.shape == (3, width) and bool((new == -1).all()) and taken.tolist() == [0]
            assert new_seq.tolist() == [0, 0, max(seq[0], 0) if seq else 0]
            new, used = kv4.compact(cache, t, i32(seq), into)
            assert new.shape == t.shape and bool((new == -1).all()) and used.tolist() == [0]
        kv4.copy_blocks(cache, i32([0, 1]), into, i32([-1, 7]))
    torch.cuda.synchronize()


def test_fork_keeps_and_copies(kv4):
    """Two children of one parent; a parent that two rows share the last block
    of; one whose last block is another's whole one; no child at all."""
    tables = np.array([[0, 1, 2], [3, 4, -1], [5, 4, -1], [6, 1, -1], [1, -1, -1]], np.int32)
    seq = np.array([40, 20, 30, 32, 7], np.int32)
    kw = dict(R=5, width=3, bs=16, nb=20, seed=1, tables=tables, seq=seq)
    new, _ = _check_fork(kv4, F=4, parents=[0, 0, 1, 2], free=[10, 11, 12, 13], **kw)
    assert new.tolist() == [[0, 1, 2], [0, 1, 10], [3, 4, -1], [5, 11, -1]]
    new, _ = _check_fork(kv4, F=2, parents=[4, 0], free=[10], **kw)  # 1 is whole in row 0
    assert new.tolist() == [[10, -1, -1], [0, 1, 2]]
    new, _ = _check_fork(kv4, F=2, parents=[4, 1], free=[10], **kw)  # 0 has no child
    assert new.tolist() == [[1, -1, -1], [3, 4, -1]]
    new, n = _check_fork(kv4, F=0, parents=[], free=[], **kw)
    assert new.shape == (0, 3) and n.shape == (0,)


def test_fork_with_too_few_free_blocks(kv4):
    tables, seq = np.array([[2, 3]], np.int32), np.array([20], np.int32)
    kw = dict(R=1, width=2, bs=16, nb=9, seed=2, tables=tables, seq=seq)
    for free in [], [7], [7, -1, 8], [-1, 9, 2 ** 31 - 1, 5]:
        _check_fork(kv4, F=6, parents=[0] * 6, free=free, **kw)


def _check_compact(kv4, R, width, bs, nb, into_blocks, seed, heads=2, D=64, dtype=F16, odd=0.1):
    tables, seq = _rows(R, width, bs, nb, seed, odd)
    host, cache = _cache(kv4, nb, heads, bs, D, dtype, seed)
    kept, into = _cache(kv4, into_blocks, heads, bs, D, dtype, seed + 1)
    want, used = pages.compact(tables, seq, bs, nb, into_blocks)
    t = _strided(tables)
    new, n = kv4.compact(cache, t, i32(seq.tolist()), into)
    assert n.tolist() == [len(used)]
    assert np.array_equal(new.cpu().numpy(), want)
    fits = used[:into_blocks]
    for x, y in zip(kept[:4], host[:4]):
        x[:len(fits)] = y[fits]
    _same(into, kept)
    _same(cache, host)


@pytest.mark.parametrize("R,width,bs,nb,into_blocks", [
    (1, 1, 16, 1, 1), (4, 5, 16, 30, 30), (4, 5, 16, 30, 3), (9, 40, 32, 5000, 400),
    (3, 2, 16, 0, 4), (3, 2, 16, 8, 0), (0, 2, 16, 8, 4), (70, 30, 16, 9000, 9000),
    (2, 1100, 16, 4500, 2300)])
def test_compact(kv4, R, width, bs, nb, into_blocks):
    _check_compact(kv4, R, width, bs, nb, into_blocks, R + nb)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,D,bs", [(1, 64, 16), (3, 128, 48), (17, 256, 128), (5, 64, 1024)])
def test_compact_of_every_block_size(kv4, dtype, heads, D, bs):
    _check_compact(kv4, 5, 4, bs, 20, 20, D + bs, heads=heads, D=D, dtype=dtype)


@pytest.mark.parametrize("n", [0, 1, 33, 500])
@pytest.mark.parametrize("heads,D,bs,dtype", [(1, 64, 16, F16), (5, 128, 48, BF16),
                                              (16, 256, 128, F16)])
def test_copy_blocks(kv4, n, heads, D, bs, dtype):
    g = torch.Generator().manual_seed(n)
    a, b = max(n // 2, 2), n + 3  # (a block may be copied twice)
    host, cache = _cache(kv4, a, heads, bs, D, dtype, n)
    kept, into = _cache(kv4, b, heads, bs, D, dtype, n + 1)
    src = torch.randint(0, a, (n,), generator=g).to(torch.int32)
    dst = torch.randperm(b, generator=g)[:n].to(torch.int32)
    src[::5] = torch.tensor([-1, a, 2 ** 31 - 1, -2 ** 31])[torch.arange(n)[::5] % 4].to(
        torch.int32)
    dst[3::7] = torch.tensor([b, -1])[torch.arange(n)[3::7] % 2].to(torch.int32)
    kv4.copy_blocks(cache, src.cuda(), into, dst.cuda())
    for i, j in zip(src.tolist(), dst.tolist()):
        if 0 <= i < a and 0 <= j < b:
            for x, y in zip(kept[:4], host[:4]):
                x[j] = y[i]
    _same(into, kept)
    _same(cache, host)


def test_copy_blocks_within_a_cache(kv4):
    host, cache = _cache(kv4, 9, 3, 32, 128, BF16, 1)
    kv4.copy_blocks(cache, i32([0, 4, 0]), cache, i32([8, 2, 3]))
    for x in host[:4]:
        x[[8, 2, 3]] = x[[0, 4, 0]]
    _same(cache, host)


def test_copies_past_32_bits(kv4):
    """Blocks beyond 4 GiB of codes, into and out of them."""
    H, D, bs, nb = 16, 256, 128, 18000
    lv = [ref.random_levels(H, F16, i).cuda() for i in (1, 2)]
    cache = kv4.Cache.empty(nb, bs, D, *lv, F16)
    assert cache.k_codes.numel() > 2 ** 32
    host, small = _cache(kv4, 3, H, bs, D, F16, 5)
    kv4.copy_blocks(small, i32([0, 1, 2]), cache, i32([nb - 1, 3, nb - 2]))
    tables = i32([[nb - 1, 3], [nb - 1, nb - 2]])
    new, seq, taken = kv4.fork(cache, tables, i32([2 * bs, 2 * bs - 5]), i32([0, 1, 1]),
                               i32([nb - 3]))
    assert new.tolist() == [[nb - 1, 3], [nb - 1, nb - 2], [nb - 1, nb - 3]]
    assert taken.tolist() == [1]
    back = kv4.Cache(*(torch.zeros_like(t).cuda() for t in host[:4]),
                     *(t.cuda() for t in host[4:]))
    kv4.copy_blocks(cache, i32([nb - 1, 3, nb - 3]), back, i32([0, 1, 2]))
    _same(back, host)
    into = kv4.Cache(*(torch.zeros_like(t).cuda() for t in host[:4]),
                     *(t.cuda() for t in host[4:]))
    moved, used = kv4.compact(cache, tables, i32([2 * bs, 2 * bs]), into)
    assert moved.tolist() == [[2, 0], [2, 1]] and used.tolist() == [3]
    _same(into, [t[[1, 2, 0]] for t in host[:4]])


def test_many_children_and_rows(kv4):
    """More children than one workgroup counts at a time, all of one parent."""
    tables, seq = np.array([[0, 1, 2, 3]], np.int32), np.array([60], np.int32)
    _check_fork(kv4, 1, 4, 16, 5000, 4990, 3, tables=tables, seq=seq, parents=[0] * 4990,
                free=list(range(4999, 9, -1)), heads=1)


# ------------------------------------------------------------ a run of them

class _Loop:
    """A server's step over one cache: free list, tables, append, attention of a
    model that caps its scores and looks back over a window."""

    def __init__(self, kv4, cache, requests, width):
        self.kv4, self.cache = kv4, cache
        self.tables = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
        self.seq = torch.zeros(requests, dtype=torch.int32, device="cuda")

    def free(self):
        c = self.cache
        return self.kv4.free_blocks(self.tables, self.seq, c.block_size, c.num_blocks)[0]

    def step(self, new, q, k, v):
        free = self.free()
        self.seq = self.seq + new
        slots, cu, _ = self.kv4.block_tables(self.seq, new, self.tables, free,
                                             self.cache.block_size, len(k))
        self.kv4.append(self.cache, k, v, slots)
        return self.kv4.attend(q, self.cache, self.tables, self.seq, cu, return_lse=True,
                               softcap=30.0, window=50)

    def fork(self, parents):
        self.tables, self.seq, _ = self.kv4.fork(self.cache, self.tables, self.seq, i32(parents),
                                                 self.free())


@pytest.mark.parametrize("dtype,D,bs", [(BF16, 128, 16), (F16, 64, 48)])
def test_a_server_that_forks_and_moves(kv4, dtype, D, bs):
    """Prompts, samples forked from them, a step, beams that are dropped and
    doubled, rows cut back into shared blocks, another step, a move into another
    cache, a last step: at every step the answer is that of a cache that is
    filled anew with each row's own tokens, bit for bit."""
    H, G = 2, 3
    g = torch.Generator(device="cuda").manual_seed(D)
    levels = [ref.random_levels(H, dtype, i).cuda() for i in (1, 2)]

    def vectors(n, heads=H):
        return torch.randn(n, heads, D, generator=g, device="cuda").to(dtype)

    loop = _Loop(kv4, kv4.Cache.empty(60, bs, D, *levels, dtype), 3, 12)
    rows = [(vectors(0), vectors(0)) for _ in range(3)]  # what each row holds

    def step(new):
        k, v, q = vectors(sum(new)), vectors(sum(new)), vectors(sum(new), H * G)
        got = loop.step(i32(new), q, k, v)
        for r, (a, b) in enumerate(zip(k.split(new), v.split(new))):
            rows[r] = torch.cat([rows[r][0], a]), torch.cat([rows[r][1], b])
        check = _Loop(kv4, kv4.Cache.empty(150, bs, D, *levels, dtype), len(rows), 12)
        n = i32([len(r[0]) for r in rows])
        check.step(n, vectors(int(n.sum()), H * G), torch.cat([r[0] for r in rows]),
                   torch.cat([r[1] for r in rows]))
        cu = i32(np.cumsum([0] + new).tolist())
        want = kv4.attend(q, check.cache, check.tables, n, cu, return_lse=True, softcap=30.0,
                          window=50)
        assert torch.equal(loop.seq, n)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        mine = kv4.read(loop.cache, _slots(loop, rows))
        theirs = kv4.read(check.cache, _slots(check, rows))
        assert torch.equal(mine[0], theirs[0]) and torch.equal(mine[1], theirs[1])

    def _slots(lp, rows):
        t = [lp.tables[r].long().repeat_interleave(bs) * bs + torch.arange(
            12 * bs, device="cuda") % bs for r in range(len(rows))]
        return torch.cat([x[:len(r[0])] for x, r in zip(t, rows)]).to(torch.int32)

    def fork(parents):
        loop.fork(parents)
        rows[:] = [rows[p] if p >= 0 else (vectors(0), vectors(0)) for p in parents]

    step([3 * bs + 5, 2 * bs, 7])
    fork([0, 0, 1, 1, 2, 2, 2, -1])
    step([1] * 8)
    fork([3, 3, 0, 1, 1, 6, 7, 5])
    step([2, 1, bs + 3, 1, 1, 4, 5, 1])
    # cut every row back, some into blocks that others hold as well
    cut = [min(len(r[0]), n) for r, n in zip(rows, (bs + 3, 2 * bs + 1, bs, 1, 3 * bs, 0, 2, 9))]
    rows[:] = [(k[:n], v[:n]) for (k, v), n in zip(rows, cut)]
    loop.seq = i32(cut)
    fork(list(range(8)))
    step([1, 2, 3, 4, 5, 6, 7, 8])
    into = kv4.Cache.empty(70, bs, D, *levels, dtype)
    loop.tables, used = kv4.compact(loop.cache, loop.tables, loop.seq, into)
    free, count = kv4.free_blocks(loop.tables, loop.seq, bs, 70)
    assert int(used) + int(count) == 70
    assert free[:int(count)].tolist() == list(range(int(used), 70))
    loop.cache = into
    step([1] * 8)


def test_captured_pages(kv4):
    """Captured once, replayed on other tables, with eager calls in between;
    two graphs of one pool."""
    host, cache = _cache(kv4, 40, 2, 16, 64, F16, 3)
    into = kv4.Cache.empty(40, 16, 64, cache.k_levels, cache.v_levels, F16)
    tables, seq = torch.zeros(6, 5, dtype=torch.int32, device="cuda"), i32([0] * 6)
    parents = i32([0, 0, 1, 2, 5, 5])

    def work():
        free, count = kv4.free_blocks(tables, seq, 16, 40)
        new, n, taken = kv4.fork(cache, tables, seq, parents, free)
        moved, used = kv4.compact(cache, new, n, into)
        return free, count, new, n, taken, moved, used

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
        t, s = _rows(6, 5, 16, 30, i, odd=0)
        s = np.clip(s, 0, 80).astype(np.int32)
        tables.copy_(torch.from_numpy(t))
        seq.copy_(torch.from_numpy(s))
        eager = [x.clone() for x in work()]
        moved = [getattr(into, n).clone() for n in NAMES]
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, eager):
                assert torch.equal(a, b)
            for n, m in zip(NAMES, moved):
                assert torch.equal(getattr(into, n)[:int(eager[-1])], m[:int(eager[-1])])


def test_pages_on_another_stream(kv4):
    tables, seq = _rows(200, 60, 16, 5000, 9)
    want, count = pages.free_blocks(tables, seq, 16, 5000)
    t, s = torch.from_numpy(tables).cuda(), i32(seq.tolist())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        free, n = kv4.free_blocks(t, s, 16, 5000)
    side.synchronize()
    assert np.array_equal(free.cpu().numpy(), want) and n.tolist() == [count]


def test_refusals(kv4):
    _, cache = _cache(kv4, 4, 2, 16, 64, F16, 1)
    _, other = _cache(kv4, 4, 2, 32, 64, F16, 1)
    t, s, f = i32([[0, 1]]), i32([3]), i32([2])
    with pytest.raises(RuntimeError, match="share memory"):
        kv4.compact(cache, t, s, cache)
    with pytest.raises(RuntimeError, match="differ"):
        kv4.compact(cache, t, s, other)
    with pytest.raises(RuntimeError, match="differ"):
        kv4.copy_blocks(cache, f, other, f)
    with pytest.raises(RuntimeError, match="one length"):
        kv4.copy_blocks(cache, f, cache, i32([1, 2]))
    with pytest.raises(RuntimeError, match="int32"):
        kv4.fork(cache, t, s, f.long(), f)
    with pytest.raises(RuntimeError, match="dense rows"):
        kv4.fork(cache, t, i32([3, 4]), f, f)
    with pytest.raises(RuntimeError, match="dense rows"):
        kv4.free_blocks(i32([[0, 1], [2, 3]]).t(), i32([1, 1]), 16, 4)
    with pytest.raises(RuntimeError, match="negative"):
        kv4.free_blocks(t, s, 16, -1)
    with pytest.raises(RuntimeError, match="range"):
        kv4.free_blocks(t, s, 0, 4)
    with pytest.raises(ValueError):
        kv4.free_blocks(t.cpu(), s.cpu(), 16, 4)
    with pytest.raises(ValueError):
        kv4.fork(cache, t, s, f.cpu(), f)
