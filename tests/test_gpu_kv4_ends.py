"""The 4-bit cache's operators at the ends of their ranges: large score
scales, steps padded far past their queries, rows of one token or head, slots
that no cache has, the cache's fixed tensors, gradients."""

from __future__ import annotations

import math

import pytest
import torch

import kv4_ref as ref
from test_gpu_kv4 import BF16, F16, _check_attend, _setup, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv4():
    from flash_kmeans_cuda import kv4
    return kv4


# ------------------------------------------------------------ score scales

SCALES = [1.0, -1.0, 8.0, 0.7]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sm_scale", SCALES)
def test_large_score_scales_of_a_few_queries(kv4, dtype, D, sm_scale):
    """Scales above ln 2, where a masked score's stand-in times the scale
    leaves fp32: tiles past an earlier query's last token, queries that see
    nothing beside some that do, 32 tokens in missing blocks, idle rows."""
    seq, nq = [100, 3, 33, 0, 70, 290], [7, 5, 1, 1, 2, 3]
    cache, tables, g = _setup(seq, 16, 2, D, dtype, D)
    tables[4, 2:4] = -1
    tables[5, 0:2] = cache[0].shape[0]
    q = (1.5 * torch.randn(sum(nq) + 3, 6, D, generator=g)).to(dtype)
    _check_attend(kv4, cache, tables, q, seq, nq, sm_scale=sm_scale)
    _check_attend(kv4, cache, tables, q, seq, nq, sm_scale=sm_scale, causal=False)
    one = [1] * len(seq)
    _check_attend(kv4, cache, tables, q[:len(seq)], seq, one, decode=True, sm_scale=sm_scale)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sm_scale", SCALES[:2])
def test_large_score_scales_of_prompts(kv4, dtype, D, sm_scale):
    """The same for prompts in shares, which begin past some rows' last
    token, and for contexts cut over workgroups."""
    seq, nq = [1300, 20, 1500], [1300, 20, 300]
    cache, tables, g = _setup(seq, 32, 1, D, dtype, D + 1)
    q = (1.5 * torch.randn(sum(nq), 2, D, generator=g)).to(dtype)
    _check_attend(kv4, cache, tables, q, seq, nq, sm_scale=sm_scale)
    seq, nq = [6000, 90, 2500], [7, 5, 1]
    cache, tables, g = _setup(seq, 16, 1, D, dtype, D + 2)
    tables[2, 4:100] = -1
    q = (1.5 * torch.randn(sum(nq), 4, D, generator=g)).to(dtype)
    _check_attend(kv4, cache, tables, q, seq, nq, sm_scale=sm_scale)


@pytest.mark.parametrize("nq", [6, 240])
def test_large_score_scales_of_missing_blocks(kv4, nq):
    seq = [100, 60, 48]
    cache, tables, g = _setup(seq, 16, 2, 64, BF16, 4)
    tables[0, 2:4] = -1
    tables[1, 0:2] = 2 ** 31 - 1
    tables[2] = -1  # nothing left
    q = torch.randn(3 * nq, 4, 64, generator=g).to(BF16)
    for sm_scale in 1.0, -2.5:
        out = _check_attend(kv4, cache, tables, q, seq, [nq] * 3, sm_scale=sm_scale)
        assert bool((out[2 * nq:] == 0).all())


# ------------------------------------------------------------ padded steps

@pytest.mark.parametrize("dtype,D,G", [(BF16, 128, 4), (F16, 64, 1), (F16, 256, 2)])
def test_rows_of_no_request_beside_cut_ones(kv4, dtype, D, G):
    """Steps padded to many times their queries, and requests with many more
    queries than tokens, where the work is cut into shares: those rows are 0,
    the others what they are without them."""
    seq, nq = [1300, 40, 0, 5], [300, 900, 500, 1]
    cache, tables, g = _setup(seq, 64, 2, D, dtype, 3)
    q = (1.5 * torch.randn(9000, 2 * G, D, generator=g)).to(dtype)
    out = _check_attend(kv4, cache, tables, q, seq, nq)
    assert bool((out[sum(nq):] == 0).all())


def test_a_padded_step_of_single_tokens(kv4):
    """Many requests' worth of padding behind a few single tokens."""
    seq, nq = [5000, 0, 700], [1, 1, 1]
    cache, tables, g = _setup(seq, 16, 2, 128, BF16, 3)
    q = torch.randn(700, 8, 128, generator=g).to(BF16)
    out = _check_attend(kv4, cache, tables, q, seq, nq)
    assert bool((out[3:] == 0).all())


# ------------------------------------------------------------ strides of one row

@pytest.mark.parametrize("T,H", [(1, 1), (1, 3), (5, 1)])
def test_strides_of_single_rows_do_not_matter(kv4, T, H):
    """A dimension of one entry may have any stride: one token or one head out
    of rows whose length is no multiple of eight."""
    D = 128
    g = torch.Generator().manual_seed(T + H)
    levels = [ref.random_levels(H, BF16, i).cuda() for i in (1, 2)]
    slots, tables, seq = i32(list(range(T))), i32([[0]] * T), i32(list(range(1, T + 1)))
    dense = [torch.randn(T, H, D, generator=g).to(BF16).cuda() for _ in range(3)]

    def odd(x, n):
        step = [n if T == 1 else H * D, n if H == 1 else D, 1]
        y = torch.zeros(4096, dtype=BF16, device="cuda").as_strided((T, H, D), step)
        return y.copy_(x)

    def step(q, k, v):
        cache = kv4.Cache.empty(2, 16, D, *levels, BF16)
        kv4.append(cache, k, v, slots)
        return (*kv4.read(cache, slots), kv4.attend(q, cache, tables, seq))

    want = step(*dense)
    for n in 132, 129, 4, 1:
        for a, b in zip(want, step(*(odd(x, n) for x in dense))):
            assert torch.equal(a, b)


# ------------------------------------------------------------ slots

@pytest.mark.parametrize("bs", [16, 48, 128])
def test_blocks_past_every_slot_give_no_slot(kv4, bs):
    """A block whose slots 31 bits do not hold, in a table or on the free list,
    gives -1, not another block's slots."""
    top = (2 ** 31 - 1) // bs  # the last slot of block top - 1 fits
    seq, new = [bs + 3, bs + 3, 2 * bs, 5], [3, 3, bs, 2]
    tables = torch.tensor([[0, -1], [0, -1], [0, -1], [0, -1]], dtype=torch.int32)
    tables[3, 0] = -(-2 ** 32 // bs)  # its slots would wrap around to the first ones
    free = [2 ** 31 - 1, top - 1, 2 ** 31 // bs + 1]
    tb = tables.cuda()
    slots, cu, taken = kv4.block_tables(i32(seq), i32(new), tb, i32(free), bs, sum(new))
    got = slots.tolist()
    assert got[:3] == [-1] * 3
    assert got[3:6] == [(top - 1) * bs + i for i in range(3)]
    assert got[6:] == [-1] * (bs + 2)
    assert tb[:3, 1].tolist() == free and taken.tolist() == [3]


# ------------------------------------------------------------ the cache's tensors

def test_a_cache_keeps_its_tensors(kv4):
    """The kernels go on reading the tensors a cache was made of: none of them,
    and no size, can be replaced or dropped."""
    lv = ref.random_levels(2, BF16, 0).cuda()
    c = kv4.Cache.empty(4, 16, 64, lv, lv, BF16)
    for name in ("k_codes", "v_codes", "k_scales", "v_scales", "k_levels", "v_levels",
                 "num_blocks", "heads", "block_size", "head_dim", "dtype", "device"):
        old = getattr(c, name)
        with pytest.raises(AttributeError, match=name):
            setattr(c, name, old)
        with pytest.raises(AttributeError, match=name):
            delattr(c, name)
        assert getattr(c, name) is old
    c.k_levels.copy_(-lv)  # their values are the caller's
    x = torch.randn(3, 2, 64, device="cuda").to(BF16)
    kv4.append(c, x, x, i32([0, 1, 2]))
    other = kv4.Cache.empty(4, 16, 64, -lv, lv, BF16)
    kv4.append(other, x, x, i32([0, 1, 2]))
    for a, b in zip(kv4.read(c, i32([0, 1, 2])), kv4.read(other, i32([0, 1, 2]))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("given", [F16, BF16, torch.float32])
def test_an_empty_cache_has_levels_of_its_own(kv4, dtype, given):
    """Cache.empty copies the levels whatever their dtype, so one tensor may be
    given for keys and values, and writing it, or one of the cache's, changes
    no other."""
    lv = ref.random_levels(2, BF16, 0).to(given).cuda()
    want = lv.to(dtype).clone()
    c = kv4.Cache.empty(4, 16, 64, lv, lv, dtype)
    x = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    kv4.append(c, x, x, i32([0, 1, 2]))
    before = kv4.read(c, i32([0, 1, 2]))
    old = lv.clone()
    lv.zero_()
    assert torch.equal(c.k_levels, want) and torch.equal(c.v_levels, want)
    for a, b in zip(kv4.read(c, i32([0, 1, 2])), before):
        assert torch.equal(a, b)
    lv.copy_(old)
    c.k_levels.zero_()
    assert torch.equal(c.v_levels, want) and torch.equal(lv, old)
    # a slice that does not begin at 16 bytes, a transposed one
    wide = torch.zeros(16, 3, dtype=given, device="cuda")
    wide[:, 1:] = lv.t()
    c = kv4.Cache.empty(4, 16, 64, wide[:, 1:].t(), wide[:, 1:].t(), dtype)
    assert torch.equal(c.k_levels, want) and c.k_levels.is_contiguous()


# ------------------------------------------------------------ gradients

def test_a_gradient_through_the_cache_is_refused(kv4):
    """Attention over codes has no gradient: its result belongs to q's graph,
    and going back through it raises instead of leaving q's out."""
    lv = ref.random_levels(2, BF16, 0).cuda()
    c = kv4.Cache.empty(4, 16, 64, lv, lv, BF16)
    x = torch.randn(3, 2, 64, device="cuda").to(BF16)
    s, tb = i32([1, 1, 1]), i32([[0], [1], [2]])
    kv4.append(c, x, x, i32([0, 16, 32]))
    want, want_lse = kv4.attend(x, c, tb, s, return_lse=True)
    assert not want.requires_grad and not want_lse.requires_grad
    q = x.clone().requires_grad_()
    out, lse = kv4.attend(q * 1, c, tb, s, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    for y in out, lse, kv4.attend(q, c, tb, s), kv4.attend(q.transpose(0, 1).contiguous()
                                                           .transpose(0, 1), c, tb, s):
        with pytest.raises(RuntimeError, match="gradient"):
            (y.float().sum() + q.float().sum()).backward()
    room = torch.empty_like(x)
    held = kv4.attend(q, c, tb, s, out=room)
    assert held is room and torch.equal(room, want)
    with pytest.raises(RuntimeError, match="gradient"):
        held.float().sum().backward()
    with torch.no_grad():
        assert not kv4.attend(q, c, tb, s).requires_grad
    assert not kv4.attend(q.detach(), c, tb, s).requires_grad


# ------------------------------------------------------------ lengths past the sums

def test_block_tables_of_lengths_past_31_bits(kv4):
    """Lengths whose sums leave 31 bits (garbage in a padded row) reach no free
    block, and nothing outside the free list is read."""
    big = 2 ** 31 - 2  # two of them: 2^32 - 4 tokens, 2^31 - 2 blocks of two
    seq = [big, big, 10, 8]
    tb = torch.full((4, 3), 5, dtype=torch.int32, device="cuda")
    slots, cu, taken = kv4.block_tables(i32(seq), i32(seq), tb, i32([7, 8, 9]), 2, 20)
    assert slots.tolist() == [-1] * 20
    assert tb[3].tolist() == [-1] * 3


def test_query_offsets_that_do_not_ascend_end(kv4):
    """Offsets that go back and forth weigh every request as the whole step; the
    sum leaves 32 bits.  What is computed is anything, but every share ends, and
    the next call is as ever."""
    T, R, bs = 65536, 7, 1 << 20
    lv = ref.random_levels(1, BF16, 0).cuda()
    c = kv4.Cache.empty(1, bs, 64, lv, lv, BF16)
    q = torch.randn(T, 4, 64, device="cuda").to(BF16)
    # four requests of 1024 tiles of 2^20 + 16 granules: 2^32 + 2^16 in all
    tables = torch.full((R, 65), -1, dtype=torch.int32, device="cuda")
    out = kv4.attend(q, c, tables, i32([64 * (2 ** 20 + 12)] * R),
                     i32([0, T] * 4), causal=False)
    torch.cuda.synchronize()
    assert out.shape == (T, 4, 64)
    seq, nq = [130, 40], [130, 3]
    cache, tables, g = _setup(seq, 16, 1, 64, BF16, 3)
    _check_attend(kv4, cache, tables, q[:133].cpu(), seq, nq)
