"""A paged key/value cache held in 4 bits, with the attention that reads it.

Every key and value vector is stored as D codes of 4 bits into the 16 levels
of its head, and one scale (its largest magnitude).  The levels are centroids:
`learn_levels` finds them with `batch_kmeans_Euclid` on a sample, and storing
a vector assigns each element to its nearest one.  (The reference has no such
cache; the conventions here are those of its other entry points: dense GPU
tensors, work on the current stream, ValueError for host tensors,
RuntimeError for everything else that does not fit.)

A serving loop, with R requests of `seq_lens` tokens, the last `new_lens` of
them new:

    levels = kv4.learn_levels(sample_k), kv4.learn_levels(sample_v)
    cache = kv4.Cache.empty(num_blocks, block_size, head_dim, *levels, torch.bfloat16)
    slots, cu_new, taken = kv4.block_tables(seq_lens, new_lens, tables, free_blocks,
                                            block_size, num_tokens)
    kv4.append(cache, k, v, slots)
    out = kv4.attend(q, cache, tables, seq_lens, cu_new)

`tables` is updated in place.  Lengths, tables and slots stay on the GPU:
nothing here waits for it.

The cache holds codes, which have no gradient: `append` and `read` take and give
values only, and going back through `attend` raises.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._C import _require
from .kmeans import batch_kmeans_Euclid

LEVELS = 16


def _on_gpu(name: str, t: torch.Tensor, device: Optional[torch.device] = None) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"{name}: expected a tensor on a GPU device, found one on {t.device}")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} must be on {device}, found on {t.device}")


# Decoding calls these functions for a few microseconds of GPU work: what usually
# holds is tested first, in one expression, and explained only if it does not.

def _i32(name: str, t: torch.Tensor, dim: int, device: torch.device) -> torch.Tensor:
    if (t.dtype is torch.int32 and t.dim() == dim and t.get_device() == device.index
            and t.is_contiguous()):
        return t
    _on_gpu(name, t, device)
    if t.dtype != torch.int32 or t.dim() != dim:
        raise RuntimeError(f"{name} must be int32 with {dim} dimension(s)")
    return t.contiguous()


def _check_tables(t: torch.Tensor, R: int, device: torch.device) -> Tuple[int, int]:
    """(max_blocks, row stride) of tables (R, max_blocks) int32 with dense rows."""
    if t.get_device() != device.index:
        _on_gpu("tables", t, device)
    _require(t.dtype is torch.int32 and t.dim() == 2, "tables must be int32 (R, max_blocks)")
    rows, width = t.shape
    stride, dense = t.stride()
    _require(rows == R and (width <= 1 or dense == 1),
             f"tables must be ({R}, max_blocks) with dense rows")
    return width, stride if rows > 1 else width


def _rows(name: str, t: torch.Tensor, heads: int, cache: "Cache") -> torch.Tensor:
    """(T, heads, D) rows of the cache's dtype that the kernels can load 16
    bytes at a time; any token and head stride (a slice of a fused projection)
    that keeps them aligned, otherwise a dense copy."""
    if t.dtype is not cache.dtype or t.get_device() != cache.index:
        _on_gpu(name, t, cache.device)
        raise RuntimeError(f"{name} must have the cache's dtype {cache.dtype}")
    if t.dim() != 3 or (heads and t.shape[1] != heads) or t.shape[2] != cache.head_dim:
        raise RuntimeError(f"{name} must be (T, {heads or 'H'}, {cache.head_dim})")
    a, b, c = t.stride()
    if c != 1 or a % 8 or b % 8 or t.data_ptr() % 16:
        T, H, D = t.shape
        # the stride of a dimension of one entry is never used: 0 does as well
        a, b = a if T > 1 else 0, b if H > 1 else 0
        if c != 1 or a % 8 or b % 8 or t.data_ptr() % 16:
            # (contiguous() and clone() may keep such strides, or the offset)
            t = torch.empty((T, H, D), dtype=t.dtype, device=t.device).copy_(t)
        else:
            t = t.as_strided((T, H, D), (a, b, 1))
    return t


class _CCache(ctypes.Structure):
    """fkc_kv4_cache of include/fkc.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k_codes", "v_codes", "k_scales", "v_scales",
                                                "k_levels", "v_levels")]
                + [(n, ctypes.c_int64) for n in ("num_blocks", "heads", "block_size", "D")]
                + [("dtype", ctypes.c_int32)])


class Cache:
    """The cache's tensors, checked once; the kernels write into them.

    k_codes, v_codes (num_blocks, heads, block_size, D/2) uint8: element d of
    a vector in byte d // 2, even d in the low half; k_scales, v_scales
    (num_blocks, heads, block_size) and k_levels, v_levels (heads, 16) of one
    dtype, fp16 or bf16.  D is 64, 128 or 256, block_size a multiple of 16.
    A token's slot is block * block_size + its position in the block.

    The calls go on reading the tensors that the cache was made of: what they
    hold may be written, but none of them, nor any size, can be replaced.
    """

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scales: torch.Tensor,
                 v_scales: torch.Tensor, k_levels: torch.Tensor, v_levels: torch.Tensor) -> None:
        _on_gpu("k_codes", k_codes)
        self.device = k_codes.device
        self.index = self.device.index
        self.dtype = k_scales.dtype
        _require(self.dtype in (torch.float16, torch.bfloat16),
                 f"the cache's dtype must be fp16 or bf16, not {self.dtype}")
        _require(k_codes.dim() == 4, "k_codes must be (num_blocks, heads, block_size, D/2)")
        self.num_blocks, self.heads, self.block_size, half = k_codes.shape
        self.head_dim = 2 * half
        _require(self.head_dim in (64, 128, 256), f"D = {self.head_dim} is not 64, 128 or 256")
        _require(self.block_size > 0 and self.block_size % 16 == 0,
                 f"block_size {self.block_size} is not a multiple of 16")
        want = {"k_codes": (k_codes, tuple(k_codes.shape), torch.uint8),
                "v_codes": (v_codes, tuple(k_codes.shape), torch.uint8),
                "k_scales": (k_scales, tuple(k_codes.shape[:3]), self.dtype),
                "v_scales": (v_scales, tuple(k_codes.shape[:3]), self.dtype),
                "k_levels": (k_levels, (self.heads, LEVELS), self.dtype),
                "v_levels": (v_levels, (self.heads, LEVELS), self.dtype)}
        for name, (t, shape, dtype) in want.items():
            _on_gpu(name, t, self.device)
            _require(tuple(t.shape) == shape and t.dtype == dtype,
                     f"{name} must be {shape} {dtype}, found {tuple(t.shape)} {t.dtype}")
            _require(t.is_contiguous() and t.data_ptr() % 16 == 0,
                     f"{name} must be contiguous and 16-byte aligned")
            setattr(self, name, t)
        self._c = _CCache(*(getattr(self, n).data_ptr() for n in want), self.num_blocks,
                          self.heads, self.block_size, self.head_dim,
                          _lib.dtype_code(self.dtype))
        self._ref = ctypes.addressof(self._c)

    def __setattr__(self, name: str, value: object) -> None:
        if name in self.__dict__:
            raise AttributeError(f"a cache's {name} cannot be replaced: make another Cache")
        super().__setattr__(name, value)

    def __delattr__(self, name: str) -> None:
        raise AttributeError(f"a cache's {name} cannot be taken from it")

    @classmethod
    def empty(cls, num_blocks: int, block_size: int, head_dim: int, k_levels: torch.Tensor,
              v_levels: torch.Tensor, dtype: torch.dtype) -> "Cache":
        """A cache of num_blocks blocks on the levels' device.  The levels
        (heads, 16), of any floating dtype, are rounded to `dtype`; what the
        blocks hold before it is stored is never used."""
        heads, dev = k_levels.shape[0], k_levels.device
        codes = [torch.empty((num_blocks, heads, block_size, head_dim // 2), dtype=torch.uint8,
                             device=dev) for _ in range(2)]
        scales = [torch.empty((num_blocks, heads, block_size), dtype=dtype, device=dev)
                  for _ in range(2)]
        return cls(*codes, *scales, k_levels.to(dtype).contiguous(),
                   v_levels.to(dtype).contiguous())


def learn_levels(sample: torch.Tensor, max_iters: int = 25, tol: float = 1e-5) -> torch.Tensor:
    """(heads, 16) fp32 levels for vectors like `sample` (T, heads, D), fp16,
    bf16 or fp32: per head, k-means over the elements of the sample's vectors,
    each divided by its largest magnitude, from the elements' quantiles on."""
    _on_gpu("sample", sample)
    _require(sample.dim() == 3 and sample.numel() > 0, "sample must be (T, heads, D), not empty")
    x = sample.float()
    top = x.abs().amax(-1, keepdim=True)
    x = torch.where(top > 0, x / top, 0.0).transpose(0, 1).reshape(sample.shape[1], -1)
    ordered = x.sort(dim=1).values
    n = ordered.shape[1]
    at = ((torch.arange(LEVELS, device=x.device) + 0.5) * (n / LEVELS)).long().clamp_(max=n - 1)
    _, levels, _ = batch_kmeans_Euclid(x.unsqueeze(-1), LEVELS, max_iters=max_iters, tol=tol,
                                       init_centroids=ordered[:, at].unsqueeze(-1).contiguous())
    return levels.squeeze(-1)


def block_tables(seq_lens: torch.Tensor, new_lens: torch.Tensor, tables: torch.Tensor,
                 free_blocks: torch.Tensor, block_size: int, num_tokens: int
                 ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Blocks and slots of a step's new tokens; -> (slots, cu_new, taken).

    Request r has seq_lens[r] tokens after the step, the last new_lens[r] of
    them new, and tables (R, max_blocks) names the blocks of its older ones.
    Each block it needs beyond them is the next of free_blocks, in request
    order, and is entered into `tables` in place.  slots (num_tokens,) int32
    holds the new tokens' slots, request after request; cu_new (R + 1) int32
    their running count; taken (1) int32 the blocks needed in all, which the
    caller takes off its list.  num_tokens is at least the sum of new_lens:
    slots past it are -1.  So are the slots and entries of blocks that
    free_blocks does not reach (taken is then more than it holds) and the
    slots past max_blocks.
    """
    dev = seq_lens.device
    if dev.type != "cuda":
        _on_gpu("seq_lens", seq_lens)
    seq_lens = _i32("seq_lens", seq_lens, 1, dev)
    new_lens = _i32("new_lens", new_lens, 1, dev)
    free_blocks = _i32("free_blocks", free_blocks, 1, dev)
    R = seq_lens.shape[0]
    _require(new_lens.shape[0] == R, "new_lens must be as long as seq_lens")
    width, stride = _check_tables(tables, R, dev)
    _require(num_tokens >= 0, "num_tokens must not be negative")
    slots, cu_new, taken = torch.split_with_sizes(seq_lens.new_empty(num_tokens + R + 2),
                                                  (num_tokens, R + 1, 1))
    with _lib.on_device(seq_lens):
        _lib.check(_lib.lib.fkc_block_tables(
            seq_lens.data_ptr(), new_lens.data_ptr(), R, tables.data_ptr(), stride, width,
            free_blocks.data_ptr(), free_blocks.shape[0], block_size, num_tokens,
            slots.data_ptr(), cu_new.data_ptr(), taken.data_ptr(), _lib.stream_of(seq_lens)),
            "block_tables")
    return slots, cu_new, taken


def append(cache: Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Store k and v (T, heads, D) of the cache's dtype at slots (T,) int32.

    A vector's scale is its largest magnitude (0 below 2^-126), an element's
    code the level nearest to element * (1 / scale), the lowest index of
    equal ones.  Slots outside the cache (-1) are skipped, and their vectors
    not read.
    """
    k, v = _rows("k", k, cache.heads, cache), _rows("v", v, cache.heads, cache)
    slots = _i32("slots", slots, 1, cache.device)
    T = slots.shape[0]
    _require(k.shape[0] == T and v.shape[0] == T, "k, v and slots must have as many tokens")
    (ka, kb, _), (va, vb, _) = k.stride(), v.stride()
    with _lib.on_device(slots):
        _lib.check(_lib.lib.fkc_kv4_append(
            cache._ref, k.data_ptr(), ka, kb, v.data_ptr(), va, vb, slots.data_ptr(), T,
            _lib.stream_of(slots)), "append")


def read(cache: Cache, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values (T, heads, D) that slots (T,) int32 hold, scale *
    level rounded once to the cache's dtype; zeros outside the cache."""
    slots = _i32("slots", slots, 1, cache.device)
    T = slots.shape[0]
    k = cache.k_scales.new_empty((T, cache.heads, cache.head_dim))
    v = torch.empty_like(k)
    with _lib.on_device(slots):
        _lib.check(_lib.lib.fkc_kv4_read(cache._ref, slots.data_ptr(), T, k.data_ptr(),
                                         v.data_ptr(), _lib.stream_of(slots)), "read")
    return k, v


class _NoGradient(torch.autograd.Function):
    """Puts attend's results into the graph of its queries, so that a gradient
    that would have to pass through them raises instead of being left out."""

    @staticmethod
    def forward(ctx, q, *results):
        ctx.mark_dirty(*results)
        return results

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("kv4.attend has no gradient: detach q, or call it under no_grad")


def attend(q: torch.Tensor, cache: Cache, tables: torch.Tensor, seq_lens: torch.Tensor,
           cu_q: Optional[torch.Tensor] = None, *, causal: bool = True,
           sm_scale: Optional[float] = None, max_seq: Optional[int] = None,
           out: Optional[torch.Tensor] = None, return_lse: bool = False
           ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of q (T, H, D) over the cached tokens of R requests.

    Request r has seq_lens[r] tokens, in the blocks tables[r], and owns the
    queries cu_q[r] .. cu_q[r+1] (cu_q (R + 1) int32 from 0 on, ascending;
    None: one query each, T = R).  They are its last tokens: with `causal`
    each sees the tokens up to itself, otherwise all of them.  Query head h
    reads cache head h // (H / heads).  Rows that see nothing, and rows past
    cu_q[R], are 0.  sm_scale: 1 / sqrt(D) if not given.  max_seq: a bound of
    seq_lens that the caller knows (the tables' width otherwise); longer
    requests are cut to it.  Where contexts are much shorter than the tables
    it is worth giving: 64 requests of 1000 to 1441 tokens take 22 us with it and
    34 without.  Scores, maxima, sums and outputs are fp32; a softmax weight
    times its value's scale is rounded to q's dtype before it meets the value,
    and the result is.  Returns (T, H, D) in q's dtype, in `out` when
    given, and with return_lse also log sum exp of each row's scores, fp32
    (T, H), -inf for rows that see nothing.  There is no gradient: going back
    through the result of a q that requires one raises RuntimeError.
    """
    q = _rows("q", q, 0, cache)
    dev = cache.device
    seq_lens = _i32("seq_lens", seq_lens, 1, dev)
    if cu_q is not None:
        cu_q = _i32("cu_q", cu_q, 1, dev)
    T, H, D = q.shape
    R = seq_lens.shape[0]
    _require(H > 0 and H % cache.heads == 0,
             f"q's heads must be a multiple of the cache's {cache.heads}")
    width, stride = _check_tables(tables, R, dev)
    _require(T == R if cu_q is None else cu_q.shape[0] == R + 1,
             "q must have one row per request, or cu_q R + 1 entries")
    if max_seq is None:
        max_seq = width * cache.block_size
    _require(0 <= max_seq <= width * cache.block_size,
             f"max_seq {max_seq} does not fit {width} blocks of {cache.block_size}")
    if out is None:
        out = q.new_empty((T, H, D))
    else:
        _on_gpu("out", out, dev)
        _require(out.dtype == q.dtype and tuple(out.shape) == (T, H, D)
                 and out.is_contiguous(), f"out must be a contiguous ({T}, {H}, {D}) {q.dtype}")
    lse = torch.empty((T, H), dtype=torch.float32, device=dev) if return_lse else None
    if sm_scale is None:
        sm_scale = D ** -0.5
    with _lib.on_device(q):
        need = _lib.lib.fkc_kv4_attend_workspace_bytes(cache._ref, H, T, R, max_seq)
        ws = _lib.workspace(need, dev) if need else None
        _lib.check(_lib.lib.fkc_kv4_attend(
            cache._ref, q.data_ptr(), q.stride(0), q.stride(1), H, T, tables.data_ptr(), stride,
            width, seq_lens.data_ptr(), _lib.ptr(cu_q), R, max_seq, int(causal), sm_scale,
            out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), need, _lib.stream_of(q)), "attend")
    if q.requires_grad and torch.is_grad_enabled():
        if lse is not None:
            out, lse = _NoGradient.apply(q, out, lse)
        else:
            out, = _NoGradient.apply(q, out)
    return (out, lse) if return_lse else out
