// Pages of the 4-bit cache: which blocks no row holds, rows that go on from
// others' tokens, the held blocks moved into another cache, blocks copied.
//
// Row r of the tables holds its first ceil(seq / bs) entries, as far as the row
// goes; entries outside the cache are nobody's.  Nothing is counted from call to
// call: a block is free when no row names it, whatever was forked, cut back or
// given up before.
#include <algorithm>

#include "device_util.hpp"
#include "fkc_internal.hpp"

namespace fkc {
namespace {

constexpr int PT = 256;          // threads per workgroup
constexpr int CHUNK = 4096;      // blocks that a workgroup of the list counts
constexpr int ENTRIES = 1024;    // table entries of a row per workgroup and turn

struct Rows {
  const int32_t* tables;
  int64_t stride;
  const int32_t* seq;
  int64_t R;
  int width;
  uint32_t bs;
  // Entries of row r that are held, and of these the ones that are full.
  __device__ inline int held(int64_t r) const {
    const uint32_t s = (uint32_t)max(seq[r], 0);
    return (int)min((s + bs - 1) / bs, (uint32_t)width);
  }
};

// ------------------------------------------------- which blocks are held

__global__ void __launch_bounds__(PT)
clear_kernel(uint32_t* __restrict__ p, int64_t words) {
  for (int64_t i = (int64_t)blockIdx.x * PT + threadIdx.x; i < words;
       i += (int64_t)gridDim.x * PT)
    p[i] = 0;
}

// A byte per block.  (Bytes rather than bits: stores of the same value need no
// atomics.)
__global__ void __launch_bounds__(PT)
mark_kernel(const Rows t, uint32_t num_blocks, uint8_t* __restrict__ named) {
  const int parts = (t.width + ENTRIES - 1) / ENTRIES;
  for (int64_t u = blockIdx.x; u < t.R * parts; u += gridDim.x) {
    const int64_t r = u / parts;
    const int lo = (int)(u - r * parts) * ENTRIES, hi = min(t.held(r), lo + ENTRIES);
    for (int e = lo + threadIdx.x; e < hi; e += PT) {
      const uint32_t b = (uint32_t)t.tables[r * t.stride + e];
      if (b < num_blocks) named[b] = 1;
    }
  }
}

__device__ inline int wg_sum(int v, int* s) {
  v = wave_sum_i(v);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int w = 0; w < PT / 64; ++w) sum += s[w];
  __syncthreads();
  return sum;
}

// The named bytes of 16 blocks as a bit mask; those past the last count as not
// named.
__device__ inline uint32_t mask16(const uint8_t* named, int64_t b, int64_t num_blocks) {
  uint32_t m = 0;
  if (b < num_blocks) {  // (the bytes are padded to whole chunks)
    const uint4 w = *reinterpret_cast<const uint4*>(named + b);
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) m |= (x[i] * 0x10204080u >> 28) << (4 * i);
  }
  return m;
}

__global__ void __launch_bounds__(PT)
count_kernel(const uint8_t* __restrict__ named, int64_t num_blocks, int32_t* __restrict__ counts) {
  __shared__ int s[PT / 64];
  const int64_t b = (int64_t)blockIdx.x * CHUNK + threadIdx.x * 16;
  const int sum = wg_sum(__popc(mask16(named, b, num_blocks)), s);
  if (threadIdx.x == 0) counts[blockIdx.x] = sum;
}

// Lists the free blocks, or the held ones and each one's place among them.
template <bool FREE>
__global__ void __launch_bounds__(PT)
list_kernel(const uint8_t* __restrict__ named, int64_t num_blocks,
            const int32_t* __restrict__ counts, int32_t* __restrict__ list,
            int32_t* __restrict__ number, int32_t* __restrict__ total) {
  __shared__ int s[PT / 64];
  const int t = threadIdx.x;
  int below = 0, all = 0;
  for (int i = t; i < (int)gridDim.x; i += PT) {
    const int c = counts[i];
    all += c;
    below += i < (int)blockIdx.x ? c : 0;
  }
  below = wg_sum(below, s);
  all = wg_sum(all, s);
  const int64_t b0 = (int64_t)blockIdx.x * CHUNK + t * 16;
  const uint32_t m = mask16(named, b0, num_blocks);
  const int mine = __popc(m);
  int incl = wave_incl_scan(mine);
  if ((t & 63) == 63) s[t >> 6] = incl;
  __syncthreads();
  for (int w = 0; w < t >> 6; ++w) incl += s[w];
  int at = below + incl - mine;  // held blocks before mine
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t b = b0 + i;
    if (b >= num_blocks) break;
    const bool held = m >> i & 1;
    if (FREE) {
      if (!held) list[b - at] = (int32_t)b;
    } else if (held) {
      list[at] = (int32_t)b;
      number[b] = at;
    }
    at += held;
  }
  if (FREE) {
    // behind the free ones, as many as are held
    for (int64_t i = (int64_t)blockIdx.x * PT + t; i < all; i += (int64_t)gridDim.x * PT)
      list[num_blocks - all + i] = -1;
  }
  if (blockIdx.x == 0 && t == 0) *total = FREE ? (int)(num_blocks - all) : all;
}

// ------------------------------------------------- moving blocks

// A block's codes and scales are four runs of 16-byte units.
struct Store {
  uint4* p[4];
  __host__ __device__ explicit Store(const fkc_kv4_cache& c)
      : p{(uint4*)c.k_codes, (uint4*)c.v_codes, (uint4*)c.k_scales, (uint4*)c.v_scales} {}
};

constexpr int PIECE = 4 * PT;  // units a workgroup copies at a time

// Piece `piece` of block sb to block db.  codes, scales: units of one run.
__device__ inline void copy_piece(const Store& from, int64_t sb, const Store& to, int64_t db,
                                  int64_t piece, int codes, int scales) {
  const int all = 2 * (codes + scales);
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t u = piece * PIECE + i * PT + threadIdx.x;
    if (u >= all) continue;
    const int run = u < 2 * (int64_t)codes ? u >= codes : 2 + (u >= 2 * (int64_t)codes + scales);
    const int64_t in = run < 2 ? u - run * (int64_t)codes
                               : u - 2 * (int64_t)codes - (run - 2) * (int64_t)scales;
    v[i] = from.p[run][sb * (run < 2 ? codes : scales) + in];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t u = piece * PIECE + i * PT + threadIdx.x;
    if (u >= all) continue;
    const int run = u < 2 * (int64_t)codes ? u >= codes : 2 + (u >= 2 * (int64_t)codes + scales);
    const int64_t in = run < 2 ? u - run * (int64_t)codes
                               : u - 2 * (int64_t)codes - (run - 2) * (int64_t)scales;
    to.p[run][db * (run < 2 ? codes : scales) + in] = v[i];
  }
}

// Blocks src[i] to dst[i] (null: i), i below n and *count (null: n).
__global__ void __launch_bounds__(PT)
copy_kernel(const Store from, uint32_t from_blocks, const Store to, uint32_t to_blocks,
            const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int64_t n,
            const int32_t* __restrict__ count, int codes, int scales) {
  const int64_t pieces = (2 * ((int64_t)codes + scales) + PIECE - 1) / PIECE;
  if (count != nullptr) n = min(n, (int64_t)*count);
  for (int64_t u = blockIdx.x; u < n * pieces; u += gridDim.x) {
    const int64_t i = u / pieces;
    const uint32_t sb = (uint32_t)src[i], db = dst == nullptr ? (uint32_t)i : (uint32_t)dst[i];
    if (sb < from_blocks && db < to_blocks)
      copy_piece(from, sb, to, db, u - i * pieces, codes, scales);
  }
}

// Tables whose entries are the blocks' places among the held ones; -1 where a
// row holds nothing, or `into` has no such block.
__global__ void __launch_bounds__(PT)
renumber_kernel(const Rows t, uint32_t num_blocks, const int32_t* __restrict__ number,
                int into_blocks, int32_t* __restrict__ out) {
  const int parts = (t.width + ENTRIES - 1) / ENTRIES;
  for (int64_t u = blockIdx.x; u < t.R * parts; u += gridDim.x) {
    const int64_t r = u / parts;
    const int lo = (int)(u - r * parts) * ENTRIES, hi = min(t.width, lo + ENTRIES);
    const int held = t.held(r);
    for (int e = lo + threadIdx.x; e < hi; e += PT) {
      int32_t v = -1;
      if (e < held) {
        const uint32_t b = (uint32_t)t.tables[r * t.stride + e];
        if (b < num_blocks) v = number[b];
        if (v >= into_blocks) v = -1;
      }
      out[r * t.width + e] = v;
    }
  }
}

// ------------------------------------------------- fork

// What child j goes on from.
struct Child {
  int64_t row;  // -1: nothing
  int seq, whole;
  int part;  // block that its last tokens share with nothing else's; -1: none
};

__device__ inline Child child_of(const Rows& t, const int32_t* parents, int64_t j,
                                 uint32_t num_blocks) {
  Child c{parents[j], 0, 0, -1};
  if (c.row < 0 || c.row >= t.R) {
    c.row = -1;
    return c;
  }
  c.seq = max(t.seq[c.row], 0);
  c.whole = (int)min((uint32_t)c.seq / t.bs, (uint32_t)t.width);
  if ((uint32_t)c.seq % t.bs != 0 && c.whole < t.width) {
    const uint32_t b = (uint32_t)t.tables[c.row * t.stride + c.whole];
    if (b < num_blocks) c.part = (int)b;
  }
  return c;
}

// first[b], for the blocks that some child ends in, becomes the lowest such
// child, or -1 where a child has b as a whole block.
__global__ void __launch_bounds__(PT)
fork_clear_kernel(const Rows t, const int32_t* __restrict__ parents, int64_t F,
                  uint32_t num_blocks, int32_t* __restrict__ first) {
  const int64_t j = (int64_t)blockIdx.x * PT + threadIdx.x;
  if (j >= F) return;
  const Child c = child_of(t, parents, j, num_blocks);
  if (c.part >= 0) first[c.part] = INT32_MAX;
}

// A workgroup per child: its row of the new tables, its length, its marks.
__global__ void __launch_bounds__(PT)
fork_mark_kernel(const Rows t, const int32_t* __restrict__ parents, int64_t F,
                 uint32_t num_blocks, int32_t* __restrict__ first, int32_t* __restrict__ out,
                 int32_t* __restrict__ out_seq) {
  const int64_t j = blockIdx.x;
  const Child c = child_of(t, parents, j, num_blocks);
  // Marks of a parent are made once, or nearly: by the first of the last 1024
  // children that go on from it.
  bool seen = false;
  for (int64_t i = max(j - 1024, (int64_t)0) + threadIdx.x; i < j; i += PT)
    seen |= parents[i] == parents[j];
  seen = __syncthreads_or(seen);
  for (int e = threadIdx.x; e < t.width; e += PT) {
    int32_t v = -1;
    if (c.row >= 0 && e < c.whole) {
      const uint32_t b = (uint32_t)t.tables[c.row * t.stride + e];
      if (b < num_blocks) {
        v = (int32_t)b;
        if (!seen) __hip_atomic_fetch_min(first + b, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    } else if (e == c.whole) {
      v = c.part;
    }
    out[j * t.width + e] = v;
  }
  if (threadIdx.x == 0) {
    out_seq[j] = c.seq;
    if (c.part >= 0)
      __hip_atomic_fetch_min(first + c.part, (int)j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// One workgroup: which children get a block of their own, in order.
constexpr int FT = 1024;
__global__ void __launch_bounds__(FT)
fork_place_kernel(const Rows t, const int32_t* __restrict__ parents, int64_t F,
                  uint32_t num_blocks, const int32_t* __restrict__ first,
                  const int32_t* __restrict__ free_blocks, int64_t num_free,
                  int32_t* __restrict__ out, int32_t* __restrict__ src,
                  int32_t* __restrict__ dst, int32_t* __restrict__ taken) {
  __shared__ int s[FT / 64];
  int base = 0;
  for (int64_t j0 = 0; j0 < F; j0 += FT) {
    const int64_t j = j0 + threadIdx.x;
    Child c{-1, 0, 0, -1};
    if (j < F) c = child_of(t, parents, j, num_blocks);
    const bool copy = c.part >= 0 && first[c.part] != (int)j;
    int at = wave_incl_scan(copy);
    if ((threadIdx.x & 63) == 63) s[threadIdx.x >> 6] = at;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < FT / 64; ++w) {
      at += w < (int)(threadIdx.x >> 6) ? s[w] : 0;
      all += s[w];
    }
    if (copy) {
      at += base - 1;
      int32_t b = at < num_free ? free_blocks[at] : -1;
      if ((uint32_t)b >= num_blocks) b = -1;
      src[at] = c.part;
      dst[at] = b;
      out[j * t.width + c.whole] = b;
    }
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *taken = base;
}

// ------------------------------------------------- workspaces, launches

struct Names {
  uint8_t* named;
  int32_t* counts;
  int64_t chunks;
  Names(Carve& w, int64_t num_blocks) : chunks((num_blocks + CHUNK - 1) / CHUNK) {
    named = w.take<uint8_t>((size_t)chunks * CHUNK);
    counts = w.take<int32_t>((size_t)chunks);
  }
};

uint32_t grid_for(int64_t items, int per_cu) {
  const int64_t most = (int64_t)device_shape().cus * per_cu;
  return (uint32_t)std::max<int64_t>(1, std::min(items, most));
}

int64_t row_parts(const Kv4Tables& t) { return t.R * ((t.max_blocks + ENTRIES - 1) / ENTRIES); }

Rows rows_of(const Kv4Tables& t, int64_t bs) {
  return Rows{t.tables, t.stride, t.seq, t.R, (int)t.max_blocks, (uint32_t)bs};
}

void launch_names(const Kv4Tables& t, int64_t bs, int64_t num_blocks, const Names& n,
                  hipStream_t s) {
  hipLaunchKernelGGL(clear_kernel, dim3(grid_for((n.chunks * CHUNK / 4 + PT - 1) / PT, 8)),
                     dim3(PT), 0, s, (uint32_t*)n.named, n.chunks * CHUNK / 4);
  if (row_parts(t) > 0)
    hipLaunchKernelGGL(mark_kernel, dim3(grid_for(row_parts(t), 16)), dim3(PT), 0, s,
                       rows_of(t, bs), (uint32_t)num_blocks, n.named);
  hipLaunchKernelGGL(count_kernel, dim3((uint32_t)n.chunks), dim3(PT), 0, s, n.named, num_blocks,
                     n.counts);
}

void launch_copy(const fkc_kv4_cache& from, const fkc_kv4_cache& to, const int32_t* src,
                 const int32_t* dst, int64_t n, const int32_t* count, hipStream_t s) {
  const int codes = (int)(from.heads * from.block_size * from.D / 32);
  const int scales = (int)(from.heads * from.block_size / 8);
  const int64_t pieces = (2 * ((int64_t)codes + scales) + PIECE - 1) / PIECE;
  hipLaunchKernelGGL(copy_kernel, dim3(grid_for(n * pieces, 8)), dim3(PT), 0, s, Store(from),
                     (uint32_t)from.num_blocks, Store(to), (uint32_t)to.num_blocks, src, dst, n,
                     count, codes, scales);
}

__global__ void zero_kernel(int32_t* p) { *p = 0; }

}  // namespace

size_t free_blocks_workspace_bytes(int64_t num_blocks) {
  Carve w(nullptr);
  Names n(w, num_blocks);
  return w.used;
}

int launch_free_blocks(const Kv4Tables& t, int64_t bs, int64_t num_blocks, int32_t* free_blocks,
                       int32_t* count, void* ws, hipStream_t s) {
  Carve w(ws);
  const Names n(w, num_blocks);
  if (num_blocks == 0) {
    hipLaunchKernelGGL(zero_kernel, dim3(1), dim3(1), 0, s, count);
    return check_launch("free_blocks");
  }
  launch_names(t, bs, num_blocks, n, s);
  hipLaunchKernelGGL(list_kernel<true>, dim3((uint32_t)n.chunks), dim3(PT), 0, s, n.named,
                     num_blocks, n.counts, free_blocks, (int32_t*)nullptr, count);
  return check_launch("free_blocks");
}

size_t kv4_compact_workspace_bytes(const fkc_kv4_cache& c) {
  Carve w(nullptr);
  Names n(w, c.num_blocks);
  w.take<int32_t>((size_t)c.num_blocks * 2);
  return w.used;
}

int launch_kv4_compact(const fkc_kv4_cache& c, const Kv4Tables& t, const fkc_kv4_cache& into,
                       int32_t* new_tables, int32_t* used, void* ws, hipStream_t s) {
  Carve w(ws);
  const Names n(w, c.num_blocks);
  int32_t* list = w.take<int32_t>((size_t)c.num_blocks * 2);
  int32_t* number = list + c.num_blocks;
  if (c.num_blocks == 0) {
    hipLaunchKernelGGL(zero_kernel, dim3(1), dim3(1), 0, s, used);
  } else {
    launch_names(t, c.block_size, c.num_blocks, n, s);
    hipLaunchKernelGGL(list_kernel<false>, dim3((uint32_t)n.chunks), dim3(PT), 0, s, n.named,
                       c.num_blocks, n.counts, list, number, used);
  }
  if (row_parts(t) > 0)
    hipLaunchKernelGGL(renumber_kernel, dim3(grid_for(row_parts(t), 16)), dim3(PT), 0, s,
                       rows_of(t, c.block_size), (uint32_t)c.num_blocks, number,
                       (int)into.num_blocks, new_tables);
  const int64_t most = std::min(c.num_blocks, into.num_blocks);
  if (most > 0) launch_copy(c, into, list, nullptr, most, used, s);
  return check_launch("kv4_compact");
}

int launch_kv4_copy_blocks(const fkc_kv4_cache& c, const int32_t* src, const fkc_kv4_cache& into,
                           const int32_t* dst, int64_t n, hipStream_t s) {
  launch_copy(c, into, src, dst, n, nullptr, s);
  return check_launch("kv4_copy_blocks");
}

size_t kv4_fork_workspace_bytes(const fkc_kv4_cache& c, int64_t F) {
  Carve w(nullptr);
  w.take<int32_t>((size_t)c.num_blocks);
  w.take<int32_t>((size_t)F * 2);
  return w.used;
}

int launch_kv4_fork(const fkc_kv4_cache& c, const Kv4Tables& t, const int32_t* parents, int64_t F,
                    const int32_t* free_blocks, int64_t num_free, int32_t* new_tables,
                    int32_t* new_seq, int32_t* taken, void* ws, hipStream_t s) {
  Carve w(ws);
  int32_t* first = w.take<int32_t>((size_t)c.num_blocks);
  int32_t* src = w.take<int32_t>((size_t)F * 2);
  int32_t* dst = src + F;
  const Rows r = rows_of(t, c.block_size);
  const uint32_t nb = (uint32_t)c.num_blocks;
  if (F > 0) {
    hipLaunchKernelGGL(fork_clear_kernel, dim3((uint32_t)((F + PT - 1) / PT)), dim3(PT), 0, s, r,
                       parents, F, nb, first);
    hipLaunchKernelGGL(fork_mark_kernel, dim3((uint32_t)F), dim3(PT), 0, s, r, parents, F, nb,
                       first, new_tables, new_seq);
  }
  hipLaunchKernelGGL(fork_place_kernel, dim3(1), dim3(FT), 0, s, r, parents, F, nb, first,
                     free_blocks, num_free, new_tables, src, dst, taken);
  if (F > 0 && nb > 0) launch_copy(c, c, src, dst, F, taken, s);
  return check_launch("kv4_fork");
}

}  // namespace fkc
