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
constexpr int CHUNK = 1024;      // blocks that a workgroup lists
constexpr int ENTRIES = 1024;    // table entries of a row per workgroup and turn

struct Rows {
  const int32_t* tables;
  int64_t stride;
  const int32_t* seq;
  int64_t R;
  int width;
  uint32_t bs;
  FastDiv by_width;
  // Entries of row r that are held.
  __device__ inline int held(int64_t r) const {
    const uint32_t s = (uint32_t)max(seq[r], 0);
    return (int)min((s + bs - 1) / bs, (uint32_t)width);
  }
};

// Inclusive scan over the workgroup's T threads; *total: the sum.
template <int T>
__device__ inline int wg_scan(int v, int* s, int* total) {
  int incl = wave_incl_scan(v);
  __syncthreads();  // s is read
  if ((threadIdx.x & 63) == 63) s[threadIdx.x >> 6] = incl;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    incl += w < (int)(threadIdx.x >> 6) ? s[w] : 0;
    all += s[w];
  }
  *total = all;
  return incl;
}

// ------------------------------------------------- which blocks are held

// -1 behind the free blocks, as many as are held; by the whole grid.
template <bool FREE, int T>
__device__ inline void finish(int64_t num_blocks, int all, int32_t* list, int32_t* total) {
  if (FREE)
    for (int64_t i = (int64_t)blockIdx.x * T + threadIdx.x; i < all; i += (int64_t)gridDim.x * T)
      list[num_blocks - all + i] = -1;
  if (blockIdx.x == 0 && threadIdx.x == 0) *total = FREE ? (int)(num_blocks - all) : all;
}

// Small tables, one launch: every workgroup marks all of them in a bitmap of
// its own, counts, and lists its part.  Bound by latency (64 rows of up to
// 128 entries over 4700 blocks 5.4 us, the three launches below 9).  More entries
// or blocks than this cost more time here than the launches that it saves.
constexpr int ST = 1024, kSmallBlocks = 1 << 16, kSmallEntries = 1 << 15;
template <bool FREE>
__global__ void __launch_bounds__(ST)
names_small_kernel(const Rows t, uint32_t num_blocks, int32_t* __restrict__ list,
                   int32_t* __restrict__ number, int32_t* __restrict__ total) {
  constexpr int PER = 2;  // words of 32 blocks per thread
  static_assert(ST * PER * 32 == kSmallBlocks, "a bit for every block");
  __shared__ uint32_t bits[ST * PER];
  __shared__ int before[ST * PER];
  __shared__ int s[ST / 64];
#pragma unroll
  for (int i = 0; i < PER; ++i) bits[threadIdx.x + i * ST] = 0;
  __syncthreads();
  const int n = (int)t.R * t.width;
  for (int e0 = threadIdx.x; e0 < n; e0 += ST * 4) {
    uint32_t b[4];
    bool in[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = min(e0 + i * ST, n - 1);
      const int r = (int)t.by_width.div(e), c = e - r * t.width;
      b[i] = (uint32_t)t.tables[r * t.stride + c];
      in[i] = c < t.held(r);  // (the last entry may be marked again)
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (in[i] && b[i] < num_blocks) atomicOr(&bits[b[i] / 32], 1u << (b[i] & 31));
  }
  __syncthreads();
  int mine = 0, all;
#pragma unroll
  for (int i = 0; i < PER; ++i) mine += __popc(bits[threadIdx.x * PER + i]);
  int at = wg_scan<ST>(mine, s, &all) - mine;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    before[threadIdx.x * PER + i] = at;
    at += __popc(bits[threadIdx.x * PER + i]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < CHUNK; i += ST) {
    const uint32_t b = blockIdx.x * CHUNK + i;
    if (b >= num_blocks) break;
    const uint32_t w = bits[b / 32];
    const int held = before[b / 32] + __popc(w & ((1u << (b & 31)) - 1));
    const bool is = w >> (b & 31) & 1;
    if (FREE) {
      if (!is) list[b - held] = (int32_t)b;
    } else if (is) {
      list[held] = (int32_t)b;
      number[b] = held;
    }
  }
  finish<FREE, ST>(num_blocks, all, list, total);
}

// Larger ones: each held entry writes its number where its block is, whichever
// comes last.  Nothing is cleared before: what stands there counts only if it is
// the number of a held entry that names this block.  Bound by latency: 2048 rows of
// up to 1024 entries over 470000 blocks take 5.4 + 5.0 + 3.4 us for marking,
// counting and listing (a byte per block, cleared first, 2.2 + 4.6 + 2.4 + 4.5).
// Every workgroup of the last adds up the counts of all, which grows with the square
// of the blocks: a call over 2^20 / 2^22 / 2^24 / 2^26 of them takes 47 / 68 / 165 /
// 1215 us, of which writing the list is 60 at most.
__global__ void __launch_bounds__(PT)
mark_kernel(const Rows t, uint32_t num_blocks, uint32_t* __restrict__ entry) {
  const int parts = (t.width + ENTRIES - 1) / ENTRIES;
  for (int64_t u = blockIdx.x; u < t.R * parts; u += gridDim.x) {
    const int64_t r = parts == 1 ? u : u / parts;
    const int lo = (int)(u - r * parts) * ENTRIES, hi = min(t.held(r), lo + ENTRIES);
    for (int e = lo + threadIdx.x; e < hi; e += PT) {
      const uint32_t b = (uint32_t)t.tables[r * t.stride + e];
      if (b < num_blocks) entry[b] = (uint32_t)(r * t.width + e);
    }
  }
}

__device__ inline bool named(const Rows& t, uint32_t b, uint32_t e) {
  if (e >= (uint64_t)t.R * t.width) return false;
  const uint32_t r = e >> 31 ? e / t.width : t.by_width.div(e);
  const int c = (int)(e - r * (uint32_t)t.width);
  return (uint32_t)t.tables[r * t.stride + c] == b && c < t.held(r);
}

// A wave's blocks, 64 at a time; masks holds a bit for each.
constexpr int GROUPS = CHUNK / PT;

__device__ inline int64_t first_of(int i) {
  return (int64_t)blockIdx.x * CHUNK + ((threadIdx.x >> 6) * GROUPS + i) * 64;
}

__global__ void __launch_bounds__(PT)
count_kernel(const Rows t, int64_t num_blocks, const uint32_t* __restrict__ entry,
             uint64_t* __restrict__ masks, int32_t* __restrict__ counts) {
  __shared__ int s[PT / 64];
  const int lane = threadIdx.x & 63;
  uint32_t e[GROUPS];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const int64_t b = first_of(i) + lane;
    e[i] = b < num_blocks ? entry[b] : 0xffffffffu;
  }
  bool is[GROUPS];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) is[i] = named(t, (uint32_t)(first_of(i) + lane), e[i]);
  int sum = 0;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const uint64_t m = __ballot(is[i]);
    sum += __popcll(m);
    if (lane == 0) masks[first_of(i) / 64] = m;
  }
  if (lane == 0) s[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
#pragma unroll
    for (int w = 0; w < PT / 64; ++w) sum += s[w];
    counts[blockIdx.x] = sum;
  }
}

template <bool FREE>
__global__ void __launch_bounds__(PT)
list_kernel(int64_t num_blocks, const uint64_t* __restrict__ masks,
            const int32_t* __restrict__ counts, int32_t* __restrict__ list,
            int32_t* __restrict__ number, int32_t* __restrict__ total) {
  __shared__ int s[PT / 64];
  uint64_t m[GROUPS];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    m[i] = masks[first_of(i) / 64];
    mine += __popcll(m[i]);
  }
  int below = 0, all = 0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += PT) {
    const int c = counts[i];
    all += c;
    below += i < (int)blockIdx.x ? c : 0;
  }
  const int lane = threadIdx.x & 63;
  int at, sum;
  wg_scan<PT>(below, s, &below);
  wg_scan<PT>(all, s, &all);
  at = below + wg_scan<PT>(lane == 63 ? mine : 0, s, &sum) - (lane == 63 ? mine : 0);
  at = __shfl(at, 63, 64);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const int64_t b = first_of(i) + lane;
    const int held = at + (int)lanes_below(m[i]);
    const bool is = m[i] >> lane & 1;
    if (FREE) {
      if (!is && b < num_blocks) list[b - held] = (int32_t)b;
    } else if (is) {
      list[held] = (int32_t)b;
      number[b] = held;
    }
    at += __popcll(m[i]);
  }
  finish<FREE, PT>(num_blocks, all, list, total);
}

// ------------------------------------------------- moving blocks

// A block's codes and scales are four runs of 16-byte units.
typedef uint32_t Unit __attribute__((ext_vector_type(4)));
struct Store {
  Unit* p[4];
  __host__ __device__ explicit Store(const fkc_kv4_cache& c)
      : p{(Unit*)c.k_codes, (Unit*)c.v_codes, (Unit*)c.k_scales, (Unit*)c.v_scales} {}
};

constexpr int LOADS = 2;             // units per thread at a time
constexpr int PIECE = LOADS * PT;    // units a workgroup copies at a time

// Blocks as pieces, dealt out to workgroups in turn.
struct Pieces {
  int codes, scales;  // units of one run
  int per;            // pieces of a block
  FastDiv by_per;
  Pieces(const fkc_kv4_cache& c)
      : codes((int)(c.heads * c.block_size * c.D / 32)),
        scales((int)(c.heads * c.block_size / 8)),
        per((2 * (codes + scales) + PIECE - 1) / PIECE),
        by_per((uint32_t)per) {}
};

// Piece `piece` of block sb to block db.  Bound by memory: 465 MB moved by
// compact_kernel take 169 us, 5.5 TB/s counting both ways, where a large
// library copy reaches 4.6.  The copies are not read here again: stored past the
// caches they leave these to the loads (us a call without / with that, and with
// loads past the caches too: 465 MB 204 / 182 / 176, 31.7 MB 23.2 / 11.7 / 15.0).
// Units per thread at a time 2 / 4 / 8: 465 MB 177 / 182 / 221.
struct Piece {
  Unit v[LOADS];
  int piece;
  // Run, units of it in a block and unit of the i-th one, -1 past the block.
  __device__ inline int place(const Pieces& p, int i, int* run, int* units) const {
    const int u = piece * PIECE + i * PT + (int)threadIdx.x;
    int in = u;
    *run = 0;
    *units = p.codes;
    if (in >= p.codes) in -= p.codes, *run = 1;
    if (u >= 2 * p.codes) {
      in -= p.codes;
      *run = 2;
      *units = p.scales;
      if (in >= p.scales) in -= p.scales, *run = 3;
    }
    return u < 2 * (p.codes + p.scales) ? in : -1;
  }
  // Nothing is loaded of a block below 0.
  __device__ inline Piece(const Store& from, int block, int piece_, const Pieces& p)
      : piece(piece_) {
    if (block < 0) return;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int run, units;
      const int in = place(p, i, &run, &units);
      if (in >= 0) v[i] = from.p[run][(int64_t)block * units + in];
    }
  }
  __device__ inline void store(const Store& to, uint32_t block, const Pieces& p) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int run, units;
      const int in = place(p, i, &run, &units);
      if (in >= 0)
        __builtin_nontemporal_store(v[i], to.p[run] + (int64_t)block * units + in);
    }
  }
};

__device__ inline void copy_piece(const Store& from, uint32_t sb, const Store& to, uint32_t db,
                                  int piece, const Pieces& p) {
  Piece(from, (int)sb, piece, p).store(to, db, p);
}

// f(block, piece) for the workgroup's pieces of n blocks; workgroup w of W.
template <typename F>
__device__ inline void for_pieces(const Pieces& p, int64_t n, uint32_t w, uint32_t W, F&& f) {
  int64_t i = p.by_per.div(w);
  int piece = (int)(w - (uint32_t)i * p.per);
  const uint32_t di = p.by_per.div(W);
  const int dp = (int)(W - di * p.per);
  while (i < n) {
    f(i, piece);
    i += di;
    piece += dp;
    if (piece >= p.per) {
      piece -= p.per;
      ++i;
    }
  }
}

// Blocks src[i] to dst[i], i below n and *count (null: n).
__global__ void __launch_bounds__(PT)
copy_kernel(const Store from, uint32_t from_blocks, const Store to, uint32_t to_blocks,
            const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int64_t n,
            const int32_t* __restrict__ count, const Pieces p) {
  if (count != nullptr) n = min(n, (int64_t)*count);
  for_pieces(p, n, blockIdx.x, gridDim.x, [&](int64_t i, int piece) {
    const uint32_t sb = (uint32_t)src[i], db = (uint32_t)dst[i];
    if (sb < from_blocks && db < to_blocks) copy_piece(from, sb, to, db, piece, p);
  });
}

// The first `movers` workgroups move the held blocks, list[i] to i; the others
// write tables whose entries are the blocks' places among the held ones, -1 where
// a row holds nothing, or `into` has no such block.
__global__ void __launch_bounds__(PT)
compact_kernel(const Store from, const Store to, uint32_t to_blocks, const Rows t,
               uint32_t num_blocks, const int32_t* __restrict__ list,
               const int32_t* __restrict__ number, const int32_t* __restrict__ used,
               int32_t* __restrict__ out, uint32_t movers, const Pieces p) {
  if (blockIdx.x < movers) {
    for_pieces(p, min(*used, (int)to_blocks), blockIdx.x, movers,
               [&](int64_t i, int piece) {
                 copy_piece(from, (uint32_t)list[i], to, (uint32_t)i, piece, p);
               });
    return;
  }
  const int parts = (t.width + ENTRIES - 1) / ENTRIES;
  for (int64_t u = blockIdx.x - movers; u < t.R * parts; u += gridDim.x - movers) {
    const int64_t r = parts == 1 ? u : u / parts;
    const int lo = (int)(u - r * parts) * ENTRIES, hi = min(t.width, lo + ENTRIES);
    const int held = t.held(r);
    for (int e = lo + threadIdx.x; e < hi; e += PT) {
      int32_t v = -1;
      if (e < held) {
        const uint32_t b = (uint32_t)t.tables[r * t.stride + e];
        if (b < num_blocks) v = number[b];
        if (v >= (int)to_blocks) v = -1;
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
  int part;  // the block that its last tokens are in, if that is not full; -1: none
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

// Whether e is the number (child, entry) of a whole entry that names block b.
__device__ inline bool whole_entry(const Rows& t, const int32_t* parents, int64_t F, uint32_t b,
                                   uint32_t e) {
  if (e >= (uint64_t)F * t.width) return false;
  const uint32_t j = e >> 31 ? e / t.width : t.by_width.div(e);
  const int c = (int)(e - j * (uint32_t)t.width);
  const int64_t r = parents[j];
  return r >= 0 && r < t.R && (uint32_t)t.tables[r * t.stride + c] == b &&
         c < (int)((uint32_t)max(t.seq[r], 0) / t.bs);
}

// A workgroup per child: its row of the new tables, its length, the block it
// ends in; and where a block is, the number of some child's whole entry that
// names it (nothing is cleared before, as for mark_kernel).
__global__ void __launch_bounds__(PT)
fork_mark_kernel(const Rows t, const int32_t* __restrict__ parents, int64_t F,
                 uint32_t num_blocks, uint32_t* __restrict__ entry, int32_t* __restrict__ part,
                 int32_t* __restrict__ out, int32_t* __restrict__ out_seq) {
  const int64_t j = blockIdx.x;
  const Child c = child_of(t, parents, j, num_blocks);
  // A parent's marks are made once, or nearly: by the first of the last 1024
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
        if (!seen) entry[b] = (uint32_t)(j * t.width + e);
      }
    } else if (e == c.whole) {
      v = c.part;
    }
    out[j * t.width + e] = v;
  }
  if (threadIdx.x == 0) {
    out_seq[j] = c.seq;
    part[j] = c.part;
  }
}

// Child j's new block b, the k-th of the free list.
__device__ inline int32_t fresh_block(const int32_t* free_blocks, int64_t num_free, int64_t k,
                                      uint32_t num_blocks) {
  const int32_t b = k < num_free ? free_blocks[k] : -1;
  return (uint32_t)b < num_blocks ? b : -1;
}

__device__ inline int64_t last_entry(const Rows& t, int64_t j, const int32_t* out_seq) {
  return j * t.width + (uint32_t)out_seq[j] / t.bs;
}

// Up to FEW children: a workgroup per child and piece finds by itself which
// children get a block of their own (those that another ends in, in LDS), and
// copies.  Bound by latency, a chain of five loads: 64 children of 8 rows, 3.8 MB
// moved, 5.8 us (and 3.1 for the marks); with launches for clearing, placing and
// copying 2.3 + 2.7 + 13.
constexpr int FEW = 1024, SLOTS = 2 * FEW;
__global__ void __launch_bounds__(PT)
fork_few_kernel(const Rows t, const int32_t* __restrict__ parents, int F, uint32_t num_blocks,
                const uint32_t* __restrict__ entry, const int32_t* __restrict__ part,
                const int32_t* __restrict__ free_blocks, int64_t num_free,
                int32_t* __restrict__ out, const int32_t* __restrict__ out_seq,
                int32_t* __restrict__ taken, const Store store, const Pieces p) {
  constexpr int PER = FEW / PT;
  __shared__ int keys[SLOTS], lowest[SLOTS];
  __shared__ int s[PT / 64];
  const int j = (int)p.by_per.div(blockIdx.x), piece = (int)blockIdx.x - j * p.per;
  int mine[PER];
  const int own = part[j];
  // On its way while it is found out whether and where to it is copied.
  const Piece data(store, own, piece, p);
  bool copies = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int k = i * PT + threadIdx.x;
    mine[i] = k < F ? part[k] : -1;
    copies |= k < j && mine[i] == own;
  }
  // Most children need no copy; the first workgroup counts them all the same.
  if (blockIdx.x != 0) {
    if (own < 0) return;
    copies = __syncthreads_or(copies || (threadIdx.x == 0 &&
                                         whole_entry(t, parents, F, own, entry[own])));
    if (!copies) return;
  }
  bool whole[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    whole[i] = mine[i] >= 0 && whole_entry(t, parents, F, mine[i], entry[mine[i]]);
  for (int i = threadIdx.x; i < SLOTS; i += PT) {
    keys[i] = -1;
    lowest[i] = INT32_MAX;
  }
  __syncthreads();
  int slot[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (mine[i] < 0) continue;
    // (at most half of the slots are ever taken: this ends)
    int h = (int)((uint32_t)mine[i] * 2654435761u >> 21) & (SLOTS - 1);
    for (;;) {
      const int was = atomicCAS(&keys[h], -1, mine[i]);
      if (was == -1 || was == mine[i]) break;
      h = (h + 1) & (SLOTS - 1);
    }
    atomicMin(&lowest[h], i * PT + (int)threadIdx.x);
    slot[i] = h;
  }
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int k = i * PT + threadIdx.x;
    const bool c = mine[i] >= 0 && (whole[i] || lowest[slot[i]] != k);
    all += c;
    before += c && k < j;
  }
  wg_scan<PT>(before, s, &before);
  wg_scan<PT>(all, s, &all);
  if (blockIdx.x == 0 && threadIdx.x == 0) *taken = all;
  if (blockIdx.x == 0) {  // does child 0 itself need one?
    copies = __syncthreads_or(threadIdx.x == 0 && mine[0] >= 0 && whole[0]);
    if (!copies) return;
  }
  const int32_t b = fresh_block(free_blocks, num_free, before, num_blocks);
  if (piece == 0 && threadIdx.x == 0) out[last_entry(t, j, out_seq)] = b;
  if (b >= 0) data.store(store, (uint32_t)b, p);
}

// Any number of children: one workgroup finds them (a call with 1024 children of 512
// rows takes 21 us with the kernel above; 1025 / 4000 / 20000 / 200000 / 10^6 here
// 26 / 43 / 139 / 1239 / 6430, ~6 ns a child), with the lowest child that
// ends in a block in `first`.
constexpr int FT = 1024;
__global__ void __launch_bounds__(FT)
fork_place_kernel(const Rows t, const int32_t* __restrict__ parents, int64_t F,
                  uint32_t num_blocks, const uint32_t* __restrict__ entry,
                  const int32_t* __restrict__ part, int32_t* first,
                  const int32_t* __restrict__ free_blocks, int64_t num_free,
                  int32_t* __restrict__ out, const int32_t* __restrict__ out_seq,
                  int32_t* __restrict__ dst, int32_t* __restrict__ src,
                  int32_t* __restrict__ taken) {
  __shared__ int s[FT / 64];
  // (Agent scope: what this workgroup's other waves wrote is past their caches.)
  for (int64_t j = threadIdx.x; j < F; j += FT)
    if (part[j] >= 0)
      __hip_atomic_store(first + part[j], INT32_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __threadfence();
  __syncthreads();
  for (int64_t j = threadIdx.x; j < F; j += FT)
    if (part[j] >= 0)
      __hip_atomic_fetch_min(first + part[j], (int)j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __threadfence();
  __syncthreads();
  int base = 0;
  for (int64_t j0 = 0; j0 < F; j0 += FT) {
    const int64_t j = j0 + threadIdx.x;
    const int mine = j < F ? part[j] : -1;
    const bool copy =
        mine >= 0 && (__hip_atomic_load(first + mine, __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT) != (int)j ||
                      whole_entry(t, parents, F, mine, entry[mine]));
    int all;
    const int at = base + wg_scan<FT>(copy, s, &all) - 1;
    if (copy) {
      const int32_t b = fresh_block(free_blocks, num_free, at, num_blocks);
      src[at] = mine;
      dst[at] = b;
      out[last_entry(t, j, out_seq)] = b;
    }
    base += all;
  }
  if (threadIdx.x == 0) *taken = base;
}

// ------------------------------------------------- workspaces, launches

struct Names {
  uint32_t* entry;
  uint64_t* masks;
  int32_t* counts;
  int64_t chunks;
  Names(Carve& w, int64_t num_blocks) : chunks((num_blocks + CHUNK - 1) / CHUNK) {
    entry = w.take<uint32_t>((size_t)num_blocks);
    masks = w.take<uint64_t>((size_t)chunks * CHUNK / 64);
    counts = w.take<int32_t>((size_t)chunks);
  }
};

uint32_t grid_for(int64_t items, int per_cu) {
  const int64_t most = (int64_t)device_shape().cus * per_cu;
  return (uint32_t)std::max<int64_t>(1, std::min(items, most));
}

int64_t row_parts(const Kv4Tables& t) { return t.R * ((t.max_blocks + ENTRIES - 1) / ENTRIES); }

Rows rows_of(const Kv4Tables& t, int64_t bs) {
  return Rows{t.tables, t.stride, t.seq, t.R, (int)t.max_blocks, (uint32_t)bs,
              FastDiv((uint32_t)t.max_blocks)};
}

__global__ void zero_kernel(int32_t* p) { *p = 0; }

template <bool FREE>
void launch_names(const Kv4Tables& t, int64_t bs, int64_t num_blocks, const Names& n,
                  int32_t* list, int32_t* number, int32_t* total, hipStream_t s) {
  if (num_blocks == 0) {
    hipLaunchKernelGGL(zero_kernel, dim3(1), dim3(1), 0, s, total);
    return;
  }
  const Rows r = rows_of(t, bs);
  const dim3 chunks((uint32_t)n.chunks);
  if (num_blocks <= kSmallBlocks && t.R * t.max_blocks <= kSmallEntries) {
    hipLaunchKernelGGL(names_small_kernel<FREE>, chunks, dim3(ST), 0, s, r, (uint32_t)num_blocks,
                       list, number, total);
    return;
  }
  if (row_parts(t) > 0)
    hipLaunchKernelGGL(mark_kernel, dim3(grid_for(row_parts(t), 16)), dim3(PT), 0, s, r,
                       (uint32_t)num_blocks, n.entry);
  hipLaunchKernelGGL(count_kernel, chunks, dim3(PT), 0, s, r, num_blocks, n.entry, n.masks,
                     n.counts);
  hipLaunchKernelGGL(list_kernel<FREE>, chunks, dim3(PT), 0, s, num_blocks, n.masks, n.counts,
                     list, number, total);
}

// (a launch has less than 2^32 threads: huge blocks are left to copy_kernel's loop)
bool few(int64_t F, const Pieces& p) { return F <= FEW && F * p.per < (int64_t)1 << 23; }

uint32_t copy_grid(int64_t blocks, const Pieces& p) { return grid_for(blocks * p.per, 8); }

}  // namespace

size_t free_blocks_workspace_bytes(int64_t num_blocks) {
  Carve w(nullptr);
  Names n(w, num_blocks);
  return w.used;
}

int launch_free_blocks(const Kv4Tables& t, int64_t bs, int64_t num_blocks, int32_t* free_blocks,
                       int32_t* count, void* ws, hipStream_t s) {
  Carve w(ws);
  launch_names<true>(t, bs, num_blocks, Names(w, num_blocks), free_blocks, nullptr, count, s);
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
  launch_names<false>(t, c.block_size, c.num_blocks, n, list, number, used, s);
  const Pieces p(c);
  const int64_t most = std::min(c.num_blocks, into.num_blocks);
  const uint32_t movers = most > 0 ? copy_grid(most, p) : 0;
  const uint32_t writers = row_parts(t) > 0 ? grid_for(row_parts(t), 2) : 0;
  if (movers + writers > 0)
    hipLaunchKernelGGL(compact_kernel, dim3(movers + writers), dim3(PT), 0, s, Store(c),
                       Store(into), (uint32_t)into.num_blocks, rows_of(t, c.block_size),
                       (uint32_t)c.num_blocks, list, number, used, new_tables, movers, p);
  return check_launch("kv4_compact");
}

int launch_kv4_copy_blocks(const fkc_kv4_cache& c, const int32_t* src, const fkc_kv4_cache& into,
                           const int32_t* dst, int64_t n, hipStream_t s) {
  const Pieces p(c);
  hipLaunchKernelGGL(copy_kernel, dim3(copy_grid(n, p)), dim3(PT), 0, s, Store(c),
                     (uint32_t)c.num_blocks, Store(into), (uint32_t)into.num_blocks, src, dst, n,
                     (const int32_t*)nullptr, p);
  return check_launch("kv4_copy_blocks");
}

size_t kv4_fork_workspace_bytes(const fkc_kv4_cache& c, int64_t F) {
  Carve w(nullptr);
  w.take<uint32_t>((size_t)c.num_blocks);
  w.take<int32_t>((size_t)F);
  if (!few(F, Pieces(c))) w.take<int32_t>((size_t)F * 2 + (size_t)c.num_blocks);
  return w.used;
}

int launch_kv4_fork(const fkc_kv4_cache& c, const Kv4Tables& t, const int32_t* parents, int64_t F,
                    const int32_t* free_blocks, int64_t num_free, int32_t* new_tables,
                    int32_t* new_seq, int32_t* taken, void* ws, hipStream_t s) {
  if (F == 0) {
    hipLaunchKernelGGL(zero_kernel, dim3(1), dim3(1), 0, s, taken);
    return check_launch("kv4_fork");
  }
  Carve w(ws);
  uint32_t* entry = w.take<uint32_t>((size_t)c.num_blocks);
  int32_t* part = w.take<int32_t>((size_t)F);
  const Rows r = rows_of(t, c.block_size);
  const uint32_t nb = (uint32_t)c.num_blocks;
  const Pieces p(c);
  hipLaunchKernelGGL(fork_mark_kernel, dim3((uint32_t)F), dim3(PT), 0, s, r, parents, F, nb,
                     entry, part, new_tables, new_seq);
  if (few(F, p)) {
    hipLaunchKernelGGL(fork_few_kernel, dim3((uint32_t)(F * p.per)), dim3(PT), 0, s, r, parents,
                       (int)F, nb, entry, part, free_blocks, num_free, new_tables, new_seq, taken,
                       Store(c), p);
    return check_launch("kv4_fork");
  }
  int32_t* first = w.take<int32_t>((size_t)F * 2 + (size_t)c.num_blocks);
  int32_t *src = first + c.num_blocks, *dst = src + F;
  hipLaunchKernelGGL(fork_place_kernel, dim3(1), dim3(FT), 0, s, r, parents, F, nb, entry, part,
                     first, free_blocks, num_free, new_tables, new_seq, dst, src, taken);
  hipLaunchKernelGGL(copy_kernel, dim3(copy_grid(F, p)), dim3(PT), 0, s, Store(c), nb, Store(c),
                     nb, src, dst, F, taken, p);
  return check_launch("kv4_fork");
}

}  // namespace fkc
