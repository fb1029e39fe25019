// Block tables and cache slots of a step's new tokens, from request lengths.
//
// With old = seq - new, have = ceil(old / bs) and need = ceil(seq / bs) - have,
// token i of request r is position p = old + i of it, in its block j = p / bs:
// a held one (j < have, read from the table) or the (j - have)-th new one,
// entry first[r] + j - have of the free list, first the running sum of need.
//
// One launch, one thread per token: a workgroup owns CHUNK consecutive tokens
// and scans the lengths itself (TILE requests at a time, in LDS), so no
// workgroup waits for another; the token at the start of a new block writes
// the table entry.  Bound by latency at every size: lengths -> scan -> search
// -> table or free list -> slot.  37 requests of one token 3.3 us, 2048 requests
// of 96000 tokens 8.9 us.
#include "device_util.hpp"
#include "fkc_internal.hpp"

namespace fkc {
namespace {

constexpr int BT = 256;        // threads per workgroup
constexpr int IPT = 8;         // requests per thread and tile
constexpr int TILE = BT * IPT;
constexpr int CHUNK = 1024;    // tokens per workgroup

struct Held {
  int old, have, need;
};

__device__ inline Held held_of(int seq, int nw, uint32_t bs, int* fresh) {
  seq = max(seq, 0);
  nw = min(max(nw, 0), seq);
  Held h;
  h.old = seq - nw;
  h.have = (int)(((uint32_t)h.old + bs - 1) / bs);
  h.need = (int)(((uint32_t)seq + bs - 1) / bs) - h.have;
  *fresh = nw;
  return h;
}

__global__ void __launch_bounds__(BT)
block_tables_kernel(const int32_t* __restrict__ seq, const int32_t* __restrict__ nw,
                    int R, int32_t* __restrict__ tables, int64_t table_stride,
                    int max_blocks, const int32_t* __restrict__ free_blocks,
                    int64_t num_free, uint32_t bs, int64_t num_tokens,
                    int32_t* __restrict__ slots, int32_t* __restrict__ cu_new,
                    int32_t* __restrict__ taken) {
  __shared__ int s_cu[TILE], s_first[TILE];
  __shared__ int s_tot[2][BT / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t lo = (int64_t)blockIdx.x * CHUNK;
  // The last workgroup also takes the tokens that slots has no room for:
  // their blocks are handed out all the same.
  const bool last = blockIdx.x + 1 == gridDim.x;
  const int64_t hi = last ? INT64_MAX : lo + CHUNK;
  int cu_base = 0, first_base = 0;
  for (int r0 = 0; r0 < R; r0 += TILE) {
    const int n = min(TILE, R - r0);
    for (int i = t; i < TILE; i += BT) {
      int fresh = 0, need = 0;
      if (i < n) need = held_of(seq[r0 + i], nw[r0 + i], bs, &fresh).need;
      s_cu[i] = fresh;
      s_first[i] = need;
    }
    __syncthreads();
    int a[IPT], b[IPT], sa = 0, sb = 0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      a[i] = sa;
      b[i] = sb;
      sa += s_cu[t * IPT + i];
      sb += s_first[t * IPT + i];
    }
    int ia = wave_incl_scan(sa), ib = wave_incl_scan(sb);
    if (lane == 63) {
      s_tot[0][wave] = ia;
      s_tot[1][wave] = ib;
    }
    __syncthreads();
    int ta = 0, tb = 0;
    ia -= sa;
    ib -= sb;
#pragma unroll
    for (int w = 0; w < BT / 64; ++w) {
      if (w < wave) {
        ia += s_tot[0][w];
        ib += s_tot[1][w];
      }
      ta += s_tot[0][w];
      tb += s_tot[1][w];
    }
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      s_cu[t * IPT + i] = cu_base + ia + a[i];
      s_first[t * IPT + i] = first_base + ib + b[i];
    }
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = t; i < n; i += BT) cu_new[r0 + i] = s_cu[i];
    const int64_t end = min(hi, (int64_t)cu_base + ta);
    for (int64_t i = max(lo, (int64_t)cu_base) + t; i < end; i += BT) {
      // The last request that starts at or before token i (requests without
      // tokens start where the next one does).
      int x = 0, len = n;
      while (len > 1) {
        const int half = len >> 1;
        if (s_cu[x + half] <= i) x += half;
        len -= half;
      }
      int fresh;
      const Held h = held_of(seq[r0 + x], nw[r0 + x], bs, &fresh);
      const uint32_t p = (uint32_t)h.old + (uint32_t)(i - s_cu[x]);
      const int j = (int)(p / bs);
      const uint32_t within = p - (uint32_t)j * bs;
      int blk = -1;
      if (j < max_blocks) {
        int32_t* entry = tables + (int64_t)(r0 + x) * table_stride + j;
        if (j < h.have) {
          blk = *entry;
        } else {
          const int64_t f = (int64_t)s_first[x] + (j - h.have);
          // (below 0 where lengths that make no sense sum past 31 bits)
          if (f >= 0 && f < num_free) blk = free_blocks[f];
          if (within == 0) *entry = blk;
        }
      }
      // (a block whose slots 31 bits do not hold has none: cut to 32, their
      // numbers could be another block's)
      const uint64_t slot = (uint64_t)(uint32_t)blk * bs + within;
      if (i < num_tokens) slots[i] = blk < 0 || slot > INT32_MAX ? -1 : (int32_t)slot;
    }
    cu_base += ta;
    first_base += tb;
    if (blockIdx.x != 0 && cu_base >= hi) return;
    __syncthreads();  // the next tile overwrites s_cu, s_first and s_tot
  }
  for (int64_t i = max(lo, (int64_t)cu_base) + t; i < min(hi, num_tokens); i += BT)
    slots[i] = -1;
  if (blockIdx.x == 0 && t == 0) {
    cu_new[R] = cu_base;
    *taken = first_base;
  }
}

}  // namespace

int launch_block_tables(const int32_t* seq, const int32_t* nw, int R,
                        int32_t* tables, int64_t table_stride, int max_blocks,
                        const int32_t* free_blocks, int64_t num_free,
                        int block_size, int64_t num_tokens, int32_t* slots,
                        int32_t* cu_new, int32_t* taken, hipStream_t s) {
  const int64_t wgs = num_tokens > 0 ? (num_tokens + CHUNK - 1) / CHUNK : 1;
  hipLaunchKernelGGL(block_tables_kernel, dim3((uint32_t)wgs), dim3(BT), 0, s, seq,
                     nw, R, tables, table_stride, max_blocks, free_blocks, num_free,
                     (uint32_t)block_size, num_tokens, slots, cu_new, taken);
  return check_launch("block_tables");
}

}  // namespace fkc
