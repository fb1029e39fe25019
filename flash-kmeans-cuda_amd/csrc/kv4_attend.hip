// Attention over the 4-bit cache on the matrix cores.
//
// A column is one query of one head; the G query heads that share a cache head
// sit next to one another, so column c of a request is query c / G, head
// c % G.  For 16 columns and 32 tokens (v_mfma_f32_16x16x32):
//   S^T = K Q^T   A = 16 tokens x 32 features, B = 32 features x 16 columns
//   O^T = V^T P^T A = 16 features x 32 tokens, B = 32 tokens x 16 columns
// A lane (n = lane % 16, g = lane / 16) gets S^T for column n and tokens 4 g + i
// of a 16-token half, which is what it has to hold of P^T if the 32 tokens of
// the second product are counted as (half, i) within g: no value changes its
// lane.  Features are counted freely in both products, so that every lane's
// codes are contiguous: lane (n, g) of the first reads the D / 4 features from
// g D / 4 on of token n, feature row n of the second is the D / 16 features from
// n D / 16 on.
//
// Codes become 16-bit levels by a table in LDS: one byte holds two codes, and
// entry b of the head's table the pair of levels (b & 15, b >> 4).  An entry is
// 256 bytes: the key pair once for each of 32 banks, then the value pair, so 32
// lanes with any 32 bytes read 32 banks, and the address (byte, lane offset) is
// one v_perm of the codes: per two elements one vector and one LDS operation.
// The products are then of levels, exact in 16 bits.  A token's scales stay
// outside: the key's multiplies the score, the value's the weight.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "device_util.hpp"
#include "fkc_internal.hpp"
#include "kv4_shares.hpp"
#include "kv4_tile.hpp"

namespace fkc {
namespace {

// Work of a launch.  An item is a tile of a request under one cache head; it
// weighs the tokens it sees, in granules of GR, and kItem granules more in
// front for what an item costs by itself.  The items in order (head, request,
// tile) are cut into equal shares, one per workgroup, wherever the cuts fall:
// lengths of any mixture fill the chip evenly, a workgroup meets few heads
// (whose tables it has to fill), and an item that is cut is joined afterwards.
//
// j tiles of a request weigh a sum in closed form (kv4_shares.hpp), from which a
// tile is found again without a list of them.  (A weight only has to be the
// same for everyone; what a share takes is in tokens.)
struct Item {
  int hc;
  Tile t;
  int n;   // its weight
  int at;  // where the share begins in it
};

template <int COLS>
__device__ inline void request(const Args& a, int r, Tile& t, int& tiles) {
  t.req = r;
  if (a.cu_q == nullptr) {
    t.row0 = r;
    t.nq = r < a.R ? 1 : 0;
  } else {
    t.row0 = min(max(a.cu_q[min(r, a.R)], 0), a.T);
    const int next = r < a.R ? min(max(a.cu_q[r + 1], 0), a.T) : a.T;
    t.nq = r <= a.R ? max(next - t.row0, 0) : 0;
  }
  t.end = tokens_of(a, r);
  tiles = (int)(((int64_t)t.nq * a.G + COLS - 1) / COLS);
}

// Weight of the first j tiles.
template <int COLS, int GR>
__device__ inline int weight(const Args& a, const Tile& t, int j) {
  return kv4_weight(COLS, GR, a.G, a.causal != 0, t.nq, t.end, j);
}

// Running sums of the requests' weights, THREADS slices of `per` requests.
template <int COLS, int THREADS, int GR>
struct Shares {
  int* s_pre;  // LDS: THREADS + THREADS / 64 rounded to a multiple of 4, then
               // four numbers of each request where every thread has one
  int per, total;
  static constexpr int kInts = THREADS + (THREADS / 64 + 3) / 4 * 4 + THREADS * 4;
  __device__ inline int4* s_req() const {
    return reinterpret_cast<int4*>(s_pre + THREADS + (THREADS / 64 + 3) / 4 * 4);
  }
  __device__ inline Shares(int* lds, int p, int n) : s_pre(lds), per(p), total(n) {}
  __device__ inline Shares(const Args& a, int* lds) : s_pre(lds) {
    const int rt = a.R + (a.cu_q != nullptr ? 1 : 0);
    per = (rt + THREADS - 1) / THREADS;
    int sum = 0;
    for (int i = 0; i < per; ++i) {
      const int r = threadIdx.x * per + i;
      if (r >= rt) break;
      Tile t;
      int tiles;
      request<COLS>(a, r, t, tiles);
      sum += weight<COLS, GR>(a, t, tiles);
      if (per == 1) s_req()[r] = int4{t.row0, t.nq, t.end, tiles};
    }
    const int incl = wave_incl_scan(sum);
    int* s_wave = s_pre + THREADS;
    if ((threadIdx.x & 63) == 63) s_wave[threadIdx.x >> 6] = incl;
    lds_barrier();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      before += w < (int)(threadIdx.x >> 6) ? s_wave[w] : 0;
      total += s_wave[w];
    }
    s_pre[threadIdx.x] = before + incl - sum;
    lds_barrier();
    total = __builtin_amdgcn_readfirstlane(total);
  }
  // The item that place u (below total) of a head's falls into.
  __device__ inline Item find(const Args& a, int hc, int u) const {
    int j = -1;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i)
      j += __builtin_popcountll(__ballot(s_pre[i * 64 + (threadIdx.x & 63)] <= u));
    u -= __builtin_amdgcn_readfirstlane(s_pre[j]);
    Item x;
    x.hc = hc;
    int tiles;
    if (per == 1) {
      const int4 q = s_req()[j];
      x.t.req = j;
      x.t.row0 = __builtin_amdgcn_readfirstlane(q.x);
      x.t.nq = __builtin_amdgcn_readfirstlane(q.y);
      x.t.end = __builtin_amdgcn_readfirstlane(q.z);
      tiles = __builtin_amdgcn_readfirstlane(q.w);
    } else {
      for (int r = j * per;; ++r) {
        request<COLS>(a, r, x.t, tiles);
        const int w = weight<COLS, GR>(a, x.t, tiles);
        if (u < w || r >= a.R) break;
        u -= w;
      }
    }
    int tile = 0;  // the last whose weights before it are u at most
    for (int len = tiles; len > 1;) {
      const int half = len >> 1;
      if (weight<COLS, GR>(a, x.t, tile + half) <= u) tile += half;
      len -= half;
    }
    const int w = weight<COLS, GR>(a, x.t, tile);
    x.n = weight<COLS, GR>(a, x.t, tile + 1) - w;
    // Query offsets that do not ascend can sum past 32 bits: within the item all
    // the same, so that every share goes forward and ends.
    x.at = min(max(u - w, 0), x.n - 1);
    x.t.col0 = tile * COLS;
    return x;
  }
};

// A share as a workgroup walks through it, item by item.
template <int COLS, int THREADS, int GR>
struct Walk {
  int64_t u = 0, u_end = 0, share = 1;  // places over all heads
  int per_head = 1;
  int* s_pre;
  // The item at hand: its tokens from .. to of the lim that its last column
  // sees are the share's; more: shares after this one that hold some of it.
  Item x;
  int from, to, lim, more;
  __device__ inline Walk(const Args& a, int* lds) : s_pre(lds) {
    const Shares<COLS, THREADS, GR> sh(a, lds);
    per_head = sh.total;
    const int64_t all = (int64_t)per_head * a.heads;
    share = max((all + gridDim.x - 1) / gridDim.x, (int64_t)a.min_share);
    share = scalar64(share);
    u = blockIdx.x * share;
    u_end = scalar64(min(u + share, all));
    if (threadIdx.x == 0) a.desc[blockIdx.x].x = 0;
  }
  __device__ inline bool next(const Args& a) {
    while (u < u_end) {
      const Shares<COLS, THREADS, GR> sh(
          s_pre, (a.R + (a.cu_q != nullptr) + THREADS - 1) / THREADS, per_head);
      const int hc = (int)(u / per_head);
      x = sh.find(a, hc, (int)(u - (int64_t)hc * per_head));
      // The same in every lane, which the compiler cannot see of loaded values.
      auto scalar = [](int& v) { v = __builtin_amdgcn_readfirstlane(v); };
      scalar(x.t.req), scalar(x.t.row0), scalar(x.t.nq), scalar(x.t.end), scalar(x.t.col0);
      scalar(x.n), scalar(x.at);
      const int end = (int)min((int64_t)x.n, x.at + (u_end - u));
      u += end - x.at;
      const int last = min(x.t.col0 + COLS, x.t.nq * a.G) - 1;
      lim = sees(a, x.t, (int)a.gdiv.div(last));
      auto tokens = [&](int place) {
        return place == x.n ? lim : (int)min((int64_t)max(place - kItem, 0) * GR, (int64_t)lim);
      };
      from = tokens(x.at);
      to = tokens(end);
      const int full = min(x.n, kItem + (lim + GR - 1) / GR);  // place where to is lim
      more = (int)((max(full - end, 0) + share - 1) / share);
      scalar(from), scalar(to), scalar(lim), scalar(more);
      u = scalar64(u);
      // The share may hold none of the item's tokens; of an item without any
      // the last place stands for it.
      if (from < to || (lim == 0 && end == x.n)) return true;
    }
    return false;
  }
  __device__ inline bool cut() const { return from > 0 || to < lim; }
  // A share cuts the item before it and the one after it at most.
  __device__ inline int64_t slot() const { return (int64_t)blockIdx.x * 2 + (from > 0 ? 0 : 1); }
  // For the join, by one thread: a cut item that begins here.
  __device__ inline void announce(const Args& a) const {
    if (!cut() || from > 0) return;
    const int cols = min(COLS, x.t.nq * a.G - x.t.col0);
    a.desc[blockIdx.x] = int4{more + 1, x.t.row0, x.t.col0, cols << 16 | x.hc};
  }
  // One item per workgroup, no cuts, without the sums.
  __device__ inline bool whole(const Args& a) {
    // Heads first: consecutive workgroups go to the eight XCDs in turn, and
    // every head has as much to do as the next.
    const int tile = blockIdx.x / a.heads;
    x.hc = blockIdx.x - tile * a.heads;
    if (!find_tile<COLS>(a, tile, x.t)) return false;
    auto scalar = [](int& v) { v = __builtin_amdgcn_readfirstlane(v); };
    scalar(x.t.req), scalar(x.t.row0), scalar(x.t.nq), scalar(x.t.end), scalar(x.t.col0);
    const int last = min(x.t.col0 + COLS, x.t.nq * a.G) - 1;
    from = 0;
    to = lim = __builtin_amdgcn_readfirstlane(sees(a, x.t, (int)a.gdiv.div(last)));
    more = 0;
    return true;
  }
  __device__ inline explicit Walk(int* lds) : s_pre(lds) {}
};

__device__ inline const Args& arguments() { return arguments_as<Args>(); }

// The split form, for few columns: the waves of a workgroup share NT tiles of 16
// columns and take 32 tokens each in turn, with their own running maxima and
// sums; they are joined in LDS at the end of an item, cut items by a second
// kernel.  Codes go straight from memory to registers, through the table and
// into the products.
//
// Bound by memory where contexts are long: one query of each of 64 ragged
// requests over 628 MB of bf16 cache (D = 128) takes 131 us, 4.8 TB/s, where a
// large copy moves 4.7 and reading alone 6.4, and the same kernel without
// look-ups and products takes 119.  An item costs about 8 us by itself (its
// table, dependent loads, joining the waves), which bounds short contexts: 48
// requests of 16 heads of 64 columns, 70 MB, take 37 us.  Two workgroups of
// eight waves per CU: four waves a SIMD with 128 registers; two with twice the
// registers and three tiles in flight measured slower (171 us to 148 then).
template <int DT, int D, int NT, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, WAVES / 2)
kv4_split_kernel(const Args args) {
  constexpr int COLS = 16 * NT, THREADS = WAVES * 64, UNIT = WAVES * 32;
  constexpr int KS = D / 32;  // steps of the first product
  constexpr int ND = D / 16;  // feature tiles of the second
  extern __shared__ __align__(16) char lds[];
  float2* sml = reinterpret_cast<float2*>(lds + kTable);
  int* s_pre = reinterpret_cast<int*>(lds + kTable + kJoin);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  typedef Walk<COLS, THREADS, UNIT> W;
  W k = args.whole ? W(s_pre) : W(arguments(), s_pre);
  if (!(args.whole ? k.whole(arguments()) : k.next(arguments()))) return;
  for (;;) {
    // Opaque, so that what derives from it is computed per item, not kept in
    // registers over the whole share.
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const Args& a = arguments();
    const int lane = tid & 63, n = lane & 15, g = lane >> 4;
    const uint32_t loff = (uint32_t)(lane & 31) * 4;
    const Item& x = k.x;
    const Tile& t = x.t;
    const int ncols = t.nq * a.G;
    const int lim_min = sees(a, t, (int)a.gdiv.div(t.col0)), lim_max = k.lim;
    const int t0 = k.from, t1 = k.to;
    const int ntile = max(t1 - t0 + 31, 0) / 32;
    const Const32 blocks = (Const32)(a.tables + (int64_t)t.req * a.table_stride);

    // Cache blocks of a tile's two halves, and from them their 16-slot group
    // over all heads: -1 where there is no block.
    auto load_blocks = [&](int it, int (&blk)[2]) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int tok = t0 + it * 32 + 16 * j;
        blk[j] = tok < t1 ? blocks[a.bs.div(tok)] : -1;
      }
    };
    auto groups = [&](int it, const int (&blk)[2], int (&base)[2]) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t b = (uint32_t)blk[j];
        const uint32_t tok = t0 + it * 32 + 16 * j;
        const uint32_t in = (tok - a.bs.div(tok) * a.bs.d) / 16;
        base[j] = b < a.num_blocks ? (int)((b * (uint32_t)a.heads + x.hc) * (a.bs.d / 16) + in)
                                   : -1;
      }
    };
    int blk[2], base[2], nbase[2];
    load_blocks(wave, blk);

    // Query and head of a column of the tile's; row -1 past the last.
    auto column = [&](const Args& a, int col, int& row, int& head, int& i) {
      col += t.col0;
      i = (int)a.gdiv.div(min(col, ncols - 1));
      row = col < ncols ? t.row0 + i : -1;
      head = x.hc * a.G + (min(col, ncols - 1) - i * a.G);
    };
    int lim[NT];
    u32x4 qf[NT][KS];
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      int row, head, i;
      column(a, 16 * y + n, row, head, i);
      const bool ok = row >= 0;
      lim[y] = ok ? sees(a, t, i) : 0;
      const uint16_t* qp = a.q + max(row, t.row0) * a.q_ts + head * a.q_hs + g * (D / 4);
#pragma unroll
      for (int s = 0; s < KS; ++s)
        qf[y][s] = (ok ? *reinterpret_cast<const u32x4*>(qp + s * 8) : u32x4{0, 0, 0, 0}) ^
                   a.qsign;
    }
    const Lane<D> lanes(n, g);
    Codes<D> cur;
    groups(wave, blk, base);
    if (wave < ntile) {
      load_keys<D>(a, base, lanes, cur);
      load_scales<D>(a, base, lanes, cur);
      load_values<D>(a, base, lanes, cur);
    }
    load_blocks(wave + WAVES, blk);
    fill_table<THREADS>(a, x.hc, lds, tid);
    lds_barrier();

    State<DT, D, NT> st;
    st.clear();
    // What a tile has used up is fetched for the next one at once, after the last
    // tile slot 0's (a load that may or may not be on its way would have to be
    // waited for with every older one), into the same registers: with a second
    // set of them four waves a SIMD do not fit, and it is they that hide the loads'
    // latency.
    for (int it = wave; it < ntile; it += WAVES) {
      groups(it + WAVES, blk, nbase);
      load_blocks(it + 2 * WAVES, blk);

      f32x4 s[NT][2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          u32x4 kf;
#pragma unroll
          for (int b = 0; b < 4; ++b) kf[b] = lookup<0>(cur.k[j][c], b, loff);
#pragma unroll
          for (int y = 0; y < NT; ++y)
            s[y][j] = mfma<DT>(kf, qf[y][c], c ? s[y][j] : f32x4{0.f, 0.f, 0.f, 0.f});
        }
      load_keys<D>(a, nbase, lanes, cur);
      const uint2 kw[2] = {cur.ks[0], cur.ks[1]}, vw[2] = {cur.vs[0], cur.vs[1]};
      load_scales<D>(a, nbase, lanes, cur);
      u32x4 pf[NT];
      st.weights(s, kw, vw, t0 + it * 32 + 32 > lim_min || (base[0] | base[1]) < 0, base[0],
                 base[1], t0 + it * 32 + 4 * g, lim, lim_max, a.zscale, pf);
      // Features 2 b and 2 b + 1 of the lane's row, two tokens a dword.
#pragma unroll
      for (int v = 0; v < (ND + 7) / 8; ++v) {
        uint32_t even[4], odd[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          pair_tokens(cur.v[k >> 1][2 * (k & 1)][v], cur.v[k >> 1][2 * (k & 1) + 1][v], even[k],
                      odd[k]);
#pragma unroll
        for (int b = 0; b < (ND < 8 ? ND / 2 : 4); ++b) {
          u32x4 lo, hi;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            lo[k] = lookup<128>(even[k], b, loff);
            hi[k] = lookup<128>(odd[k], b, loff);
          }
#pragma unroll
          for (int y = 0; y < NT; ++y) {
            st.o[y][8 * v + 2 * b] = mfma<DT>(lo, pf[y], st.o[y][8 * v + 2 * b]);
            st.o[y][8 * v + 2 * b + 1] = mfma<DT>(hi, pf[y], st.o[y][8 * v + 2 * b + 1]);
          }
        }
      }
      load_values<D>(a, nbase, lanes, cur);
      base[0] = nbase[0];
      base[1] = nbase[1];
    }

    st.join_lanes();
    // Join the waves that had tokens: their outputs, relative to the largest
    // maximum, go to LDS as rows of features (over the table, 16-byte pieces
    // turned by the column so that no two lanes meet in a bank) and are summed
    // as they are written.
    const int waves = min(ntile, WAVES);
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      if (y) lds_barrier();  // the last tile's pieces are read
      const float rel = st.base2(y, a.zscale);
      if (g == 0) sml[wave * 16 + n] = float2{rel, st.l[y]};
      lds_barrier();
      const Args& a = arguments();
      float top = kLowest;
      for (int w = 0; w < waves; ++w) top = fmaxf(top, sml[w * 16 + n].x);
      const float f = __builtin_amdgcn_exp2f(rel - top);
      f32x4* so = reinterpret_cast<f32x4*>(lds);
      if (wave < waves) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < ND / 4; ++d) {
            const int piece = (4 * g + i) * (ND / 4) + d;
            so[(wave * 16 + n) * (D / 4) + (piece ^ n)] =
                f32x4{st.o[y][4 * d][i], st.o[y][4 * d + 1][i], st.o[y][4 * d + 2][i],
                      st.o[y][4 * d + 3][i]} * f;
          }
      }
      lds_barrier();
      const bool cut = k.cut();
      const int64_t slot = k.slot();
#pragma unroll 1
      for (int e = tid; e < 16 * D / 4; e += THREADS) {
        const int col = e / (D / 4), piece = e % (D / 4);
        int row, head, i;
        column(a, 16 * y + col, row, head, i);
        if (row < 0) continue;
        float top = kLowest, sum = 0.f;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < waves; ++w) top = fmaxf(top, sml[w * 16 + col].x);
        for (int w = 0; w < waves; ++w) {
          const float2 ml = sml[w * 16 + col];
          sum += ml.y * __builtin_amdgcn_exp2f(ml.x - top);
          v += so[(w * 16 + col) * (D / 4) + (piece ^ col)];
        }
        const int64_t at = (int64_t)row * a.H + head;
        if (!cut) {
          const float f = inverse(sum);
          uint2 w;
          w.x = pack2<DT>(v[0] * f, v[1] * f);
          w.y = pack2<DT>(v[2] * f, v[3] * f);
          *reinterpret_cast<uint2*>(a.out + at * D + 4 * piece) = w;
          if (piece == 0 && a.lse != nullptr)
            a.lse[at] = log_sum(top, sum);
        } else {
          const int64_t at = slot * COLS + 16 * y + col;
          *reinterpret_cast<f32x4*>(a.part + at * D + 4 * piece) = v;
          if (piece == 0)
            *reinterpret_cast<float2*>(a.part_ml + 2 * at) = float2{top, sum};
        }
      }
    }
    if (args.whole) return;
    if (tid == 0) k.announce(arguments());
    if (!k.next(arguments())) return;
    lds_barrier();  // the next item fills the table again
  }
}

// The wide form, for prompts: every wave has NT tiles of 16 columns of its own,
// and all of a workgroup's go over the same TT tokens at a time.  These are
// looked up once for all: each wave turns its share of the codes into the
// fragments of both products, laid out so that a fragment is read by 64 lanes
// in a row (16 bytes each, no bank conflict), in one of two buffers; while a
// tile is computed on, the next one is filled into the other.
//
// No unit is busy half of the time; what bounds it is that a wave's phases (score
// products, softmax, value products of 32 tokens) follow one another with two
// waves a SIMD to overlap them, and all eight meet at a barrier every TT tokens.
// Ragged prompts of 700 to 4096 tokens, 32 heads of 128 columns, bf16, 366 us a call
// (0.52 PFLOP/s): vector unit 46%, matrix cores 21%, LDS 18%, waves waiting for
// data or a barrier 37% and for an issue slot 22%; 341 if the buffers are neither
// loaded nor filled, 289 if the scores are packed as they are, 228 with neither.
// D = 256, where NT = 1 and a fragment of 1 KB feeds one product, 12000 to 16000
// tokens: 1002 us, 45 / 21 / 32 / 36 / 24%; 807 / 851 / 741.  Four waves with NT = 4,
// or NT = 3, need more registers than the compiler finds (spills cost more than
// the reads); waves that looked up for themselves were slower (prompts 438 to 420
// then, D = 256 1264 to 1044).
//
// Feature row n of fragment d of the second product is feature 32 (d / 2) + 2 n +
// d % 2: the two codes of one byte go to two fragments, and 16 lanes read 16
// bytes of a token.
template <int DT, int D, int NT, int TT>
__global__ void __launch_bounds__(512, 2)
kv4_wide_kernel(const Args args) {
  constexpr int WAVES = 8, COLS = 16 * NT * WAVES, THREADS = WAVES * 64;
  constexpr int KS = D / 32, ND = D / 16, HALVES = TT / 16, GROUPS = TT / 32;
  constexpr int KPW = HALVES * KS / WAVES;  // key fragments a wave fills
  constexpr int VW = GROUPS * ND / 2;       // waves that fill two value fragments
  static_assert(KPW >= 1 && KS % KPW == 0 && VW <= WAVES, "a wave fills within one half");
  constexpr int KBYTES = TT * D * 2, BUF = 2 * KBYTES;
  typedef int Groups __attribute__((ext_vector_type(HALVES)));
  extern __shared__ __align__(16) char lds[];
  int* s_pre = reinterpret_cast<int*>(lds + kTable + 2 * BUF);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kj = wave * KPW / KS, kc0 = wave * KPW % KS;  // its half, first step
  const int vg = wave % VW / (ND / 2), vu = wave % (ND / 2);  // its group, fragment pair
  int table = -1;  // head whose table is in LDS
  typedef Walk<COLS, THREADS, TT> W;
  W k = args.whole ? W(s_pre) : W(arguments(), s_pre);
  if (!(args.whole ? k.whole(arguments()) : k.next(arguments()))) return;
  for (;;) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const Args& a = arguments();
    const int lane = tid & 63, n = lane & 15, g = lane >> 4;
    const uint32_t loff = (uint32_t)(lane & 31) * 4;
    const Item& x = k.x;
    const Tile& t = x.t;
    const int ncols = t.nq * a.G;
    // The wave's columns, counted in the request, and what the first and the
    // last of them see.
    const int col0 = t.col0 + wave * 16 * NT;
    const int lim_min = sees(a, t, (int)a.gdiv.div(min(col0, ncols - 1)));
    const int lim_max =
        col0 < ncols ? sees(a, t, (int)a.gdiv.div(min(col0 + 16 * NT, ncols) - 1)) : 0;
    const int t0 = k.from, t1 = k.to, tiles = (max(t1 - t0, 0) + TT - 1) / TT;

    // The arguments that every tile needs, in scalar registers (left to itself
    // the compiler reads them again at each use, and waits).
    // (Global addresses by type: behind the asm nothing else says so, and a
    // load that might be LDS's would be waited for with every LDS read.)
    Global k_codes = (Global)a.k_codes, v_codes = (Global)a.v_codes;
    Global k_scales = (Global)a.k_scales, v_scales = (Global)a.v_scales;
    uint32_t bs = a.bs.d, bs_m = a.bs.m, num_blocks = a.num_blocks;
    int bs_sh = a.bs.sh, heads = a.heads;
    float zscale = a.zscale;
    asm volatile("" : "+s"(k_codes), "+s"(v_codes), "+s"(k_scales), "+s"(v_scales));
    asm volatile("" : "+s"(bs), "+s"(bs_m), "+s"(num_blocks), "+s"(bs_sh), "+s"(heads),
                 "+s"(zscale));
    const Const32 blocks = (Const32)(a.tables + (int64_t)t.req * a.table_stride);
    // 16-slot groups of a tile's halves over all heads, -1 where there is none.
    auto find_groups = [&](int tile, Groups& base) {
#pragma unroll
      for (int j = 0; j < HALVES; ++j) {
        const uint32_t tok = t0 + tile * TT + 16 * j;
        const uint32_t at = __umulhi(tok, bs_m) >> bs_sh;  // (block sizes are 16 at least)
        const uint32_t b = (int)tok < t1 ? (uint32_t)blocks[at] : 0xffffffffu;
        base[j] = b < num_blocks ? (int)((b * heads + x.hc) * (bs / 16) + (tok - at * bs) / 16)
                                 : -1;
      }
    };
    uint32_t kcode[KPW], vcode[8];
    uint2 ks[HALVES], vs[HALVES];
    auto pick = [](const Groups& base, int j) {
      int v = base[0];
#pragma unroll
      for (int i = 1; i < HALVES; ++i) v = j == i ? base[i] : v;
      return (int64_t)max(v, 0);  // a missing half reads slot 0
    };
    auto load_tile = [&](const Groups& base) {
      const Global kp = k_codes + pick(base, kj) * (16 * D / 2);
#pragma unroll
      for (int e = 0; e < KPW; ++e)
        kcode[e] = at<uint32_t>(kp, n * (D / 2) + g * (D / 8) + (kc0 + e) * 4);
      // (waves without value fragments load those of others)
      {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const Global vp = v_codes + pick(base, 2 * vg + j) * (16 * D / 2);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            vcode[4 * j + i] = at<uint8_t>(vp, (4 * g + i) * (D / 2) + 16 * vu + n);
        }
      }
    };
    auto load_scales = [&](const Groups& base, int j) {
      const int64_t row = (int64_t)max(base[j], 0) * 32;  // bytes
      ks[j] = at<uint2>(k_scales + row, 8 * g);
      vs[j] = at<uint2>(v_scales + row, 8 * g);
    };
    auto fill_buffer = [&](int tile) {
      char* buf = lds + kTable + (tile & 1) * BUF + lane * 16;
#pragma unroll
      for (int e = 0; e < KPW; ++e) {
        u32x4 f;
#pragma unroll
        for (int b = 0; b < 4; ++b) f[b] = lookup<0>(kcode[e], b, loff);
        *reinterpret_cast<u32x4*>(buf + (kj * KS + kc0 + e) * 1024) = f;
      }
      if (wave < VW) {
        u32x4 even, odd;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t b0 = vcode[2 * c], b1 = vcode[2 * c + 1];
          even[c] = lookup<128>((b0 & 15u) | (b1 << 4 & 0xf0u), 0, loff);
          odd[c] = lookup<128>(b0 >> 4 | (b1 & 0xf0u), 0, loff);
        }
        char* vb = buf + KBYTES + (vg * ND + 2 * vu) * 1024;
        *reinterpret_cast<u32x4*>(vb) = even;
        *reinterpret_cast<u32x4*>(vb + 1024) = odd;
      }
    };
    auto column = [&](const Args& a, int y, int& row, int& head, int& i) {
      const int col = col0 + 16 * y + n;
      i = (int)a.gdiv.div(min(col, ncols - 1));
      row = col < ncols ? t.row0 + i : -1;
      head = x.hc * a.G + (min(col, ncols - 1) - i * a.G);
    };

    Groups base, nbase;  // of this tile and the next
    find_groups(0, base);
    find_groups(1, nbase);
    if (tiles > 0) {
      load_tile(base);
#pragma unroll
      for (int j = 0; j < HALVES; ++j) load_scales(base, j);
    }
    int lim[NT];
    u32x4 qf[NT][KS];
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      int row, head, i;
      column(a, y, row, head, i);
      const bool ok = row >= 0;
      lim[y] = ok ? sees(a, t, i) : 0;
      const uint16_t* qp = a.q + max(row, t.row0) * a.q_ts + head * a.q_hs + g * (D / 4);
#pragma unroll
      for (int c = 0; c < KS; ++c)
        qf[y][c] = (ok ? *reinterpret_cast<const u32x4*>(qp + c * 8) : u32x4{0, 0, 0, 0}) ^
                   a.qsign;
    }
    if (table != x.hc) {  // (every look-up of the last item was before its last barrier)
      table = x.hc;
      fill_table<THREADS>(a, x.hc, lds, tid);
      lds_barrier();
    }
    if (tiles > 0) fill_buffer(0);
    if (tiles > 0) load_tile(nbase);
    lds_barrier();

    State<DT, D, NT> st;
    st.clear();
    for (int tile = 0; tile < tiles; ++tile) {
      Groups after;
      if (tile + 1 < tiles) fill_buffer(tile + 1);
      find_groups(tile + 2, after);
      // Past the last tile slot 0's codes, unused: a load that may or may not be
      // on its way would have to be waited for with every older one.
      load_tile(after);
      const char* buf = lds + kTable + (tile & 1) * BUF + lane * 16;
      auto group = [&](auto H) {
        constexpr int h = H.value;
        const int tok = t0 + tile * TT + 32 * h;
        const uint2 kw[2] = {ks[2 * h], ks[2 * h + 1]}, vw[2] = {vs[2 * h], vs[2 * h + 1]};
        load_scales(nbase, 2 * h);
        load_scales(nbase, 2 * h + 1);
        if (tok >= lim_max) return;  // none of the wave's columns sees them
        f32x4 s[NT][2];
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const u32x4 kf =
                *reinterpret_cast<const u32x4*>(buf + ((2 * h + j) * KS + c) * 1024);
#pragma unroll
            for (int y = 0; y < NT; ++y)
              s[y][j] = mfma<DT>(kf, qf[y][c], c ? s[y][j] : f32x4{0.f, 0.f, 0.f, 0.f});
          }
        u32x4 pf[NT];
        st.weights(s, kw, vw, tok + 32 > lim_min || (base[2 * h] | base[2 * h + 1]) < 0,
                   base[2 * h], base[2 * h + 1], tok + 4 * g, lim, lim_max, zscale, pf);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const u32x4 vf = *reinterpret_cast<const u32x4*>(buf + KBYTES + (h * ND + d) * 1024);
#pragma unroll
          for (int y = 0; y < NT; ++y) st.o[y][d] = mfma<DT>(vf, pf[y], st.o[y][d]);
        }
      };
      group(std::integral_constant<int, 0>{});
      if constexpr (GROUPS > 1) group(std::integral_constant<int, 1>{});
      base = nbase;
      nbase = after;
      lds_barrier();
    }

    st.join_lanes();
    {
      const Args& a = arguments();
#pragma unroll
      for (int y = 0; y < NT; ++y) {
        int row, head, i;
        column(a, y, row, head, i);
        if (row < 0) continue;
        if (!k.cut()) {
          const float f = inverse(st.l[y]);
          const int64_t at = (int64_t)row * a.H + head;
#pragma unroll
          for (int u = 0; u < ND / 2; ++u) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = pack2<DT>(st.o[y][2 * u][i] * f, st.o[y][2 * u + 1][i] * f);
            *reinterpret_cast<u32x4*>(a.out + at * D + 32 * u + 8 * g) = w;
          }
          if (g == 0 && a.lse != nullptr) a.lse[at] = log_sum(st.base2(y, a.zscale), st.l[y]);
        } else {
          const int64_t at = k.slot() * COLS + wave * 16 * NT + 16 * y + n;
#pragma unroll
          for (int u = 0; u < ND / 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; i += 2)
              *reinterpret_cast<f32x4*>(a.part + at * D + 32 * u + 8 * g + 2 * i) =
                  f32x4{st.o[y][2 * u][i], st.o[y][2 * u + 1][i], st.o[y][2 * u][i + 1],
                        st.o[y][2 * u + 1][i + 1]};
          if (g == 0)
            *reinterpret_cast<float2*>(a.part_ml + 2 * at) =
                float2{st.base2(y, a.zscale), st.l[y]};
        }
      }
    }
    if (args.whole) return;
    if (tid == 0) k.announce(arguments());
    if (!k.next(arguments())) return;
  }
}

// Granules of a share at least, and up to how many granules a context is never
// cut: every item then goes to a workgroup of its own, and nothing has to be
// joined by a second kernel.  (bf16, D = 128, 8 heads, 4 query heads each, one
// query, us: contexts of 1536 whole 16.2 / 16.8 / 24.7 for 1 / 8 / 64 requests,
// cut 17.2 / 19.2 / 29.7; of 3000 whole 24.6 / 25.0 / 39.3, cut 18.3 / 22.4 /
// 42.6.)
constexpr int kMinShare = 2, kWhole = 8, kWideWhole = 32;

struct Plan {
  bool wide;
  int nt;             // column tiles per wave
  int waves;
  bool whole;         // one item per workgroup
  int64_t wgs;
  int tiles_per_req;  // without cu_q
  int cols() const { return 16 * nt * (wide ? waves : 1); }
  size_t part_rows() const { return (size_t)wgs * 2 * cols(); }
};

constexpr int kWide = 8;  // waves of the wide form
constexpr int wide_tiles(int D) { return D == 256 ? 1 : 2; }
constexpr int wide_tokens(int D) { return D == 256 ? 32 : 64; }
constexpr int waves_of(int D) { return D == 256 ? 4 : 8; }

Plan make_plan(const fkc_kv4_cache& c, int64_t H, int64_t T, int64_t R, int64_t max_seq,
               bool ragged) {
  Plan p;
  const int64_t G = H / c.heads;
  // By the columns of an average request.  Measured on 8 requests of 4096
  // tokens, 8 heads of 4 query heads, bf16, us with one tile per workgroup /
  // with two / in the wide form, for so many columns each:
  //   D =  64    32: 25 / 25 / 52    96: 44 / 38 / 60    256:  86 /  72 /  89
  //             512: 148 / 114 / 111
  //   D = 128    32: 29 / 33 / 60    96: 54 / 49 / 74    256: 110 /  94 / 109
  //             512: 205 / 149 / 139
  //   D = 256    32: 51 / 77 / 84    96: 89 / 129 / 140  256: 193 / 268 / 171
  const int64_t avg = R > 0 ? T * G / R : 0;
  p.wide = avg > (c.D == 256 ? 224 : 448);
  p.nt = p.wide ? wide_tiles((int)c.D) : c.D < 256 && avg > 64 ? 2 : 1;
  p.waves = p.wide ? kWide : p.nt == 2 ? 4 : waves_of((int)c.D);
  const int64_t cols = p.cols();
  p.tiles_per_req = (int)((G + cols - 1) / cols);
  const int64_t tiles = ragged ? T * G / cols + R + 1 : R * p.tiles_per_req;
  p.whole = max_seq <= (p.wide ? kWideWhole * 32 : kWhole * 32 * p.waves) &&
            tiles * c.heads < kMostThreads / (64 * p.waves);
  p.wgs = p.whole ? tiles * c.heads : (p.wide ? 1 : 2) * (int64_t)device_shape().cus;
  return p;
}

template <int DT, int D, int COLS, int THREADS, typename K>
int launch(K kernel, std::atomic<uint64_t>& set, int bytes, const Args& a, const Plan& p,
           hipStream_t s) {
  // The attribute stays with the kernel: once per device is enough.
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess) dev = -1;
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  if ((set.load(std::memory_order_relaxed) & bit) == 0) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                            hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
      return fail(FKC_ERR_LAUNCH, "kv4_attend: %d bytes of LDS refused", bytes);
    set.fetch_or(bit, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL(kernel, dim3((uint32_t)p.wgs), dim3(THREADS), bytes, s, a);
  if (int rc = check_launch("kv4_attend")) return rc;
  if (p.whole) return FKC_OK;
  const int64_t cols = std::min<int64_t>(COLS, a.cu_q ? COLS : a.G);
  hipLaunchKernelGGL((kv4_join_kernel<DT, D, COLS>),
                     dim3((uint32_t)p.wgs, (uint32_t)std::min<int64_t>((cols + 3) / 4, 16)),
                     dim3(256), 0, s, a);
  return check_launch("kv4_attend (join)");
}

template <int DT, int D, int NT, int WAVES>
int launch_split(const Args& a, const Plan& p, hipStream_t s) {
  static std::atomic<uint64_t> set{0};
  return launch<DT, D, 16 * NT, WAVES * 64>(
      &kv4_split_kernel<DT, D, NT, WAVES>, set,
      kTable + kJoin + Shares<16 * NT, WAVES * 64, 1>::kInts * 4, a, p, s);
}

template <int DT, int D>
int launch_wide(const Args& a, const Plan& p, hipStream_t s) {
  static std::atomic<uint64_t> set{0};
  constexpr int NT = wide_tiles(D), TT = wide_tokens(D), COLS = 16 * NT * kWide;
  return launch<DT, D, COLS, kWide * 64>(
      &kv4_wide_kernel<DT, D, NT, TT>, set,
      kTable + 2 * (TT * D * 4) + Shares<COLS, kWide * 64, 1>::kInts * 4, a, p, s);
}

}  // namespace

size_t kv4_attend_workspace_bytes(const fkc_kv4_cache& c, int64_t H, int64_t T, int64_t R,
                                  int64_t max_seq) {
  const Plan p = make_plan(c, H, T, R, max_seq, true);
  if (p.whole) return 0;
  Carve w(nullptr);
  w.take<float>(p.part_rows() * c.D);
  w.take<float>(p.part_rows() * 2);
  w.take<int4>((size_t)p.wgs);
  return w.used;
}

int launch_kv4_attend(const fkc_kv4_cache& c, const Kv4Attend& x, void* ws, size_t,
                      hipStream_t s) {
  const Plan p = make_plan(c, x.H, x.T, x.R, x.max_seq, x.cu_q != nullptr);
  const int G = (int)(x.H / c.heads);
  // Weights of a head's items are summed in 32 bits.
  const int64_t most =
      kv4_most_weight(p.cols(), p.wide ? wide_tokens((int)c.D) : 32 * p.waves, G, x.max_seq);
  if (x.T * G / p.cols() + x.R + 1 > INT32_MAX / most)
    return fail(FKC_ERR_UNSUPPORTED, "kv4_attend: too many rows times tokens");
  Args a{(const uint16_t*)x.q.p, x.q.token_stride, x.q.head_stride,
         (const uint8_t*)c.k_codes, (const uint8_t*)c.v_codes,
         (const uint16_t*)c.k_scales, (const uint16_t*)c.v_scales,
         (const uint16_t*)c.k_levels, (const uint16_t*)c.v_levels,
         x.tables, x.table_stride, x.seq, x.cu_q, (uint16_t*)x.out, x.lse, nullptr, nullptr,
         nullptr, FastDiv((uint32_t)c.block_size), FastDiv((uint32_t)G), (uint32_t)c.num_blocks,
         (int)c.heads, (int)x.H, G, (int)x.T, (int)x.R, (int)x.max_seq, (int)x.causal,
         (int)p.whole, kMinShare, p.tiles_per_req,
         // (of scores times 0 the masked ones would be NaN)
         std::max(std::fabs(x.sm_scale) * kLog2e, 1e-30f),
         std::signbit(x.sm_scale) ? 0x80008000u : 0u};
  if (!p.whole) {
    Carve w(ws);
    a.part = w.take<float>(p.part_rows() * c.D);
    a.part_ml = w.take<float>(p.part_rows() * 2);
    a.desc = w.take<int4>((size_t)p.wgs);
  }
  return kv4_by_shape(c.dtype, c.D, [&](auto dt, auto d) {
    constexpr int DT = dt.value, DD = d.value;
    if (p.wide) return launch_wide<DT, DD>(a, p, s);
    if constexpr (DD < 256)
      if (p.nt == 2) return launch_split<DT, DD, 2, 4>(a, p, s);
    return launch_split<DT, DD, 1, waves_of(DD)>(a, p, s);
  });
}

}  // namespace fkc
