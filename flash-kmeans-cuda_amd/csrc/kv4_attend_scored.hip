// Attention over the 4-bit cache whose scores are capped, lowered with the
// distance, or masked row by row.  With p the position of a query among its
// request's tokens,
//   z_t = cap tanh(s_t / cap) - slope |p - t|,   s_t = sm_scale <q, k_t>,
// over the tokens first <= t < last of its own:
//   last  = its own position and, with a prefix, the whole prefix; or all tokens,
//   first = the larger of its document's first token and p - window + 1.
// Every mask here leaves a row one interval, so a tile of rows is one range of
// tokens [lo, hi) in which what lies before some row's first or behind some row's
// last token is masked element by element.
//
// A tile is computed as in kv4_attend.hip.  The tanh is 1 - 2 / (1 + e^2x): one
// exponential, one reciprocal, and nothing to tell apart for small or large x.
// Scores are in powers of two from there on, so a weight is 2^(z - m).
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

// What is done to a score between the products.
constexpr int kMask = 0;  // nothing
constexpr int kCap = 1;   // the cap
constexpr int kBias = 2;  // the distance, and the cap where cap2 is not 0

struct MArgs {
  Args a;
  const int32_t* starts;
  const int32_t* prefix;
  const float* slopes;
  int window;        // INT_MAX: none
  int ntiles;
  float cap2;        // 2 cap log2(e); 0: none
  float cap_scale;   // 2 |sm_scale| log2(e) / cap
  int4* tiles;       // two per tile: request, row0, nq, col0; end, prefix, lo, hi
  int* weights;      // per tile, 0 where there is none
};

struct MTile : Tile {
  int prefix;  // tokens that every query of the request sees
  int lo, hi;  // tokens that some row of the tile sees lie within
};

struct Bounds {
  int first, last;
};

// Tokens that query i of a request sees.
__device__ inline Bounds bounds(const MArgs& m, const MTile& t, int i) {
  const int p = t.end - t.nq + i;
  Bounds b{0, t.end};
  if (m.a.causal) b.last = max(min(b.last, max(p + 1, t.prefix)), 0);
  if (m.starts != nullptr) b.first = max(b.first, m.starts[t.row0 + i]);
  if (p >= m.window) b.first = max(b.first, p - m.window + 1);
  return b;
}

// The tile's range, by a wave.  Without starts both bounds rise with the row.
template <int COLS>
__device__ inline void find_range(const MArgs& m, MTile& t) {
  const int cols = (int)min((int64_t)t.nq * m.a.G - t.col0, (int64_t)COLS);
  const int i0 = (int)m.a.gdiv.div(t.col0), i1 = (int)m.a.gdiv.div(t.col0 + cols - 1);
  t.prefix = m.prefix != nullptr && t.req < m.a.R ? m.prefix[t.req] : 0;
  t.lo = INT32_MAX;
  t.hi = 0;
  if (m.starts == nullptr) {
    t.lo = bounds(m, t, i0).first;
    t.hi = bounds(m, t, i1).last;
  } else {
    for (int i = i0 + (int)(threadIdx.x & 63); i <= i1; i += 64) {
      const Bounds b = bounds(m, t, i);
      if (b.first >= b.last) continue;
      t.lo = min(t.lo, b.first);
      t.hi = max(t.hi, b.last);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      t.lo = min(t.lo, __shfl_xor(t.lo, off, 64));
      t.hi = max(t.hi, __shfl_xor(t.hi, off, 64));
    }
  }
  if (t.lo >= t.hi) t.lo = t.hi = 0;
  t.lo &= ~15;  // codes are loaded by groups of 16 slots
}

// Weighs the tiles: granules of GR tokens and kItem more for what a tile costs by
// itself, kIdle where it sees nothing.  One wave per tile.
template <int COLS, int GR>
__global__ void __launch_bounds__(256)
kv4_tiles_kernel(const MArgs m) {
  const int tile = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= m.ntiles) return;
  MTile t;
  int w = 0;
  if (find_tile<COLS>(m.a, tile, t)) {
    find_range<COLS>(m, t);
    w = t.hi > t.lo ? kItem + (t.hi - t.lo + GR - 1) / GR : kIdle;
  }
  if ((threadIdx.x & 63) != 0) return;
  m.weights[tile] = w;
  m.tiles[2 * tile] = int4{t.req, t.row0, t.nq, t.col0};
  m.tiles[2 * tile + 1] = int4{t.end, t.prefix, t.lo, t.hi};
}

// The tiles' weights over all heads are cut into equal shares, one per
// workgroup, wherever the cuts fall; an item (a tile under one head) that is cut
// is joined afterwards.
template <int COLS, int THREADS, int GR>
struct MWalk {
  int64_t u = 0, u_end = 0, share = 1;
  int tile = 0, at = 0, hc = 0;  // where the share goes on
  // The item at hand.
  MTile t;
  int head;
  int from, to, more;
  static constexpr int kInts = THREADS + (THREADS / 64 + 3) / 4 * 4;

  __device__ inline MWalk() {}
  __device__ inline MWalk(const MArgs& m, int* s_pre) {
    int* s_wave = s_pre + THREADS;
    const int per = (m.ntiles + THREADS - 1) / THREADS;
    int sum = 0;
    for (int i = 0; i < per; ++i) {
      const int x = threadIdx.x * per + i;
      if (x < m.ntiles) sum += m.weights[x];
    }
    const int incl = wave_incl_scan(sum);
    if ((threadIdx.x & 63) == 63) s_wave[threadIdx.x >> 6] = incl;
    lds_barrier();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      before += w < (int)(threadIdx.x >> 6) ? s_wave[w] : 0;
      total += s_wave[w];
    }
    s_pre[threadIdx.x] = before + incl - sum;
    lds_barrier();
    total = __builtin_amdgcn_readfirstlane(total);
    const int64_t all = (int64_t)total * m.a.heads;
    share = scalar64(max((all + gridDim.x - 1) / gridDim.x, (int64_t)m.a.min_share));
    u = blockIdx.x * share;
    u_end = scalar64(min(u + share, all));
    if (threadIdx.x == 0) m.a.desc[blockIdx.x].x = 0;
    if (u >= u_end) return;
    hc = (int)(u / total);
    int place = (int)(u - (int64_t)hc * total);
    int j = -1;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i)
      j += __builtin_popcountll(__ballot(s_pre[i * 64 + (threadIdx.x & 63)] <= place));
    place -= __builtin_amdgcn_readfirstlane(s_pre[j]);
    tile = j * per;
    for (;; ++tile) {
      const int w = __builtin_amdgcn_readfirstlane(m.weights[tile]);
      if (place < w) break;
      place -= w;
    }
    at = place;
  }
  __device__ inline bool next(const MArgs& m) {
    while (u < u_end) {
      if (tile == m.ntiles) {
        tile = 0;
        ++hc;
      }
      const int n = __builtin_amdgcn_readfirstlane(m.weights[tile]);
      if (n == 0) {
        ++tile;
        continue;
      }
      const int4 x = m.tiles[2 * tile], y = m.tiles[2 * tile + 1];
      t.req = __builtin_amdgcn_readfirstlane(x.x);
      t.row0 = __builtin_amdgcn_readfirstlane(x.y);
      t.nq = __builtin_amdgcn_readfirstlane(x.z);
      t.col0 = __builtin_amdgcn_readfirstlane(x.w);
      t.end = __builtin_amdgcn_readfirstlane(y.x);
      t.prefix = __builtin_amdgcn_readfirstlane(y.y);
      t.lo = __builtin_amdgcn_readfirstlane(y.z);
      t.hi = __builtin_amdgcn_readfirstlane(y.w);
      head = hc;
      const int end = (int)min((int64_t)n, at + (u_end - u));
      u += end - at;
      auto token = [&](int place) {
        return place == n ? t.hi : min(t.lo + max(place - kItem, 0) * GR, t.hi);
      };
      from = token(at);
      to = token(end);
      more = (int)((n - end + share - 1) / share);
      at = end;
      if (end == n) {
        ++tile;
        at = 0;
      }
      // The share may hold none of the item's tokens; of an item without any
      // the last place stands for it.
      if (from < to || (t.lo == t.hi && end == n)) return true;
    }
    return false;
  }
  __device__ inline bool cut() const { return from > t.lo || to < t.hi; }
  // A share cuts the item before it and the one after it at most.
  __device__ inline int64_t slot() const {
    return (int64_t)blockIdx.x * 2 + (from > t.lo ? 0 : 1);
  }
  // For the join, by one thread: a cut item that begins here.
  __device__ inline void announce(const MArgs& m) const {
    if (!cut() || from > t.lo) return;
    const int cols = (int)min((int64_t)COLS, (int64_t)t.nq * m.a.G - t.col0);
    m.a.desc[blockIdx.x] = int4{more + 1, t.row0, t.col0, cols << 16 | head};
  }
  // One item per workgroup, no cuts, without the weights.
  __device__ inline bool whole(const MArgs& m) {
    // Heads first: consecutive workgroups go to the eight XCDs in turn.
    const int i = blockIdx.x / m.a.heads;
    head = blockIdx.x - i * m.a.heads;
    if (!find_tile<COLS>(m.a, i, t)) return false;
    find_range<COLS>(m, t);
    auto scalar = [](int& v) { v = __builtin_amdgcn_readfirstlane(v); };
    scalar(t.req), scalar(t.row0), scalar(t.nq), scalar(t.end), scalar(t.col0);
    scalar(t.prefix), scalar(t.lo), scalar(t.hi);
    from = t.lo;
    to = t.hi;
    more = 0;
    return true;
  }
};

// A wave's columns' bounds, position and slope, per lane.
template <int MODE, int NT>
struct Columns {
  int first[NT], last[NT];
  int pos[MODE == kBias ? NT : 1];
  float slope[MODE == kBias ? NT : 1];  // in powers of two
  // Every token from .. to - 1 is seen by all columns; none outside lo .. hi is
  // seen by any.
  int from, to, lo, hi;
  __device__ inline void clear() {
    from = lo = 0;
    to = INT32_MAX;
    hi = 0;
    lo = INT32_MAX;
  }
  __device__ inline void set(const MArgs& m, const MTile& t, int y, bool ok, int i, int h) {
    const Bounds b = bounds(m, t, i);
    first[y] = ok ? b.first : 0;
    last[y] = ok ? b.last : 0;
    if constexpr (MODE == kBias) {
      pos[y] = t.end - t.nq + i;
      slope[y] = m.slopes[h] * kLog2e;
    }
    if (!ok) return;  // computed along, and dropped
    from = max(from, b.first);
    to = min(to, b.last);
    if (b.first < b.last) {
      lo = min(lo, b.first);
      hi = max(hi, b.last);
    }
  }
  // Over the 16 columns of a row of lanes (the other rows hold the same).
  __device__ inline void reduce() {
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      from = max(from, __shfl_xor(from, off, 64));
      to = min(to, __shfl_xor(to, off, 64));
      lo = min(lo, __shfl_xor(lo, off, 64));
      hi = max(hi, __shfl_xor(hi, off, 64));
    }
    from = __builtin_amdgcn_readfirstlane(from);
    to = __builtin_amdgcn_readfirstlane(to);
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
  }
};

// As State (kv4_tile.hpp), with scores as above.  kMask keeps scores before their
// scale zscale, as there; the others have them in powers of two.
template <int DT, int D, int NT, int MODE>
struct MState : State<DT, D, NT> {
  typedef State<DT, D, NT> S;
  using S::l;
  using S::m;
  using S::o;
  static constexpr int ND = S::ND;
  __device__ inline float base2(int y, float zscale) const {
    if constexpr (DT == FKC_F16) return m[y] - kLead;
    return __builtin_amdgcn_fmed3f(MODE == kMask ? m[y] * zscale : m[y], kLowest, -kLowest);
  }
  // What m may lag behind the largest score (powers of two) before everything is
  // made relative to a new one; fp16: 2^kLead is the largest weight times scale
  // without a lag, so 2^14 with it.
  static constexpr float kLag = DT == FKC_F16 ? 6.f : 8.f, kLead = 8.f;
  // tok: this lane's first token.  zscale: of the mode's first step.
  __device__ inline void weights(f32x4 (&s)[NT][2], const uint2 (&kw)[2], const uint2 (&vw)[2],
                                 bool masked, int base0, int base1, int tok,
                                 const Columns<MODE, NT>& c, float zscale, float cap2,
                                 u32x4 (&pf)[NT]) {
    float ks[2][4], vs[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t kx = i < 2 ? kw[j].x : kw[j].y, vx = i < 2 ? vw[j].x : vw[j].y;
        ks[j][i] = from16<DT>((i & 1) ? kx >> 16 : kx & 0xffffu);
        vs[j][i] = from16<DT>((i & 1) ? vx >> 16 : vx & 0xffffu);
        if constexpr (MODE != kMask) ks[j][i] *= zscale;
      }
    if (masked) {  // what lies past the requests' tokens is anything
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((j ? base1 : base0) < 0 || tok + 16 * j + i >= c.hi) vs[j][i] = 0.f;
          rare(vs[j][i]);
        }
    }
    float ve[2][4];  // fp16: the value scales' exponents; zero counts as 2^-60
    if constexpr (DT == FKC_F16) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ve[j][i] = fmaxf((float)(int)(__float_as_uint(fabsf(vs[j][i])) >> 23) - 126.f, -60.f);
    }
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      float z[2][4], top = kLowest;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[j][i] = s[y][j][i] * ks[j][i];
      if (MODE == kCap || (MODE == kBias && cap2 != 0.f)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            z[j][i] = __builtin_fmaf(
                -cap2, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z[j][i])), 0.5f * cap2);
      }
      if constexpr (MODE == kBias) {
        const float away = (float)(c.pos[y] - tok);  // rounded past 2^24 only
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            z[j][i] = __builtin_fmaf(-c.slope[y], fabsf(away - (float)(16 * j + i)), z[j][i]);
      }
      if (masked) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int x = tok + 16 * j + i;
            if ((j ? base1 : base0) < 0 || x < c.first[y] || x >= c.last[y])
              z[j][i] = -INFINITY;
            rare(z[j][i]);
          }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = DT != FKC_F16   ? z[j][i]
                          : MODE == kMask ? __builtin_fmaf(z[j][i], zscale, ve[j][i])
                                          : z[j][i] + ve[j][i];
          top = fmaxf(top, v);
        }
      if (__any(DT == FKC_F16 || MODE != kMask ? top > m[y] + kLag : (top - m[y]) * zscale > kLag)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float nm = fmaxf(m[y], top);
        const float f = __builtin_amdgcn_exp2f(
            DT == FKC_F16 || MODE != kMask ? m[y] - nm : (m[y] - nm) * zscale);
        m[y] = nm;
        l[y] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[y][d] *= f;
      }
      const float mz = base2(y, zscale);
      float w[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __builtin_amdgcn_exp2f(
              MODE == kMask ? __builtin_fmaf(z[j][i], zscale, -mz) : z[j][i] - mz);
          l[y] += p;
          w[j][i] = p * vs[j][i];
        }
      if (masked) {  // a scale that is not finite counts where it is seen
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[j][i] = z[j][i] == -INFINITY ? 0.f : w[j][i];
            rare(w[j][i]);
          }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        pf[y][e] = pack2<DT>(w[e >> 1][2 * (e & 1)], w[e >> 1][2 * (e & 1) + 1]);
    }
  }
};

__device__ inline const MArgs& arguments() { return arguments_as<MArgs>(); }

template <int DT, int D, int NT, int WAVES, int MODE>
__global__ void __launch_bounds__(WAVES * 64, WAVES / 2)
kv4_masked_split_kernel(const MArgs margs) {
  constexpr int COLS = 16 * NT, THREADS = WAVES * 64, UNIT = WAVES * 32;
  constexpr int KS = D / 32;  // steps of the first product
  constexpr int ND = D / 16;  // feature tiles of the second
  const Args& args = margs.a;
  extern __shared__ __align__(16) char lds[];
  float2* sml = reinterpret_cast<float2*>(lds + kTable);
  int* s_pre = reinterpret_cast<int*>(lds + kTable + kJoin);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  typedef MWalk<COLS, THREADS, UNIT> W;
  W k = args.whole ? W() : W(arguments(), s_pre);
  if (!(args.whole ? k.whole(arguments()) : k.next(arguments()))) return;
  for (;;) {
    // Opaque, so that what derives from it is computed per item, not kept in
    // registers over the whole share.
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const MArgs& ma = arguments();
    const Args& a = ma.a;
    const int lane = tid & 63, n = lane & 15, g = lane >> 4;
    const uint32_t loff = (uint32_t)(lane & 31) * 4;
    const MTile& t = k.t;
    const int ncols = t.nq * a.G;
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
        base[j] = b < a.num_blocks ? (int)((b * (uint32_t)a.heads + k.head) * (a.bs.d / 16) + in)
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
      head = k.head * a.G + (min(col, ncols - 1) - i * a.G);
    };
    Columns<MODE, NT> cols;
    cols.clear();
    u32x4 qf[NT][KS];
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      int row, head, i;
      column(a, 16 * y + n, row, head, i);
      const bool ok = row >= 0;
      cols.set(ma, t, y, ok, i, head);
      const uint16_t* qp = a.q + max(row, t.row0) * a.q_ts + head * a.q_hs + g * (D / 4);
#pragma unroll
      for (int s = 0; s < KS; ++s)
        qf[y][s] = (ok ? *reinterpret_cast<const u32x4*>(qp + s * 8) : u32x4{0, 0, 0, 0}) ^
                   a.qsign;
    }
    cols.reduce();
    const float zscale = MODE == kCap || (MODE == kBias && ma.cap2 != 0.f) ? ma.cap_scale
                                                                         : a.zscale;
    const float cap2 = ma.cap2;
    const Lane<D> lanes(n, g);
    Codes<D> cur;
    groups(wave, blk, base);
    if (wave < ntile) {
      load_keys<D>(a, base, lanes, cur);
      load_scales<D>(a, base, lanes, cur);
      load_values<D>(a, base, lanes, cur);
    }
    load_blocks(wave + WAVES, blk);
    fill_table<THREADS>(a, k.head, lds, tid);
    lds_barrier();

    MState<DT, D, NT, MODE> st;
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
      const int tok = t0 + it * 32;
      st.weights(s, kw, vw, tok + 32 > cols.to || tok < cols.from || (base[0] | base[1]) < 0,
                 base[0], base[1], tok + 4 * g, cols, zscale, cap2, pf);
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
      const float rel = st.base2(y, zscale);
      if (g == 0) sml[wave * 16 + n] = float2{rel, st.l[y]};
      lds_barrier();
      const Args& a = arguments().a;
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

template <int DT, int D, int NT, int TT, int MODE>
__global__ void __launch_bounds__(512, 2)
kv4_masked_wide_kernel(const MArgs margs) {
  constexpr int WAVES = 8, COLS = 16 * NT * WAVES, THREADS = WAVES * 64;
  constexpr int KS = D / 32, ND = D / 16, HALVES = TT / 16, GROUPS = TT / 32;
  constexpr int KPW = HALVES * KS / WAVES;  // key fragments a wave fills
  constexpr int VW = GROUPS * ND / 2;       // waves that fill two value fragments
  static_assert(KPW >= 1 && KS % KPW == 0 && VW <= WAVES, "a wave fills within one half");
  constexpr int KBYTES = TT * D * 2, BUF = 2 * KBYTES;
  typedef int Groups __attribute__((ext_vector_type(HALVES)));
  const Args& args = margs.a;
  extern __shared__ __align__(16) char lds[];
  int* s_pre = reinterpret_cast<int*>(lds + kTable + 2 * BUF);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kj = wave * KPW / KS, kc0 = wave * KPW % KS;  // its half, first step
  const int vg = wave % VW / (ND / 2), vu = wave % (ND / 2);  // its group, fragment pair
  int table = -1;  // head whose table is in LDS
  typedef MWalk<COLS, THREADS, TT> W;
  W k = args.whole ? W() : W(arguments(), s_pre);
  if (!(args.whole ? k.whole(arguments()) : k.next(arguments()))) return;
  for (;;) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const MArgs& ma = arguments();
    const Args& a = ma.a;
    const int lane = tid & 63, n = lane & 15, g = lane >> 4;
    const uint32_t loff = (uint32_t)(lane & 31) * 4;
    const MTile& t = k.t;
    const int ncols = t.nq * a.G;
    const int col0 = t.col0 + wave * 16 * NT;  // the wave's columns, in the request
    const int t0 = k.from, t1 = k.to, tiles = (max(t1 - t0, 0) + TT - 1) / TT;

    // The arguments that every tile needs, in scalar registers (left to itself
    // the compiler reads them again at each use, and waits).
    // (Global addresses by type: behind the asm nothing else says so, and a
    // load that might be LDS's would be waited for with every LDS read.)
    Global k_codes = (Global)a.k_codes, v_codes = (Global)a.v_codes;
    Global k_scales = (Global)a.k_scales, v_scales = (Global)a.v_scales;
    uint32_t bs = a.bs.d, bs_m = a.bs.m, num_blocks = a.num_blocks;
    int bs_sh = a.bs.sh, heads = a.heads;
    float zscale = MODE == kCap || (MODE == kBias && ma.cap2 != 0.f) ? ma.cap_scale : a.zscale;
    float cap2 = ma.cap2;
    asm volatile("" : "+s"(k_codes), "+s"(v_codes), "+s"(k_scales), "+s"(v_scales));
    asm volatile("" : "+s"(bs), "+s"(bs_m), "+s"(num_blocks), "+s"(bs_sh), "+s"(heads),
                 "+s"(zscale), "+s"(cap2));
    const Const32 blocks = (Const32)(a.tables + (int64_t)t.req * a.table_stride);
    // 16-slot groups of a tile's halves over all heads, -1 where there is none.
    auto find_groups = [&](int tile, Groups& base) {
#pragma unroll
      for (int j = 0; j < HALVES; ++j) {
        const uint32_t tok = t0 + tile * TT + 16 * j;
        const uint32_t at = __umulhi(tok, bs_m) >> bs_sh;  // (block sizes are 16 at least)
        const uint32_t b = (int)tok < t1 ? (uint32_t)blocks[at] : 0xffffffffu;
        base[j] = b < num_blocks ? (int)((b * heads + k.head) * (bs / 16) + (tok - at * bs) / 16)
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
      head = k.head * a.G + (min(col, ncols - 1) - i * a.G);
    };

    Groups base, nbase;  // of this tile and the next
    find_groups(0, base);
    find_groups(1, nbase);
    if (tiles > 0) {
      load_tile(base);
#pragma unroll
      for (int j = 0; j < HALVES; ++j) load_scales(base, j);
    }
    Columns<MODE, NT> cols;
    cols.clear();
    u32x4 qf[NT][KS];
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      int row, head, i;
      column(a, y, row, head, i);
      const bool ok = row >= 0;
      cols.set(ma, t, y, ok, i, head);
      const uint16_t* qp = a.q + max(row, t.row0) * a.q_ts + head * a.q_hs + g * (D / 4);
#pragma unroll
      for (int c = 0; c < KS; ++c)
        qf[y][c] = (ok ? *reinterpret_cast<const u32x4*>(qp + c * 8) : u32x4{0, 0, 0, 0}) ^
                   a.qsign;
    }
    cols.reduce();
    if (table != k.head) {  // (every look-up of the last item was before its last barrier)
      table = k.head;
      fill_table<THREADS>(a, k.head, lds, tid);
      lds_barrier();
    }
    if (tiles > 0) fill_buffer(0);
    if (tiles > 0) load_tile(nbase);
    lds_barrier();

    MState<DT, D, NT, MODE> st;
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
        if (tok >= cols.hi || tok + 32 <= cols.lo) return;  // none of the wave's columns sees them
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
        st.weights(s, kw, vw,
                   tok + 32 > cols.to || tok < cols.from || (base[2 * h] | base[2 * h + 1]) < 0,
                   base[2 * h], base[2 * h + 1], tok + 4 * g, cols, zscale, cap2, pf);
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
      const Args& a = arguments().a;
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
          if (g == 0 && a.lse != nullptr) a.lse[at] = log_sum(st.base2(y, zscale), st.l[y]);
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
                float2{st.base2(y, zscale), st.l[y]};
        }
      }
    }
    if (args.whole) return;
    if (tid == 0) k.announce(arguments());
    if (!k.next(arguments())) return;
  }
}

// As for kv4_attend.hip; a window bounds what a tile of a causal call sees.
constexpr int kMinShare = 2, kWhole = 8, kWideWhole = 32;

struct Plan {
  bool wide;
  int nt;             // column tiles per wave
  int waves;
  bool whole;         // one item per workgroup
  int64_t wgs, ntiles;
  int tiles_per_req;  // without cu_q
  int cols() const { return 16 * nt * (wide ? waves : 1); }
  size_t part_rows() const { return (size_t)wgs * 2 * cols(); }
};

constexpr int kWide = 8;  // waves of the wide form
constexpr int wide_tiles(int D) { return D == 256 ? 1 : 2; }
constexpr int wide_tokens(int D) { return D == 256 ? 32 : 64; }
constexpr int waves_of(int D) { return D == 256 ? 4 : 8; }

// reach: tokens that one query sees at most (max_seq, or the window).
Plan make_plan(const fkc_kv4_cache& c, int64_t H, int64_t T, int64_t R, int64_t max_seq,
               int64_t reach, bool ragged) {
  Plan p;
  const int64_t G = H / c.heads;
  const int64_t avg = R > 0 ? T * G / R : 0;
  p.wide = avg > (c.D == 256 ? 224 : 448);
  p.nt = p.wide ? wide_tiles((int)c.D) : c.D < 256 && avg > 64 ? 2 : 1;
  p.waves = p.wide ? kWide : p.nt == 2 ? 4 : waves_of((int)c.D);
  const int64_t cols = p.cols();
  p.tiles_per_req = (int)((G + cols - 1) / cols);
  p.ntiles = ragged ? T * G / cols + R + 1 : R * p.tiles_per_req;
  const int64_t len = std::min(max_seq, reach + (cols + G - 1) / G + 16);
  p.whole = len <= (p.wide ? kWideWhole * 32 : kWhole * 32 * p.waves);
  p.wgs = p.whole ? p.ntiles * c.heads : (p.wide ? 1 : 2) * (int64_t)device_shape().cus;
  return p;
}

template <int DT, int D, int COLS, int GR, int THREADS, typename K>
int launch(K kernel, std::atomic<uint64_t>& set, int bytes, const MArgs& m, const Plan& p,
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
  if (!p.whole)
    hipLaunchKernelGGL((kv4_tiles_kernel<COLS, GR>), dim3((uint32_t)((p.ntiles + 3) / 4)),
                       dim3(256), 0, s, m);
  hipLaunchKernelGGL(kernel, dim3((uint32_t)p.wgs), dim3(THREADS), bytes, s, m);
  if (int rc = check_launch("kv4_attend")) return rc;
  if (p.whole) return FKC_OK;
  const int64_t cols = std::min<int64_t>(COLS, m.a.cu_q ? COLS : m.a.G);
  hipLaunchKernelGGL((kv4_join_kernel<DT, D, COLS>),
                     dim3((uint32_t)p.wgs, (uint32_t)std::min<int64_t>((cols + 3) / 4, 16)),
                     dim3(256), 0, s, m.a);
  return check_launch("kv4_attend (join)");
}

template <int DT, int D, int NT, int WAVES, int MODE>
int launch_split(const MArgs& m, const Plan& p, hipStream_t s) {
  static std::atomic<uint64_t> set{0};
  return launch<DT, D, 16 * NT, WAVES * 32, WAVES * 64>(
      &kv4_masked_split_kernel<DT, D, NT, WAVES, MODE>, set,
      kTable + kJoin + MWalk<16 * NT, WAVES * 64, 1>::kInts * 4, m, p, s);
}

template <int DT, int D, int MODE>
int launch_wide(const MArgs& m, const Plan& p, hipStream_t s) {
  static std::atomic<uint64_t> set{0};
  constexpr int NT = wide_tiles(D), TT = wide_tokens(D), COLS = 16 * NT * kWide;
  return launch<DT, D, COLS, TT, kWide * 64>(
      &kv4_masked_wide_kernel<DT, D, NT, TT, MODE>, set,
      kTable + 2 * (TT * D * 4) + MWalk<COLS, kWide * 64, 1>::kInts * 4, m, p, s);
}

template <int DT, int D, int MODE>
int launch_mode(const MArgs& m, const Plan& p, hipStream_t s) {
  if (p.wide) return launch_wide<DT, D, MODE>(m, p, s);
  if constexpr (D < 256)
    if (p.nt == 2) return launch_split<DT, D, 2, 4, MODE>(m, p, s);
  return launch_split<DT, D, 1, waves_of(D), MODE>(m, p, s);
}

// Tokens that a query sees at most.
int64_t reach_of(int64_t max_seq, const Kv4Scores& x, bool causal) {
  return causal && !x.prefix && x.window > 0 ? std::min(max_seq, x.window) : max_seq;
}

struct Scratch {
  float *part, *part_ml;
  int4 *desc, *tiles;
  int* weights;
  size_t bytes;
  Scratch(void* ws, const fkc_kv4_cache& c, const Plan& p) {
    Carve w(ws);
    part = w.take<float>(p.part_rows() * c.D);
    part_ml = w.take<float>(p.part_rows() * 2);
    desc = w.take<int4>((size_t)p.wgs);
    tiles = w.take<int4>((size_t)p.ntiles * 2);
    weights = w.take<int>((size_t)p.ntiles);
    bytes = w.used;
  }
};

}  // namespace

size_t kv4_attend_scored_workspace_bytes(const fkc_kv4_cache& c, int64_t H, int64_t T, int64_t R,
                                         int64_t max_seq, bool causal, const Kv4Scores& x) {
  const Plan p = make_plan(c, H, T, R, max_seq, reach_of(max_seq, x, causal), true);
  return p.whole ? 0 : Scratch(nullptr, c, p).bytes;
}

int launch_kv4_attend_scored(const fkc_kv4_cache& c, const Kv4Attend& x, const Kv4Scores& sc,
                             void* ws, hipStream_t s) {
  const Plan p = make_plan(c, x.H, x.T, x.R, x.max_seq, reach_of(x.max_seq, sc, x.causal),
                           x.cu_q != nullptr);
  const int G = (int)(x.H / c.heads);
  // Weights of a head's items are summed in 32 bits.
  const int64_t gr = p.wide ? wide_tokens((int)c.D) : 32 * p.waves;
  if (p.wgs > INT32_MAX || p.ntiles > INT32_MAX / (x.max_seq / gr + 2 + kItem))
    return fail(FKC_ERR_UNSUPPORTED, "kv4_attend: too many rows times tokens");
  // (of scores times 0 the masked ones would be NaN)
  const double scale = std::max(std::fabs((double)x.sm_scale) * 1.4426950408889634, 1e-30);
  Args a{(const uint16_t*)x.q.p, x.q.token_stride, x.q.head_stride,
         (const uint8_t*)c.k_codes, (const uint8_t*)c.v_codes,
             (const uint16_t*)c.k_scales, (const uint16_t*)c.v_scales,
             (const uint16_t*)c.k_levels, (const uint16_t*)c.v_levels,
             x.tables, x.table_stride, x.seq, x.cu_q, (uint16_t*)x.out, x.lse, nullptr, nullptr,
             nullptr, FastDiv((uint32_t)c.block_size), FastDiv((uint32_t)G),
             (uint32_t)c.num_blocks, (int)c.heads, (int)x.H, G, (int)x.T, (int)x.R,
             (int)x.max_seq, (int)x.causal, (int)p.whole, kMinShare, p.tiles_per_req,
             (float)scale, std::signbit(x.sm_scale) ? 0x80008000u : 0u};
  MArgs m{a, sc.starts, sc.prefix, sc.slopes, sc.window > 0 ? (int)sc.window : INT32_MAX,
          (int)p.ntiles, 0.f, 0.f, nullptr, nullptr};
  if (sc.softcap > 0.f) {
    m.cap2 = (float)(2 * 1.4426950408889634 * sc.softcap);
    m.cap_scale = (float)std::min(2 * scale / sc.softcap, 3e38);
  }
  if (!p.whole) {
    const Scratch w(ws, c, p);
    m.a.part = w.part;
    m.a.part_ml = w.part_ml;
    m.a.desc = w.desc;
    m.tiles = w.tiles;
    m.weights = w.weights;
  }
  return kv4_by_shape(c.dtype, c.D, [&](auto dt, auto d) {
    constexpr int DT = dt.value, DD = d.value;
    if (sc.slopes != nullptr) return launch_mode<DT, DD, kBias>(m, p, s);
    if (sc.softcap > 0.f) return launch_mode<DT, DD, kCap>(m, p, s);
    return launch_mode<DT, DD, kMask>(m, p, s);
  });
}

}  // namespace fkc
