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
// A tile's products are those of kv4_attend.hip.  The tanh is 1 - 2 / (1 + e^2x):
// one exponential, one reciprocal, and nothing to tell apart for small or large x.
// It is off by units in the last place of 1, not of itself: with one unit (2^-23)
// each of exponential and reciprocal and the sum rounded by half of one, by
// 1.5 * 2^-22 at most, so a score by 2^-21 of the cap, however small the score
// (measured: 2^-21.5; a cap of 50: 2.4e-5, where rounding a weight near 1 to fp16
// is 4.9e-4; large caps: sharp_tanh).  Scores are in powers of two from there on,
// so a weight is 2^(z - m).
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
constexpr int kBias = 2;  // the distance; in the wide form the cap too, if there is one
constexpr int kBoth = 3;  // the cap, by sharp_tanh, and the distance
constexpr bool capped(int mode) { return mode == kCap || mode == kBoth; }
constexpr bool biased(int mode) { return mode >= kBias; }

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

// The range of a single token's tile, by one lane.
template <int COLS>
__device__ inline bool find_single(const MArgs& m, int tile, MTile& t) {
  if (!find_tile<COLS>(m.a, tile, t)) return false;
  t.prefix = m.prefix != nullptr ? m.prefix[t.req] : 0;
  const Bounds b = bounds(m, t, 0);
  t.lo = b.first < b.last ? b.first & ~15 : 0;
  t.hi = b.first < b.last ? b.last : 0;
  return true;
}

template <int GR, int ITEM>
__device__ inline int weight_of(const MTile& t) {
  return t.hi > t.lo ? ITEM + (t.hi - t.lo + GR - 1) / GR : kIdle;
}

// Weighs the tiles: granules of GR tokens and ITEM more for what a tile costs by
// itself, kIdle where it sees nothing.  One wave per tile.  (Single tokens' tiles
// are weighed by the workgroups that share them: one load or two each.)
template <int COLS, int GR, int ITEM>
__global__ void __launch_bounds__(256)
kv4_tiles_kernel(const MArgs m) {
  const int tile = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= m.ntiles) return;
  MTile t;
  int w = 0;
  if (find_tile<COLS>(m.a, tile, t)) {
    find_range<COLS>(m, t);
    w = weight_of<GR, ITEM>(t);
  }
  if ((threadIdx.x & 63) != 0) return;
  m.weights[tile] = w;
  m.tiles[2 * tile] = int4{t.req, t.row0, t.nq, t.col0};
  m.tiles[2 * tile + 1] = int4{t.end, t.prefix, t.lo, t.hi};
}

// The tiles' weights over all heads are cut into equal shares, one per
// workgroup, wherever the cuts fall; an item (a tile under one head) that is cut
// is joined afterwards.  (Weights of a sum in closed form, as kv4_attend.hip has
// them, do not know where documents begin; every workgroup adds up all of them
// instead, about 1 us.)
template <int COLS, int THREADS, int GR, int ITEM>
struct MWalk {
  int64_t u = 0, u_end = 0, share = 1;
  int tile = 0, at = 0, hc = 0;  // where the share goes on
  // The item at hand.
  MTile t;
  int head;
  int from, to, more;
  static constexpr int kInts = THREADS + (THREADS / 64 + 3) / 4 * 4;

  __device__ inline MWalk() {}
  __device__ inline int weigh(const MArgs& m, int i) const {
    if (m.a.cu_q != nullptr) return m.weights[i];
    MTile x;
    return find_single<COLS>(m, i, x) ? weight_of<GR, ITEM>(x) : 0;
  }
  __device__ inline MWalk(const MArgs& m, int* s_pre) {
    int* s_wave = s_pre + THREADS;
    const int per = (m.ntiles + THREADS - 1) / THREADS;
    int sum = 0;
    for (int i = 0; i < per; ++i) {
      const int x = threadIdx.x * per + i;
      if (x < m.ntiles) sum += weigh(m, x);
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
      const int w = __builtin_amdgcn_readfirstlane(weigh(m, tile));
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
      int n;
      if (m.a.cu_q == nullptr) {
        n = find_single<COLS>(m, tile, t) ? weight_of<GR, ITEM>(t) : 0;
      } else {
        n = m.weights[tile];
        const int4 x = m.tiles[2 * tile], y = m.tiles[2 * tile + 1];
        t.req = x.x, t.row0 = x.y, t.nq = x.z, t.col0 = x.w;
        t.end = y.x, t.prefix = y.y, t.lo = y.z, t.hi = y.w;
      }
      auto scalar = [](int& v) { v = __builtin_amdgcn_readfirstlane(v); };
      scalar(n);
      if (n == 0) {
        ++tile;
        continue;
      }
      scalar(t.req), scalar(t.row0), scalar(t.nq), scalar(t.end), scalar(t.col0);
      scalar(t.prefix), scalar(t.lo), scalar(t.hi);
      head = hc;
      const int end = (int)min((int64_t)n, at + (u_end - u));
      u += end - at;
      auto token = [&](int place) {
        return place == n ? t.hi : min(t.lo + max(place - ITEM, 0) * GR, t.hi);
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
  int pos[biased(MODE) ? NT : 1];
  float slope[biased(MODE) ? NT : 1];  // in powers of two
  // Every token from .. to - 1 is seen by all columns; none outside lo .. hi is
  // seen by any.
  int from, to, lo, hi;
  __device__ inline void clear() {
    from = hi = 0;
    to = lo = INT32_MAX;
  }
  __device__ inline void set(const MArgs& m, const MTile& t, int y, bool ok, int i, int h) {
    const Bounds b = bounds(m, t, i);
    first[y] = ok ? b.first : 0;
    last[y] = ok ? b.last : 0;
    if constexpr (biased(MODE)) {
      pos[y] = t.end - t.nq + i;
      slope[y] = m.slopes != nullptr ? m.slopes[h] * kLog2e : 0.f;
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

// fp16: what a value scale adds to the maximum, its logarithm; zero counts as 2^-60,
// infinity as 2^129.
__device__ inline float exponent_of(float scale) {
  return __builtin_amdgcn_fmed3f(__builtin_amdgcn_logf(fabsf(scale)), -60.f, 129.f);
}

// tanh x of e = 2 log2(e) x within 2^-18 of itself: for |x| < 0.35 the series, whose
// first term left out is 2^-22 of it, and 1 - 2 / (1 + 2^e), off by 2^-21 of 1,
// beyond.
__device__ inline float sharp_tanh(float e) {
  const float r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(e));
  const float x = e * 0.34657359f, xx = x * x;
  float p = __builtin_fmaf(xx, 62.f / 2835, -17.f / 315);
  p = __builtin_fmaf(p, xx, 2.f / 15);
  p = __builtin_fmaf(p, xx, -1.f / 3);
  p = __builtin_fmaf(p * xx, x, x);
  return fabsf(e) < 1.f ? p : __builtin_fmaf(-2.f, r, 1.f);
}

// As State (kv4_tile.hpp), with scores as above, in the steps that a kernel may
// put between its products.  What stands for a score z in powers of two:
//   kMask  z / zscale,
//   kCap   r = 1 / (1 + e^2x), with z = cap2 / 2 - cap2 r (hidden: r = infinity),
//   kBias, kBoth  z - shift, one shift per column and tile,
// so that the last multiplication is the one that the weight's exponent needs
// anyway.
template <int DT, int D, int NT, int MODE, bool WIDE>
struct MState : State<DT, D, NT> {
  typedef State<DT, D, NT> S;
  using S::l;
  using S::m;
  using S::o;
  static constexpr int ND = S::ND;
  // m is the largest score so far, so the largest weight is 1 and its product with
  // its scale is exact (fp16: the largest product is 2^kLead).  A maximum left
  // behind by up to 2^8 (fp16 2^6) spares most of the scaling, capped prompts 658 us
  // instead of 690, documents 181 instead of 188, and rounds the largest product
  // too: capped prompts 2.05e-3 off the plain form instead of 0.99e-3, documents
  // 2.5e-4 instead of 1.6e-4.
  static constexpr float kLead = 14.f;
  static constexpr float kHidden = MODE == kCap ? INFINITY : -INFINITY;
  // Of the tile at hand: the keys' scales, times the first step's factor but for
  // kMask, the values', and (fp16) exponent_of these.
  f32x4 ks[2], vs[2], ve[DT == FKC_F16 ? 2 : 1];
  float shift[biased(MODE) ? NT : 1];
  __device__ inline float base2(int y, float zscale) const {
    if constexpr (DT == FKC_F16) return m[y] - kLead;
    return __builtin_amdgcn_fmed3f(MODE == kMask ? m[y] * zscale : m[y], kLowest, -kLowest);
  }
  __device__ inline void scales(const uint2 (&kw)[2], const uint2 (&vw)[2], float zscale) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t kx = i < 2 ? kw[j].x : kw[j].y, vx = i < 2 ? vw[j].x : vw[j].y;
        ks[j][i] = from16<DT>((i & 1) ? kx >> 16 : kx & 0xffffu);
        vs[j][i] = from16<DT>((i & 1) ? vx >> 16 : vx & 0xffffu);
        if constexpr (MODE != kMask) ks[j][i] *= zscale;
        if constexpr (DT == FKC_F16) ve[j][i] = exponent_of(vs[j][i]);
      }
  }
  // Products to scores, in place.  tok: this lane's first token, first: the tile's.
  __device__ inline void score(f32x4 (&z)[NT][2], int tok, int first,
                               const Columns<MODE, NT>& c, float cap2) {
#pragma unroll
    for (int y = 0; y < NT; ++y) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[y][j][i] *= ks[j][i];
      // (WIDE: the wide form, where asking as it runs is the faster way: prefixes under
      // slopes 702 us, without the question 737, registers being given out otherwise.
      // Drafts 93.4, with it 94.9.)
      if (capped(MODE) || (WIDE && MODE == kBias && cap2 != 0.f)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = z[y][j][i];
            z[y][j][i] = MODE == kCap
                             ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(e))
                             : 0.5f * cap2 * sharp_tanh(e);
          }
      }
      if constexpr (biased(MODE)) {
        // Before all of the tile or behind it a column's distances rise or fall by
        // one from token to token.
        const int away = c.pos[y] - tok;  // (exact in fp32 below 2^24)
        if (!__any(c.pos[y] > first && c.pos[y] < first + 31)) {
          const float per = c.pos[y] > first ? c.slope[y] : -c.slope[y];
          shift[y] = -per * (float)away;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              z[y][j][i] = __builtin_fmaf(per, (float)(16 * j + i), z[y][j][i]);
        } else {
          shift[y] = 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              z[y][j][i] =
                  __builtin_fmaf(-c.slope[y], fabsf((float)(away - 16 * j - i)), z[y][j][i]);
        }
      }
    }
  }
  // For tiles that some column does not see all of; there: a bit for each half that
  // has a block.
  __device__ inline void mask(f32x4 (&z)[NT][2], int there, int tok,
                              const Columns<MODE, NT>& c) {
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      // (one comparison for both ends: what is before the first wraps)
      const uint32_t at = (uint32_t)(tok - c.first[y]);
      const uint32_t len = (uint32_t)max(c.last[y] - c.first[y], 0);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = z[y][j][i];
          if (at + (16 * j + i) >= len) v = kHidden;
          rare(v);
          z[y][j][i] = v;
        }
    }
    if (there != 3) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (!(there >> j & 1))
#pragma unroll
          for (int y = 0; y < NT; ++y) z[y][j] = f32x4{kHidden, kHidden, kHidden, kHidden};
    }
  }
  // And their values' scales: 0 for what no column sees, which may be anything.
  // Returns whether one is not finite all the same, so that its product with a
  // hidden column's weight, 0, would not be 0.
  __device__ inline bool mask_values(int there, int tok, const Columns<MODE, NT>& c) {
    bool odd = false;
    const uint32_t at = (uint32_t)(tok - c.lo), len = (uint32_t)max(c.hi - c.lo, 0);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float s = vs[j][i];
        if (at + (16 * j + i) >= len || !(there >> j & 1)) s = 0.f;
        rare(s);
        vs[j][i] = s;
        odd |= !(fabsf(s) < INFINITY);
      }
    return __any(odd);
  }
  // The maxima, and what follows from new ones.
  __device__ inline void settle(const f32x4 (&z)[NT][2], float zscale, float cap2) {
    float top[NT];
    bool more = false;
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      float t = DT != FKC_F16 && MODE == kCap ? INFINITY : -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = z[y][j][i];
          if constexpr (DT != FKC_F16)
            t = MODE == kCap ? fminf(t, v) : fmaxf(t, v);
          else
            t = fmaxf(t, MODE == kMask  ? __builtin_fmaf(v, zscale, ve[j][i])
                         : MODE == kCap ? __builtin_fmaf(-cap2, v, ve[j][i])
                                        : v + ve[j][i]);
        }
      if constexpr (MODE == kCap)
        t = DT != FKC_F16 ? __builtin_fmaf(-cap2, t, 0.5f * cap2) : t + 0.5f * cap2;
      if constexpr (biased(MODE)) t += shift[y];
      top[y] = t;
      more |= t > m[y];
    }
    if (__any(more)) {
#pragma unroll
      for (int y = 0; y < NT; ++y) {
        float t = fmaxf(top[y], __shfl_xor(top[y], 16, 64));
        t = fmaxf(t, __shfl_xor(t, 32, 64));
        const float nm = fmaxf(m[y], t);
        const float f = __builtin_amdgcn_exp2f(
            DT == FKC_F16 || MODE != kMask ? m[y] - nm : (m[y] - nm) * zscale);
        m[y] = nm;
        l[y] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[y][d] *= f;
      }
    }
  }
  // What the exponent of a weight is: one operation from what stands for z.
  __device__ inline float exponent(float v, float base, float zscale, float cap2) const {
    return MODE == kMask  ? __builtin_fmaf(v, zscale, base)
           : MODE == kCap ? __builtin_fmaf(-cap2, v, base)
                          : v + base;
  }
  __device__ inline float base_of(int y, float zscale, float cap2) const {
    const float b = -base2(y, zscale);
    return MODE == kCap ? 0.5f * cap2 + b : biased(MODE) ? shift[y] + b : b;
  }
  // Scores to weights, packed as the second product reads them.
  __device__ inline void weigh(const f32x4 (&z)[NT][2], float zscale, float cap2,
                               u32x4 (&pf)[NT]) {
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      const float base = base_of(y, zscale, cap2);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __builtin_amdgcn_exp2f(exponent(z[y][j][i], base, zscale, cap2));
          l[y] += p;
          w[i] = p * vs[j][i];
        }
        pf[y][2 * j] = pack2<DT>(w[0], w[1]);
        pf[y][2 * j + 1] = pack2<DT>(w[2], w[3]);
      }
    }
  }
  // After mask's true: the weights once more, 0 for what is hidden.
  __device__ inline void weigh_odd(const f32x4 (&z)[NT][2], float zscale, float cap2,
                                   u32x4 (&pf)[NT]) {
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      const float base = base_of(y, zscale, cap2);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = z[y][j][i];
          w[i] = __builtin_amdgcn_exp2f(exponent(v, base, zscale, cap2)) * vs[j][i];
          w[i] = v == kHidden ? 0.f : w[i];
          rare(w[i]);
        }
        pf[y][2 * j] = pack2<DT>(w[0], w[1]);
        pf[y][2 * j + 1] = pack2<DT>(w[2], w[3]);
      }
    }
  }
};

__device__ inline const MArgs& arguments() { return arguments_as<MArgs>(); }

// The split form, for few columns, as in kv4_attend.hip: the waves of a workgroup
// share NT tiles of 16 columns and take 32 tokens each in turn, are joined in LDS at
// the end of an item, and cut items by a second kernel.
//
// Bound by memory where contexts are long: one query of each of 64 ragged requests
// that look back over 4096 tokens, 435 MB of bf16 cache (D = 256, 8 heads of 2
// capped), takes 97 us (89 at least), 4.5 TB/s, where a large copy moves 4.6 and
// reading alone 6.4.  Drafts of 2 to 7 tokens under slopes (fp16, D = 128, 4 heads of 8,
// contexts of 300 to 65536, 175 MB) take 77 us: tiles of 16 columns look the same codes up 2.75
// times, 128 look-ups a tile of 32 tokens, beside ~230 vector and 16 matrix
// operations.  (Two tiles a wave look up half as often with half the waves: the
// same.)
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
  typedef MWalk<COLS, THREADS, UNIT, kItem> W;
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
    // What is loaded where there is no block, or no tile any more: what the wave
    // loaded last, not slot 0, the same for every workgroup.
    int from[2] = {0, 0};
    auto loads = [&](const int (&b)[2]) {
#pragma unroll
      for (int j = 0; j < 2; ++j) from[j] = b[j] >= 0 ? b[j] : from[j];
    };
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
    const float zscale = capped(MODE) ? ma.cap_scale : a.zscale;
    const float cap2 = ma.cap2;
    const Lane<D> lanes(n, g);
    Codes<D> cur;
    groups(wave, blk, base);
    loads(base);
    if (wave < ntile) {
      load_keys<D>(a, from, lanes, cur);
      load_scales<D>(a, from, lanes, cur);
      load_values<D>(a, from, lanes, cur);
    }
    load_blocks(wave + WAVES, blk);
    fill_table<THREADS>(a, k.head, lds, tid);
    lds_barrier();

    MState<DT, D, NT, MODE, false> st;
    st.clear();
    // What a tile has used up is fetched for the next one at once, after the last
    // tile its own again (a load that may or may not be on its way would have to
    // be waited for with every older one), into the same registers: with a second
    // set of them four waves a SIMD do not fit, and it is they that hide the loads'
    // latency.
    for (int it = wave; it < ntile; it += WAVES) {
      groups(it + WAVES, blk, nbase);
      loads(nbase);
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
      load_keys<D>(a, from, lanes, cur);
      const uint2 kw[2] = {cur.ks[0], cur.ks[1]}, vw[2] = {cur.vs[0], cur.vs[1]};
      load_scales<D>(a, from, lanes, cur);
      u32x4 pf[NT];
      const int tok = t0 + it * 32;
      const bool masked = tok + 32 > cols.to || tok < cols.from || (base[0] | base[1]) < 0;
      st.scales(kw, vw, zscale);
      st.score(s, tok + 4 * g, tok, cols, cap2);
      bool odd = false;
      if (masked) {
        const int there = (base[0] >= 0) + 2 * (base[1] >= 0);
        st.mask(s, there, tok + 4 * g, cols);
        odd = st.mask_values(there, tok + 4 * g, cols);
      }
      st.settle(s, zscale, cap2);
      st.weigh(s, zscale, cap2, pf);
      if (odd) st.weigh_odd(s, zscale, cap2, pf);
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
      load_values<D>(a, from, lanes, cur);
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

// The wide form, for prompts: every wave has a tile of 16 columns of its own, and
// all of a workgroup's go over the same tokens.  These are looked up once for
// all: each wave turns its share of the codes into the fragments of both
// products, laid out so that a fragment is read by 64 lanes in a row (16 bytes
// each, no bank conflict), in one of two buffers; while a stage of G groups of
// two halves of 16 tokens is computed on, the next one is filled into the other.
//
// Bound by the vector unit and the matrix cores one after the other: of four waves
// a SIMD 64 vector operations take 310 ns, 16 exponentials 233, 16 products 476, the
// first two together 543, the first and the last 696, all 862.  A group's 256
// capped columns (D = 128) are 16 products, 24 exponentials and reciprocals and
// ~95 others a wave, 1.3 us by that sum, and take 1.65: ragged prompts of 900 to 5600
// tokens, 32 heads of 128 columns, bf16, 676 us (0.57 PFLOP/s).  Prefixes with
// slopes, D = 256, 2000 to 5000 tokens, 662 us (0.55 PFLOP/s) with the vector unit 41%
// and the matrix cores 24% busy: the waves wait 60% of their cycles.  Documents of 700
// tokens in requests of 9000 and 16000, fp16, D = 64, 172 us, a third of it what an
// item costs by itself, the rest waves whose columns see nothing of a stage beside
// others' that do.  What was measured while a maximum could lag behind, 5% less of
// everything (us): two waves a SIMD of two tiles each with the scores of one group
// beside the weights of the last 770 (capped), with three and four waves a SIMD of
// one tile 751, without each wave converting the scales and with one operation less
// a weight 673, items weighed right 650; an item's first stage loaded and filled
// during the last one's no faster.
//
// Four waves a SIMD leave 128 registers (D = 256: three, 168), and the compiler
// spills: of D = 64 none or two, of D = 128 14 to 18, with slopes 26 and 33, of
// D = 256 30 to 40.  Most of them are stored and read once an item.  In the loop over
// groups stand three (masks alone) or four reads of scratch memory at D = 256, and in
// that over stages two at D = 128 with slopes, none without; such a read comes back
// behind the codes that are on their way for the next stage.  Steps of 64 tokens a
// wave are no faster at D = 64, and spill more at D = 128.
//
// Feature row n of fragment d of the second product is feature 32 (d / 2) + 2 n +
// d % 2: the two codes of one byte go to two fragments, and 16 lanes read 16
// bytes of a token.
template <int D>
struct Wide {
  static constexpr int WAVES = D == 256 ? 12 : 16, PER_SIMD = WAVES / 4;
  static constexpr int COLS = 16 * WAVES, THREADS = WAVES * 64;
  static constexpr int KS = D / 32, ND = D / 16;
  static constexpr int G = 256 / D;           // groups of a stage
  // Groups that an item costs by itself (us with 4 / 6 / 9: capped prompts 713 / 690 /
  // 696, prefixes 704 / 702 / 705; documents with 7 / 10 / 14: 191 / 188 / 188).
  static constexpr int ITEM = D == 64 ? 10 : 6;
  static constexpr int RUN = G * 32 * D * 2;  // bytes of a stage's keys or values
  static constexpr int BUF = 2 * RUN;         // keys, then values
  // Scales of a stage in fp32, per group: keys', values', and (fp16)
  // exponent_of these.
  static constexpr int SCALES = 3 * 32 * 4;
  static constexpr int kBuffers = kTable, kScales = kBuffers + 2 * BUF,
                       kShares = kScales + 2 * G * SCALES;
  // Eight waves fill two of a stage's 16 key fragments each, eight a pair of its 16
  // value fragments; where there are no sixteen, the same.
  static constexpr int VALUES_FROM = WAVES == 16 ? 8 : 0;
  static_assert(G * 2 * KS == 16 && G * ND == 16, "a stage");
};

// fill_table (kv4_tile.hpp) by THREADS threads, any multiple of 256.
template <int THREADS>
__device__ inline void fill_table_any(const Args& a, int hc, char* lds, int tid) {
  constexpr int UNITS = kTable / 16, TURNS = (UNITS + THREADS - 1) / THREADS;
  const uint16_t* lv = ((tid & 8) ? a.v_levels : a.k_levels) + hc * 16;
  const uint32_t low = lv[tid / 16 % 16];
  uint32_t high[TURNS];
#pragma unroll
  for (int r = 0; r < TURNS; ++r) high[r] = lv[min((r * THREADS + tid) / 256, 15)];
#pragma unroll
  for (int r = 0; r < TURNS; ++r) {
    const uint32_t w = high[r] << 16 | low;
    if (r * THREADS + tid < UNITS)
      *reinterpret_cast<u32x4*>(lds + (r * THREADS + tid) * 16) = u32x4{w, w, w, w};
  }
}

template <int DT, int D, int MODE>
__global__ void __launch_bounds__(Wide<D>::THREADS, Wide<D>::PER_SIMD)
kv4_masked_wide_kernel(const MArgs margs) {
  typedef Wide<D> L;
  constexpr int G = L::G, COLS = L::COLS, THREADS = L::THREADS;
  constexpr int KS = L::KS, ND = L::ND, NT = 1;
  const Args& args = margs.a;
  extern __shared__ __align__(16) char lds[];
  int* s_pre = reinterpret_cast<int*>(lds + L::kShares);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int table = -1;  // head whose table is in LDS
  typedef MWalk<COLS, THREADS, 32, L::ITEM> W;
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
    const int col0 = t.col0 + wave * 16;  // the wave's columns, in the request
    const int t0 = k.from, t1 = k.to, groups = (max(t1 - t0, 0) + 31) / 32;

    // The arguments that every tile needs, in scalar registers (left to itself
    // the compiler reads them again at each use, and waits).
    // (Global addresses by type: behind the asm nothing else says so, and a
    // load that might be LDS's would be waited for with every LDS read.)
    Global k_codes = (Global)a.k_codes, v_codes = (Global)a.v_codes;
    Global k_scales = (Global)a.k_scales, v_scales = (Global)a.v_scales;
    uint32_t bs = a.bs.d, bs_m = a.bs.m, num_blocks = a.num_blocks;
    int bs_sh = a.bs.sh, heads = a.heads;
    float zscale = capped(MODE) || (MODE == kBias && ma.cap2 != 0.f) ? ma.cap_scale : a.zscale;
    float cap2 = ma.cap2;
    asm volatile("" : "+s"(k_codes), "+s"(v_codes), "+s"(k_scales), "+s"(v_scales));
    asm volatile("" : "+s"(bs), "+s"(bs_m), "+s"(num_blocks), "+s"(bs_sh), "+s"(heads),
                 "+s"(zscale), "+s"(cap2));
    const int32_t* blocks = a.tables + (int64_t)t.req * a.table_stride;
    // 16-slot groups of the item's halves (of 16 tokens) over all heads, -1 where
    // there is none.  A lane has one of 64 halves, so that none is loaded in the
    // loop's way (scalar loads would be waited for with every LDS read).
    auto load_halves = [&](int part) {
      const int tok = t0 + (part * 64 + lane) * 16;
      const uint32_t at = __umulhi((uint32_t)tok, bs_m) >> bs_sh;  // (block sizes are 16 at least)
      const uint32_t b = tok < t1 ? (uint32_t)blocks[at] : 0xffffffffu;
      return b < num_blocks
                 ? (int)((b * heads + k.head) * (bs / 16) + ((uint32_t)tok - at * bs) / 16)
                 : -1;
    };
    int part = 0, halves = load_halves(0), more_halves = load_halves(1);
    // Half x, of this part or the next; past the item's end its last one, which is
    // at hand.  (Called where all lanes go the same way only: the registers are read
    // whatever lanes are active.)
    auto half = [&](int x) {
      x = min(x, 2 * groups - 1);
      if (x >> 6 != part) return __builtin_amdgcn_readlane(more_halves, x & 63);
      return __builtin_amdgcn_readlane(halves, x & 63);
    };
    // What the wave fills: key fragments of half kj of the stage, from step kc0 on; a
    // pair of value fragments of group vg.  The first G waves also have a group's
    // scales, a lane one of a key (the first 32) or of a value.
    constexpr int VAT = L::VALUES_FROM ? 0 : 2;  // place of the values' codes
    const bool keys = wave < 8, values = wave >= L::VALUES_FROM && wave < L::VALUES_FROM + 8;
    const int kj = wave * 2 / KS, kc0 = wave * 2 % KS;
    const int pair = wave - L::VALUES_FROM, vg = pair / (ND / 2), vu = pair % (ND / 2);
    uint32_t code[8 + VAT], scale = 0;
    auto load = [&](int x0) {  // of the stage from half x0 on
      if (keys) {
        const Global kp = k_codes + (int64_t)max(half(x0 + kj), 0) * (16 * D / 2);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          code[e] = at<uint32_t>(kp, n * (D / 2) + g * (D / 8) + (kc0 + e) * 4);
      }
      if (values) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const Global vp = v_codes + (int64_t)max(half(x0 + 2 * vg + j), 0) * (16 * D / 2);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            code[VAT + 4 * j + i] = at<uint8_t>(vp, (4 * g + i) * (D / 2) + 16 * vu + n);
        }
      }
      if (wave < G) {
        const int base0 = half(x0 + 2 * wave), base1 = half(x0 + 2 * wave + 1);
        const int base = max((lane & 16) ? base1 : base0, 0);
        const Global from = lane < 32 ? k_scales : v_scales;
        scale = *(const uint16_t __attribute__((address_space(1)))*)(from + (int64_t)base * 32 +
                                                                     2 * n);
      }
    };
    auto fill = [&](int buffer) {
      char* buf = lds + L::kBuffers + buffer * L::BUF + lane * 16;
      if (keys) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          u32x4 f;
#pragma unroll
          for (int b = 0; b < 4; ++b) f[b] = lookup<0>(code[e], b, loff);
          *reinterpret_cast<u32x4*>(buf + (kj * KS + kc0 + e) * 1024) = f;
        }
      }
      if (values) {
        u32x4 even, odd;
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // (a look-up takes its byte alone)
          const uint32_t b0 = code[VAT + 2 * c], b1 = code[VAT + 2 * c + 1];
          even[c] = lookup<128>((b0 & 15u) | b1 << 4, 0, loff);
          odd[c] = lookup<128>(b0 >> 4 | (b1 & 0xf0u), 0, loff);
        }
        char* vb = buf + L::RUN + 2 * pair * 1024;
        *reinterpret_cast<u32x4*>(vb) = even;
        *reinterpret_cast<u32x4*>(vb + 1024) = odd;
      }
      if (wave < G) {
        float* to =
            reinterpret_cast<float*>(lds + L::kScales + (buffer * G + wave) * L::SCALES);
        float v = from16<DT>(scale);
        if (MODE != kMask && lane < 32) v *= zscale;
        to[lane] = v;
        if (DT == FKC_F16 && lane >= 32) to[32 + lane] = exponent_of(v);
      }
    };
    auto column = [&](const Args& a, int y, int& row, int& head, int& i) {
      const int col = col0 + 16 * y + n;
      i = (int)a.gdiv.div(min(col, ncols - 1));
      row = col < ncols ? t.row0 + i : -1;
      head = k.head * a.G + (min(col, ncols - 1) - i * a.G);
    };

    if (groups > 0) load(0);
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
    // The wave's groups g0 .. g1 - 1 of the item's.
    int g0 = INT32_MAX, g1 = INT32_MAX;
    if (max(cols.lo, t0) < min(cols.hi, t1)) {
      g0 = (max(cols.lo, t0) - t0) / 32;
      g1 = (min(cols.hi, t1) - t0 + 31) / 32;
    }
    if (table != k.head) {  // (every look-up of the last item was before its last barrier)
      table = k.head;
      fill_table_any<THREADS>(a, k.head, lds, tid);
      lds_barrier();
    }

    MState<DT, D, NT, MODE, true> st;
    st.clear();
    if (groups > 0) {
      fill(0);
      load(2 * G);
      lds_barrier();
      uint64_t there = __ballot(halves >= 0);  // a bit for each half of the part
      for (int i0 = 0, buffer = 0; i0 < groups; i0 += G, buffer ^= 1) {
        fill(buffer ^ 1);
        load(2 * i0 + 4 * G);
        const char* buf = lds + L::kBuffers + buffer * L::BUF + lane * 16;
#pragma unroll
        for (int h = 0; h < G; ++h) {
          const int i = i0 + h;
          if (i < g0 || i >= g1) continue;  // none of the wave's columns sees them
          const int tok = t0 + i * 32;
          const f32x4* sc = reinterpret_cast<const f32x4*>(
              lds + L::kScales + (buffer * G + h) * L::SCALES) + g;
          f32x4 z[NT][2];
#pragma unroll
          for (int c = 0; c < KS; ++c)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const u32x4 kf =
                  *reinterpret_cast<const u32x4*>(buf + ((2 * h + j) * KS + c) * 1024);
#pragma unroll
              for (int y = 0; y < NT; ++y)
                z[y][j] = mfma<DT>(kf, qf[y][c], c ? z[y][j] : f32x4{0.f, 0.f, 0.f, 0.f});
            }
          const int both = (int)(there >> (2 * i & 63)) & 3;
          const bool masked = tok + 32 > cols.to || tok < cols.from || both != 3;
          st.ks[0] = sc[0];
          st.ks[1] = sc[4];
          st.score(z, tok + 4 * g, tok, cols, cap2);
          if (masked) st.mask(z, both, tok + 4 * g, cols);
          if constexpr (DT == FKC_F16) {
            st.ve[0] = sc[16];
            st.ve[1] = sc[20];
          }
          st.settle(z, zscale, cap2);
          st.vs[0] = sc[8];
          st.vs[1] = sc[12];
          bool odd = false;
          if (masked) odd = st.mask_values(both, tok + 4 * g, cols);
          u32x4 pf[NT];
          st.weigh(z, zscale, cap2, pf);
          if (odd) st.weigh_odd(z, zscale, cap2, pf);
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const u32x4 vf = *reinterpret_cast<const u32x4*>(buf + L::RUN + (h * ND + d) * 1024);
#pragma unroll
            for (int y = 0; y < NT; ++y) st.o[y][d] = mfma<DT>(vf, pf[y], st.o[y][d]);
          }
        }
        if ((2 * (i0 + G)) >> 6 != part) {
          ++part;
          halves = more_halves;
          there = __ballot(halves >= 0);
          more_halves = load_halves(part + 1);
        }
        lds_barrier();
      }
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
          const int64_t at = k.slot() * COLS + wave * 16 + 16 * y + n;
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

// Granules of a share at least, and up to how many granules a context is never
// cut, as for kv4_attend.hip; a window bounds what a tile of a causal call sees.
// (Capped, bf16, 8 heads of 4 query heads, us whole / cut.  One query of 1, 8 or
// 64 requests: D = 128, 1536 tokens 16.9 / 16.8, 17.4 / 19.6, 27.0 / 30.4, 3000 tokens
// 25.8 / 18.2, 26.7 / 23.4, 43.4 / 45.0; D = 256, 777 tokens 21.1 / 17.0, 21.2 / 19.1,
// 28.5 / 30.9, 1536 tokens 29.8 / 20.0, 30.6 / 23.9, 41.0 / 42.3.  1, 4 or 16 prompts:
// D = 128, 512 tokens 38 / 38, 43 / 65, 132 / 111, 1024 tokens 65 / 54, 120 / 115,
// 376 / 349; D = 256, 1024 tokens 93 / 105, 211 / 221, 728 / 724, 2048 tokens 220 / 199,
// 638 / 609, 2276 / 2220.)
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

constexpr int wide_waves(int D) { return D == 256 ? 12 : 16; }
// Columns of an average request up to which the split form is taken.
constexpr int wide_from(int D) { return D == 64 ? 352 : D == 128 ? 448 : 288; }
constexpr int waves_of(int D) { return D == 256 ? 4 : 8; }

// reach: tokens that one query sees at most (max_seq, or the window).
Plan make_plan(const fkc_kv4_cache& c, int64_t H, int64_t T, int64_t R, int64_t max_seq,
               int64_t reach, bool ragged) {
  Plan p;
  const int64_t G = H / c.heads;
  // By the columns of an average request.  Measured on 8 requests of 4096 tokens, 8
  // heads of 4 query heads, bf16, capped, us with one tile per workgroup / with two /
  // in the wide form, for so many columns each (slopes and masks the same within
  // 10%, and better in the wide form by 5 to 20% at D = 64):
  //   D =  64     64: 39 / 39 / 44     96: 47 / 42 / 52     256: 82 / 71 / 88
  //              320: 106 / 95 / 106  384: 118 / 110 / 105  512: 153 / 130 / 106
  //   D = 128     64: 48 / 48 / 64     96: 59 / 53 / 74     256: 106 / 88 / 115
  //              384: 155 / 139 / 148 512: 203 / 160 / 147
  //   D = 256     96: 94 / - / 144    256: 182 / - / 234    320: 247 / - / 236
  const int64_t avg = R > 0 ? T * G / R : 0;
  p.wide = avg > wide_from((int)c.D);
  p.nt = p.wide ? 1 : c.D < 256 && avg > 64 ? 2 : 1;
  p.waves = p.wide ? wide_waves((int)c.D) : p.nt == 2 ? 4 : waves_of((int)c.D);
  const int64_t cols = p.cols();
  p.tiles_per_req = (int)((G + cols - 1) / cols);
  p.ntiles = ragged ? T * G / cols + R + 1 : R * p.tiles_per_req;
  const int64_t len = std::min(max_seq, reach + (cols + G - 1) / G + 16);
  p.whole = len <= (p.wide ? kWideWhole * 32 : kWhole * 32 * p.waves) &&
            p.ntiles * c.heads < kMostThreads / (64 * p.waves);
  p.wgs = p.whole ? p.ntiles * c.heads : (p.wide ? 1 : 2) * (int64_t)device_shape().cus;
  return p;
}

template <int DT, int D, int COLS, int GR, int ITEM, int THREADS, typename K>
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
  if (!p.whole && m.a.cu_q != nullptr)
    hipLaunchKernelGGL((kv4_tiles_kernel<COLS, GR, ITEM>), dim3((uint32_t)((p.ntiles + 3) / 4)),
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
  return launch<DT, D, 16 * NT, WAVES * 32, kItem, WAVES * 64>(
      &kv4_masked_split_kernel<DT, D, NT, WAVES, MODE>, set,
      kTable + kJoin + MWalk<16 * NT, WAVES * 64, 1, 0>::kInts * 4, m, p, s);
}

template <int DT, int D, int MODE>
int launch_wide(const MArgs& m, const Plan& p, hipStream_t s) {
  static std::atomic<uint64_t> set{0};
  typedef Wide<D> L;
  return launch<DT, D, L::COLS, 32, L::ITEM, L::THREADS>(
      &kv4_masked_wide_kernel<DT, D, MODE>, set,
      L::kShares + MWalk<L::COLS, L::THREADS, 1, 0>::kInts * 4, m, p, s);
}

template <int DT, int D, int MODE>
int launch_mode(const MArgs& m, const Plan& p, hipStream_t s) {
  if (p.wide) return launch_wide<DT, D, MODE == kBoth ? kBias : MODE>(m, p, s);
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

// Caps above this take kBoth, with slopes of 0: kCap's tanh is off by 2^-21 of the cap,
// 2^-13 of a weight here, a quarter of what rounding one to fp16 may cost.  Prompts
// capped at 30 take 690 us with kCap and 951 with the series, single tokens 13.4 and
// 14.6.
constexpr float kSharp = 256.f;

int launch_kv4_attend_scored(const fkc_kv4_cache& c, const Kv4Attend& x, const Kv4Scores& sc,
                             void* ws, hipStream_t s) {
  const Plan p = make_plan(c, x.H, x.T, x.R, x.max_seq, reach_of(x.max_seq, sc, x.causal),
                           x.cu_q != nullptr);
  const int G = (int)(x.H / c.heads);
  // Weights of a head's items are summed in 32 bits.
  constexpr int kMostItem = 10;
  static_assert(kItem <= kMostItem && Wide<64>::ITEM <= kMostItem &&
                Wide<128>::ITEM <= kMostItem && Wide<256>::ITEM <= kMostItem, "");
  const int64_t gr = p.wide ? 32 : 32 * p.waves;
  if (p.ntiles > INT32_MAX / (x.max_seq / gr + 2 + kMostItem) ||
      (!p.whole && p.ntiles + 3 >= kMostThreads / 64))  // (kv4_tiles_kernel: a wave each)
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
    // (a product of it with a key's scale stays finite for these up to 2^28)
    m.cap_scale = (float)std::min(2 * scale / sc.softcap, 0x1p100);
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
    if (sc.softcap > (sc.slopes != nullptr ? 0.f : kSharp))
      return launch_mode<DT, DD, kBoth>(m, p, s);
    if (sc.slopes != nullptr) return launch_mode<DT, DD, kBias>(m, p, s);
    if (sc.softcap > 0.f) return launch_mode<DT, DD, kCap>(m, p, s);
    return launch_mode<DT, DD, kMask>(m, p, s);
  });
}

}  // namespace fkc
