// What the kernels of attention over the 4-bit cache share: fragments of codes
// and levels, the running softmax, the joining of cut items.  (How a tile is
// computed: kv4_attend.hip.)
#pragma once

#include <type_traits>

#include "device_util.hpp"
#include "fkc_internal.hpp"

namespace fkc {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ inline f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == FKC_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two floats to 16 bits each, to nearest even.
template <int DT>
__device__ inline uint32_t pack2(float a, float b) {
  const f32x2 v = {a, b};
  if constexpr (DT == FKC_F16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// A barrier for what is passed through LDS.  (__syncthreads also waits for every
// global load and store that is on its way: those prefetched for the next tile
// and the results of the last item.)
__device__ inline void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int DT>
__device__ inline float from16(uint32_t bits) {
  using E = Elem<DT>;
  return E::load(__builtin_bit_cast(typename E::T, (uint16_t)bits));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.4028235e38f;  // below every score; finite, so that a
                                           // difference of two is no NaN (products
                                           // of it are kept finite: State::base2)
constexpr int kEntry = 256;                // bytes of a table entry
constexpr int kTable = 256 * kEntry;
constexpr int kJoin = 8 * 16 * 8;          // maxima and sums of up to 8 waves

// Threads of a launch stay below this; more workgroups of whole items than that
// leaves room for become shares.
constexpr int64_t kMostThreads = (int64_t)1 << 32;

// 1 / l for a sum of weights, 0 where nothing was seen; NaN stays.
__device__ inline float inverse(float l) { return l != 0.f ? 1.f / l : 0.f; }

// log(2^m l): the exponents of both are added before anything is rounded.
__device__ inline float log_sum(float m, float l) {
  const int e = (int)(__float_as_uint(l) >> 23) - 127;
  return l != 0.f ? (m + e) * kLn2 + __logf(ldexpf(l, -e)) : -INFINITY;
}

// Read by scalar loads: nothing writes it while the kernel runs.
typedef const int32_t __attribute__((address_space(4))) * Const32;

struct Args {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  const uint8_t* k_codes;
  const uint8_t* v_codes;
  const uint16_t* k_scales;
  const uint16_t* v_scales;
  const uint16_t* k_levels;
  const uint16_t* v_levels;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* seq;
  const int32_t* cu_q;
  uint16_t* out;
  float* lse;
  float* part;     // two partial results of COLS columns per workgroup:
  float* part_ml;  // unnormalised outputs; maximum (base 2) and sum
  int4* desc;      // per workgroup: what is to be joined from it on
  FastDiv bs, gdiv;
  uint32_t num_blocks;
  int heads, H, G, T, R, max_seq, causal;
  int whole;          // one item per workgroup, else equal shares
  int min_share;      // granules a share has at least
  int tiles_per_req;  // without cu_q
  float zscale;       // |sm_scale| * log2(e), above 0
  uint32_t qsign;     // flips the queries' signs where sm_scale is negative
};

// What a tile of COLS columns is.  With cu_q the tiles of request r are
// numbered from floor(cu_q[r] G / COLS) + r on, which leaves each request room
// for all of its own whatever the lengths; rows past the last request are a
// request R without tokens.
struct Tile {
  int row0, nq;  // first query and number of queries of the request
  int col0;      // first column of the tile
  int end;       // tokens of the request
  int req;
};

__device__ inline int tokens_of(const Args& a, int r) {
  return r < a.R && a.num_blocks != 0 ? min(max(a.seq[r], 0), a.max_seq) : 0;
}

template <int COLS>
__device__ inline bool find_tile(const Args& a, int tile, Tile& t) {
  if (a.cu_q == nullptr) {
    t.req = tile / a.tiles_per_req;
    if (t.req >= a.R) return false;
    t.row0 = t.req;
    t.nq = 1;
    t.col0 = (tile - t.req * a.tiles_per_req) * COLS;
  } else {
    auto first = [&](int r) {
      const int64_t c = min(max(a.cu_q[r], 0), a.T);
      return (int)((uint64_t)(c * a.G) / COLS) + r;
    };
    int lo = 0, len = a.R + 1;
    while (len > 1) {
      const int half = len >> 1;
      if (first(lo + half) <= tile) lo += half;
      len -= half;
    }
    t.req = lo;
    t.row0 = min(max(a.cu_q[lo], 0), a.T);
    const int next = lo < a.R ? min(max(a.cu_q[lo + 1], 0), a.T) : a.T;
    t.nq = max(next - t.row0, 0);
    t.col0 = (tile - first(lo)) * COLS;
  }
  t.end = tokens_of(a, t.req);
  return t.col0 >= 0 && (int64_t)t.col0 < (int64_t)t.nq * a.G;
}

// Tokens that query i of a request sees.
__device__ inline int sees(const Args& a, const Tile& t, int i) {
  return a.causal ? min(max(0, t.end - t.nq + 1 + i), t.end) : t.end;
}

// Tables of a head's level pairs, by the whole workgroup: thread tid writes
// entries of low level tid / 16 % 16 only, so it needs that one and, of the
// high ones, those its turns r come to.
template <int THREADS>
__device__ inline void fill_table(const Args& a, int hc, char* lds, int tid) {
  constexpr int TURNS = kTable / 16 / THREADS, PER = 16 / TURNS;  // high levels per turn
  const uint16_t* lv = ((tid & 8) ? a.v_levels : a.k_levels) + hc * 16;
  const uint32_t low = lv[tid / 16 % 16];
  u32x4 high[2];
  high[0] = reinterpret_cast<const u32x4*>(lv)[0];
  high[1] = reinterpret_cast<const u32x4*>(lv)[1];
  const bool odd = tid / 256;  // with two high levels per turn: the second
#pragma unroll
  for (int r = 0; r < TURNS; ++r) {
    const int h = r * PER;
    const uint32_t two = high[h / 8][h / 2 % 4];
    const uint32_t w = ((PER == 2 ? odd : h & 1) ? two & 0xffff0000u : two << 16) | low;
    *reinterpret_cast<u32x4*>(lds + (r * THREADS + tid) * 16) = u32x4{w, w, w, w};
  }
}

// The codes and scales of 32 tokens, as lane (n, g) needs them.
template <int D>
struct Codes {
  static constexpr int KD = D / 32;          // dwords of codes: D / 4 features
  static constexpr int VB = D / 32;          // bytes of codes per token: D / 16
  uint32_t k[2][KD];                         // token n of each half
  uint32_t v[2][4][VB > 4 ? VB / 4 : 1];     // tokens 4 g + i
  uint2 ks[2], vs[2];                        // their scales, 16 bits each
};

// A lane's byte offsets into a 16-slot group: keys and values (token 4 g).
template <int D>
struct Lane {
  uint32_t k, v, s;
  __device__ inline Lane(int n, int g)
      : k(n * (D / 2) + g * (D / 8)), v(4 * g * (D / 2) + n * (D / 32)), s(8 * g) {}
};

typedef const char __attribute__((address_space(1))) * Global;

template <typename T>
__device__ inline T at(Global base, uint32_t off) {
  typedef uint32_t Two __attribute__((ext_vector_type(2)));
  if constexpr (std::is_same<T, uint2>::value) {
    const Two v = *(const Two __attribute__((address_space(1)))*)(base + off);
    return uint2{v[0], v[1]};
  } else {
    return *(const T __attribute__((address_space(1)))*)(base + off);
  }
}

template <typename T>
__device__ inline T at(const void* base, uint32_t off) {
  return *reinterpret_cast<const T*>(static_cast<const char*>(base) + off);
}

template <int D>
__device__ inline void load_keys(const Args& a, const int (&base)[2], const Lane<D>& p,
                                 Codes<D>& c) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    // a missing half reads slot 0
    const uint8_t* kp = a.k_codes + (int64_t)max(base[j], 0) * (16 * D / 2);
    if constexpr (D == 64) {
      const uint2 x = at<uint2>(kp, p.k);
      c.k[j][0] = x.x;
      c.k[j][1] = x.y;
    } else {
#pragma unroll
      for (int w = 0; w < Codes<D>::KD; w += 4) {
        const u32x4 x = at<u32x4>(kp, p.k + w * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) c.k[j][w + e] = x[e];
      }
    }
  }
}

template <int D>
__device__ inline void load_values(const Args& a, const int (&base)[2], const Lane<D>& p,
                                   Codes<D>& c) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint8_t* vp = a.v_codes + (int64_t)max(base[j], 0) * (16 * D / 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (D == 64) {
        c.v[j][i][0] = at<uint16_t>(vp, p.v + i * (D / 2));
      } else if constexpr (D == 128) {
        c.v[j][i][0] = at<uint32_t>(vp, p.v + i * (D / 2));
      } else {
        const uint2 x = at<uint2>(vp, p.v + i * (D / 2));
        c.v[j][i][0] = x.x;
        c.v[j][i][1] = x.y;
      }
    }
  }
}

template <int D>
__device__ inline void load_scales(const Args& a, const int (&base)[2], const Lane<D>& p,
                                   Codes<D>& c) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t row = (int64_t)max(base[j], 0) * 16;
    c.ks[j] = at<uint2>(a.k_scales + row, p.s);
    c.vs[j] = at<uint2>(a.v_scales + row, p.s);
  }
}

// Codes of two tokens, eight features each, as pairs of one feature: byte f of
// even holds feature 2 f of both, of odd feature 2 f + 1.
__device__ inline void pair_tokens(uint32_t t0, uint32_t t1, uint32_t& even, uint32_t& odd) {
  constexpr uint32_t lo = 0x0f0f0f0fu;
  even = (t0 & lo) | (t1 << 4 & ~lo);
  odd = (t0 >> 4 & lo) | (t1 & ~lo);
}

// Entry of byte b of w in the table: `off` is the lane's offset in an entry.
// The table is the start of the workgroup's LDS (its kernels have dynamic LDS
// only), so the v_perm is the whole address; through the pointer to the table
// every look-up would cost an addition of that 0.
template <int PART>  // 0: keys, 128: values
__device__ inline uint32_t lookup(uint32_t w, int b, uint32_t off) {
  typedef const char __attribute__((address_space(3))) * LdsPtr;
  typedef const uint32_t __attribute__((address_space(3))) * LdsWord;
  const uint32_t at = __builtin_amdgcn_perm(w, off, 0x0c0c0000u | (uint32_t)(4 + b) << 8);
  return *(LdsWord)((LdsPtr)(uintptr_t)at + PART);
}

__device__ inline int64_t scalar64(int64_t v) {
  return (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

// Keeps what a rarely taken branch computes inside it (selects in its place
// would run for every tile).
__device__ inline void rare(float& v) { asm volatile("" : "+v"(v)); }

// A wave's NT tiles of 16 columns: outputs and running maxima and sums, all fp32.
// What is rounded to the type is a weight times its value scale, for the second
// product: matrix cores take both factors in 16 bits or both in 32 at a sixteenth
// of the rate.  The sum of weights is that of the unrounded ones, so each term of
// an output is off by half a unit in the last place at most, and these errors
// average out: relative to 64-bit results single bf16 tokens are 1.69e-3 off and
// prompts 1.76e-3, of which 1.66e-3 is the rounding of the result, fp16 prompts of 256
// columns 2.16e-4 and 2.07e-4.
//   bf16: m is the largest score before its (positive) scale zscale, and a
// weight is 2^(z zscale - m zscale).
//   fp16 has few exponents, and a token's value scale is part of what is rounded
// to it: m is the largest z zscale + log2 of the value scale (rounded up), and a
// weight 2^(z zscale - m + 14), so that weight times scale is at most 2^14 and
// the column's largest above 2^12, whatever the scales are.
template <int DT, int D, int NT>
struct State {
  static constexpr int ND = D / 16;
  float m[NT], l[NT];
  f32x4 o[NT][ND];
  __device__ inline void clear() {
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      m[y] = kLowest;
      l[y] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[y][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  // What the weights so far are relative to, as a power of two.  Finite: of a
  // column that has seen nothing m is kLowest, and with a scale above 1 the
  // product would be -inf, from which a masked score's own -inf differs by NaN.
  // (Nor +inf: of scores that large every weight would be 0 instead.)
  __device__ inline float base2(int y, float zscale) const {
    return DT == FKC_F16 ? m[y] - 14.f
                         : __builtin_amdgcn_fmed3f(m[y] * zscale, kLowest, -kLowest);
  }
  // Scores s of 32 tokens (their halves' groups base, this lane's first token
  // tok) to weights, packed as the second product reads them.  masked: some
  // column does not see all of them; lim: what each column sees, lim_max the
  // last.
  __device__ inline void weights(f32x4 (&s)[NT][2], const uint2 (&kw)[2], const uint2 (&vw)[2],
                                 bool masked, int base0, int base1, int tok, const int (&lim)[NT],
                                 int lim_max, float zscale, u32x4 (&pf)[NT]) {
    float ks[2][4], vs[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t kx = i < 2 ? kw[j].x : kw[j].y, vx = i < 2 ? vw[j].x : vw[j].y;
        ks[j][i] = from16<DT>((i & 1) ? kx >> 16 : kx & 0xffffu);
        vs[j][i] = from16<DT>((i & 1) ? vx >> 16 : vx & 0xffffu);
      }
    if (masked) {  // what lies past the requests' tokens is anything
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((j ? base1 : base0) < 0 || tok + 16 * j + i >= lim_max) vs[j][i] = 0.f;
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
      if (masked) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if ((j ? base1 : base0) < 0 || tok + 16 * j + i >= lim[y]) z[j][i] = -INFINITY;
            rare(z[j][i]);
          }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top = fmaxf(top, DT == FKC_F16 ? __builtin_fmaf(z[j][i], zscale, ve[j][i]) : z[j][i]);
      if (__any(top > m[y])) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float nm = fmaxf(m[y], top);
        const float f =
            __builtin_amdgcn_exp2f(DT == FKC_F16 ? m[y] - nm : (m[y] - nm) * zscale);
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
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[j][i], zscale, -mz));
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
  // Sums of a column over its four lanes (which share m).
  __device__ inline void join_lanes() {
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      l[y] += __shfl_xor(l[y], 16, 64);
      l[y] += __shfl_xor(l[y], 32, 64);
    }
  }
};

// The kernel's (only) argument, read again from where it lies: what is not used
// between two such places takes no registers there.
template <typename A>
__device__ inline const A& arguments_as() {
  auto p = (const A __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const A*)p;
}

// Joins the parts of a cut item: the workgroup's that its first unit was in
// (its second slot) and the following ones' (their first).  D / 4 lanes per
// column; of few parts each thread adds its own up, of many all threads share
// the parts of JC columns: weights into LDS, PARTS parts at a time, every load
// independent of the others.
template <int DT, int D>
__device__ inline void write_joined(const Args& a, const int4& item, int col, int sub, f32x4 v,
                                    float m, float l) {
  const int i = (int)a.gdiv.div(item.z + col);
  const int64_t at =
      (int64_t)(item.y + i) * a.H + (item.w & 0xffff) * a.G + (item.z + col - i * a.G);
  const float f = inverse(l);
  uint2 w;
  w.x = pack2<DT>(v[0] * f, v[1] * f);
  w.y = pack2<DT>(v[2] * f, v[3] * f);
  *reinterpret_cast<uint2*>(a.out + at * D + 4 * sub) = w;
  if (sub == 0 && a.lse != nullptr) a.lse[at] = log_sum(m, l);
}

template <int DT, int D, int COLS>
__global__ void __launch_bounds__(256)
kv4_join_kernel(const Args a) {
  constexpr int LPC = D / 4, CP = 256 / LPC, JC = 4, PARTS = 64, FEW = 4;
  __shared__ f32x4 so[256];
  __shared__ float sw[JC][PARTS];
  int4 item = a.desc[blockIdx.x];
  if (item.x == 0) return;
  item.x = min(item.x, (int)(gridDim.x - blockIdx.x));  // (see Shares::find)
  const int ncols = item.w >> 16;
  const int sub = threadIdx.x % LPC, part = threadIdx.x / LPC;
  // row of part c, column col in part and part_ml
  auto place = [&](int c, int col) {
    return (((int64_t)blockIdx.x + c) * 2 + (c ? 0 : 1)) * COLS + min(col, COLS - 1);
  };
  if (item.x <= FEW) {
    for (int col = blockIdx.y * CP + part; col < ncols; col += gridDim.y * CP) {
      f32x4 v[FEW];
      float2 ml[FEW];
      float m = kLowest, l = 0.f;
#pragma unroll
      for (int c = 0; c < FEW; ++c) {
        if (c >= item.x) break;
        ml[c] = *reinterpret_cast<const float2*>(a.part_ml + 2 * place(c, col));
        v[c] = *reinterpret_cast<const f32x4*>(a.part + place(c, col) * D + 4 * sub);
      }
#pragma unroll
      for (int c = 0; c < FEW; ++c)
        if (c < item.x) m = fmaxf(m, ml[c].x);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < FEW; ++c) {
        if (c >= item.x) break;
        const float w = __builtin_amdgcn_exp2f(ml[c].x - m);
        l += ml[c].y * w;
        o += v[c] * w;
      }
      write_joined<DT, D>(a, item, col, sub, o, m, l);
    }
    return;
  }
  // One wave per column: a lane per part.
  const int j = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int col0 = blockIdx.y * JC; col0 < ncols; col0 += gridDim.y * JC) {
    float m = kLowest, l = 0.f;
    f32x4 o[JC];
#pragma unroll
    for (int x = 0; x < JC; ++x) o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c0 = 0; c0 < item.x; c0 += PARTS) {
      f32x4 v[JC][PARTS / CP];
#pragma unroll
      for (int i = 0; i < PARTS / CP; ++i)
#pragma unroll
        for (int x = 0; x < JC; ++x)
          if (c0 + i * CP < item.x)
            v[x][i] = *reinterpret_cast<const f32x4*>(
                a.part + place(min(c0 + i * CP + part, item.x - 1), col0 + x) * D + 4 * sub);
      float m2 = kLowest, l2 = 0.f;
      if (c0 + lane < item.x) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * place(c0 + lane, col0 + j));
        m2 = ml.x;
        l2 = ml.y;
      }
      float nm = fmaxf(m, m2);
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) nm = fmaxf(nm, __shfl_xor(nm, off, 64));
      const float f = __builtin_amdgcn_exp2f(m - nm), w = __builtin_amdgcn_exp2f(m2 - nm);
      m = nm;
      l = l * f + wave_sum(l2 * w);
      __syncthreads();  // sw is read
      sw[j][lane] = c0 + lane < item.x ? w : 0.f;
      if (lane == 0) reinterpret_cast<float*>(so)[j] = f;
      __syncthreads();
#pragma unroll
      for (int x = 0; x < JC; ++x) {
        o[x] *= reinterpret_cast<const float*>(so)[x];
#pragma unroll
        for (int i = 0; i < PARTS / CP; ++i) {
          const float wt = sw[x][i * CP + part];
          // (the column or part may not exist; what stands there may be NaN)
          if (wt != 0.f) o[x] += v[x][i] * wt;
        }
      }
    }
    __syncthreads();
    if (lane == 0) {
      sw[j][0] = l;
      sw[j][1] = m;
    }
#pragma unroll
    for (int x = 0; x < JC; ++x) {
      __syncthreads();
      so[threadIdx.x] = o[x];
      __syncthreads();
      if (threadIdx.x >= LPC || col0 + x >= ncols) continue;
      f32x4 sum = so[sub];
#pragma unroll
      for (int c = 1; c < CP; ++c) sum += so[c * LPC + sub];
      write_joined<DT, D>(a, item, col0 + x, sub, sum, sw[x][1], sw[x][0]);
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace fkc
