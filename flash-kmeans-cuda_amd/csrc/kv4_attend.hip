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

template <int DT>
__device__ inline float from16(uint32_t bits) {
  using E = Elem<DT>;
  return E::load(__builtin_bit_cast(typename E::T, (uint16_t)bits));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.4028235e38f;  // below every score; finite, so that
                                           // a difference of two is no NaN
constexpr int kEntry = 256;                // bytes of a table entry
constexpr int kTable = 256 * kEntry;

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
  float* part;     // (T, H, chunks, D) unnormalised outputs
  float* part_ml;  // (T, H, chunks, 2) maximum (base 2), sum
  FastDiv bs, gdiv;
  uint32_t num_blocks;
  int heads, H, G, T, R, max_seq, causal;
  int chunk, chunks;  // tokens per workgroup, workgroups along the context
  int tiles_per_req;  // without cu_q
  float zscale;       // sm_scale * log2(e)
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
  return a.causal ? max(0, t.end - t.nq + 1 + i) : t.end;
}

// Tables of a head's level pairs, by the whole workgroup.
template <int THREADS>
__device__ inline void fill_table(const Args& a, int hc, char* lds) {
  const uint16_t* kl = a.k_levels + hc * 16;
  const uint16_t* vl = a.v_levels + hc * 16;
#pragma unroll
  for (int r = 0; r < kTable / 16 / THREADS; ++r) {
    const int i = r * THREADS + threadIdx.x;
    const int e = i / (kEntry / 16);
    const uint16_t* lv = (i & 8) ? vl : kl;
    const uint32_t w = lv[e & 15] | (uint32_t)lv[e >> 4] << 16;
    *reinterpret_cast<u32x4*>(lds + i * 16) = u32x4{w, w, w, w};
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

template <int D>
__device__ inline void load_codes(const Args& a, const int (&base)[2], int n, int g,
                                  Codes<D>& c) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t row = (int64_t)max(base[j], 0) * 16;  // a missing half reads slot 0
    const uint8_t* kp = a.k_codes + row * (D / 2) + (uint32_t)(n * (D / 2) + g * (D / 8));
#pragma unroll
    for (int w = 0; w < Codes<D>::KD; w += 4) {
      if constexpr (D == 64) {
        const uint2 x = *reinterpret_cast<const uint2*>(kp);
        c.k[j][0] = x.x;
        c.k[j][1] = x.y;
      } else {
        const u32x4 x = *reinterpret_cast<const u32x4*>(kp + w * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) c.k[j][w + e] = x[e];
      }
    }
    const uint8_t* vp = a.v_codes + row * (D / 2) + (uint32_t)(4 * g * (D / 2) + n * (D / 32));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (D == 64) {
        c.v[j][i][0] = *reinterpret_cast<const uint16_t*>(vp + i * (D / 2));
      } else if constexpr (D == 128) {
        c.v[j][i][0] = *reinterpret_cast<const uint32_t*>(vp + i * (D / 2));
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(vp + i * (D / 2));
        c.v[j][i][0] = x.x;
        c.v[j][i][1] = x.y;
      }
    }
    c.ks[j] = *reinterpret_cast<const uint2*>(a.k_scales + row + 4 * g);
    c.vs[j] = *reinterpret_cast<const uint2*>(a.v_scales + row + 4 * g);
  }
}

// Entry of byte b of w in the table: `off` is the lane's offset in an entry.
// The table is the start of the workgroup's LDS (its kernels have dynamic LDS
// only), so the v_perm is the whole address; through the pointer to the table
// every look-up would cost an addition of that 0.
__device__ inline uint32_t lookup(uint32_t w, int b, uint32_t off) {
  typedef const uint32_t __attribute__((address_space(3))) * LdsPtr;
  return *(LdsPtr)(uintptr_t)__builtin_amdgcn_perm(w, off,
                                                   0x0c0c0000u | (uint32_t)(4 + b) << 8);
}

// The split form: the WAVES waves of a workgroup share NT tiles of 16 columns
// and take 32 tokens of its chunk in turn, each with its own running maximum
// and sum; they are joined in LDS at the end, chunks by a second kernel.
template <int DT, int D, int NT, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, WAVES * (NT * D > 256 ? 1 : 2) / 4)
kv4_split_kernel(const Args a) {
  constexpr int COLS = 16 * NT;
  constexpr int KS = D / 32;  // steps of the first product
  constexpr int ND = D / 16;  // feature tiles of the second
  extern __shared__ __align__(16) char lds[];
  int* s_base = reinterpret_cast<int*>(lds + kTable);

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  // Heads first, chunks last: consecutive workgroups go to the eight XCDs in
  // turn, and every head has as much to do as the next, while later chunks
  // are those of the longest requests only.
  const int items = gridDim.x / a.chunks;
  const int c = blockIdx.x / items, idx = blockIdx.x - c * items;
  const int hc = idx % a.heads;
  Tile t;
  if (!find_tile<COLS>(a, idx / a.heads, t)) return;
  const int ncols = t.nq * a.G;
  const int last = min(t.col0 + COLS, ncols) - 1;
  const int lim_min = sees(a, t, (int)a.gdiv.div(t.col0));
  const int lim_max = sees(a, t, (int)a.gdiv.div(last));
  const int t0 = c * a.chunk;
  if (t0 >= lim_max && c != 0) return;
  const int t1 = min(t0 + a.chunk, lim_max);

  // 16-token groups of the chunk: their place in the cache, -1 where there
  // is no block.
  for (int i = threadIdx.x; i < (t1 - t0 + 31) / 32 * 2; i += WAVES * 64) {
    const int tok = t0 + i * 16;
    int base = -1;
    if (tok < t1) {
      const uint32_t b = a.bs.div(tok);
      const uint32_t blk = (uint32_t)a.tables[(int64_t)t.req * a.table_stride + b];
      if (blk < a.num_blocks)
        base = (int)((blk * (uint32_t)a.heads + hc) * (a.bs.d / 16) + (tok - b * a.bs.d) / 16);
    }
    s_base[i] = base;
  }
  fill_table<WAVES * 64>(a, hc, lds);

  int lim[NT], row[NT], head[NT];
  u32x4 qf[NT][KS];
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    const int col = t.col0 + 16 * x + n;
    const bool ok = col < ncols;
    const int i = (int)a.gdiv.div(ok ? col : 0);
    row[x] = t.row0 + i;
    head[x] = hc * a.G + (ok ? col - i * a.G : 0);
    lim[x] = ok ? sees(a, t, i) : 0;
    const uint16_t* qp = a.q + row[x] * a.q_ts + head[x] * a.q_hs + g * (D / 4);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qf[x][s] = ok ? *reinterpret_cast<const u32x4*>(qp + s * 8) : u32x4{0, 0, 0, 0};
    if (!ok) row[x] = -1;
  }
  __syncthreads();

  float m[NT], l[NT];
  f32x4 o[NT][ND];
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    m[x] = kLowest;
    l[x] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[x][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // fp16 weights are kept within the type's range whatever the scales are:
  // times 2^14 over a power of two that no scale so far exceeds.
  float vref = 0.f, vmul = 1.f;
  const uint32_t koff = (uint32_t)(lane & 31) * 4, voff = koff + 128;
  const int ntile = (t1 - t0 + 31) / 32;

  auto bases = [&](int it, int (&base)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      base[j] = __builtin_amdgcn_readfirstlane(s_base[min(it, ntile - 1) * 2 + j]);
  };
  int base[2], nbase[2];
  Codes<D> cur, nxt;
  if (wave < ntile) {
    bases(wave, base);
    load_codes<D>(a, base, n, g, cur);
  }
  for (int it = wave; it < ntile; it += WAVES) {
    bases(it + WAVES, nbase);
    load_codes<D>(a, nbase, n, g, nxt);

    f32x4 s[NT][2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        u32x4 kf;
#pragma unroll
        for (int b = 0; b < 4; ++b) kf[b] = lookup(cur.k[j][k], b, koff);
#pragma unroll
        for (int x = 0; x < NT; ++x)
          s[x][j] = mfma<DT>(kf, qf[x][k], k ? s[x][j] : f32x4{0.f, 0.f, 0.f, 0.f});
      }
    const int tok = t0 + it * 32 + 4 * g;  // token (j, i): tok + 16 j + i
    const bool masked = t0 + it * 32 + 32 > lim_min || (base[0] | base[1]) < 0;
    float ks[2][4], vs[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t kw = i < 2 ? cur.ks[j].x : cur.ks[j].y;
        const uint32_t vw = i < 2 ? cur.vs[j].x : cur.vs[j].y;
        ks[j][i] = from16<DT>((i & 1) ? kw >> 16 : kw & 0xffffu) * a.zscale;
        vs[j][i] = from16<DT>((i & 1) ? vw >> 16 : vw & 0xffffu);
        // What lies past the requests' tokens is anything.
        if (masked && (base[j] < 0 || tok + 16 * j + i >= lim_max)) vs[j][i] = 0.f;
      }
    if constexpr (DT == FKC_F16) {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(vs[j][i]) < INFINITY ? fabsf(vs[j][i]) : 0.f);
      if (__any(top > vref)) {
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        // next power of two: times 2^14 over it stays in range
        const float ref = __uint_as_float((__float_as_uint(top) + 0x7fffffu) & 0x7f800000u);
        const float mul = 16384.f / ref;
        const float f = vref > 0.f ? mul / vmul : 0.f;  // nothing yet: o is 0
        vref = ref;
        vmul = mul;
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int d = 0; d < ND; ++d) o[x][d] *= f;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[j][i] *= vmul;
    }
    u32x4 pf[NT];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      float z[2][4], top = kLowest;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          z[j][i] = s[x][j][i] * ks[j][i];
          if (masked && (base[j] < 0 || tok + 16 * j + i >= lim[x])) z[j][i] = -INFINITY;
          top = fmaxf(top, z[j][i]);
        }
      if (__any(top > m[x])) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float nm = fmaxf(m[x], top);
        const float f = __builtin_amdgcn_exp2f(m[x] - nm);
        m[x] = nm;
        l[x] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[x][d] *= f;
      }
      float w[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __builtin_amdgcn_exp2f(z[j][i] - m[x]);
          l[x] += p;
          w[j][i] = masked && z[j][i] == -INFINITY ? 0.f : p * vs[j][i];
        }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        pf[x][e] = pack2<DT>(w[e >> 1][2 * (e & 1)], w[e >> 1][2 * (e & 1) + 1]);
    }
#pragma unroll
    for (int b = 0; b < ND / 2; ++b) {
      uint32_t e[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) e[j][i] = lookup(cur.v[j][i][b / 4], b % 4, voff);
      u32x4 lo, hi;  // features 2 b and 2 b + 1 of the lane's row, by token
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t x0 = e[k >> 1][2 * (k & 1)], x1 = e[k >> 1][2 * (k & 1) + 1];
        lo[k] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
        hi[k] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        o[x][2 * b] = mfma<DT>(lo, pf[x], o[x][2 * b]);
        o[x][2 * b + 1] = mfma<DT>(hi, pf[x], o[x][2 * b + 1]);
      }
    }
    cur = nxt;
    base[0] = nbase[0];
    base[1] = nbase[1];
  }

  // Join the lanes of a column (they share m), then the waves, half of them
  // at a time, the later one into the earlier.
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    l[x] += __shfl_xor(l[x], 16, 64);
    l[x] += __shfl_xor(l[x], 32, 64);
    if constexpr (DT == FKC_F16)
#pragma unroll
      for (int d = 0; d < ND; ++d) o[x][d] *= 1.f / vmul;
  }
#pragma unroll
  for (int half = WAVES / 2; half > 0; half /= 2) {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      f32x4* so = reinterpret_cast<f32x4*>(lds);
      float* sml = reinterpret_cast<float*>(lds + kTable);
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int d = 0; d < ND; ++d) so[((wave - half) * ND + d) * 64 + lane] = o[x][d];
        if (g == 0) {
          sml[(wave - half) * 32 + n] = m[x];
          sml[(wave - half) * 32 + 16 + n] = l[x];
        }
      }
      __syncthreads();
      if (wave < half) {
        const float m2 = sml[wave * 32 + n], l2 = sml[wave * 32 + 16 + n];
        const float nm = fmaxf(m[x], m2);
        const float f1 = __builtin_amdgcn_exp2f(m[x] - nm);
        const float f2 = __builtin_amdgcn_exp2f(m2 - nm);
        m[x] = nm;
        l[x] = l[x] * f1 + l2 * f2;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[x][d] = o[x][d] * f1 + so[(wave * ND + d) * 64 + lane] * f2;
      }
    }
  }
  if (wave != 0) return;
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    if (row[x] < 0) continue;
    const int64_t at = (int64_t)row[x] * a.H + head[x];
    if (lim[x] <= a.chunk) {  // all of the row is here
      if (c != 0) continue;
      const float f = l[x] > 0.f ? 1.f / l[x] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[ND / 2];
#pragma unroll
        for (int d = 0; d < ND / 2; ++d)
          w[d] = pack2<DT>(o[x][2 * d][i] * f, o[x][2 * d + 1][i] * f);
        uint32_t* op = reinterpret_cast<uint32_t*>(a.out + at * D + (4 * g + i) * ND);
#pragma unroll
        for (int d = 0; d < ND / 2; ++d) op[d] = w[d];
      }
      if (g == 0 && a.lse != nullptr)
        a.lse[at] = l[x] > 0.f ? m[x] * kLn2 + __logf(l[x]) : -INFINITY;
    } else if (t0 < lim[x]) {
      float* op = a.part + (at * a.chunks + c) * D;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < ND; ++d) op[(4 * g + i) * ND + d] = o[x][d][i];
      if (g == 0) {
        a.part_ml[(at * a.chunks + c) * 2] = m[x];
        a.part_ml[(at * a.chunks + c) * 2 + 1] = l[x];
      }
    }
  }
}

// Joins the chunks of a row that needed more than one: a workgroup per query
// and head, D / 4 lanes per chunk.
template <int DT, int D>
__global__ void __launch_bounds__(256)
kv4_join_kernel(const Args a) {
  constexpr int LPC = D / 4, CP = 256 / LPC;
  __shared__ f32x4 so[256];
  __shared__ float sm[CP], sl[CP];
  const int64_t at = (int64_t)blockIdx.x * a.H + blockIdx.y;
  const int row = blockIdx.x;
  Tile t{row, 1, 0, 0, row};
  if (a.cu_q != nullptr) {
    int lo = 0, len = a.R + 1;
    while (len > 1) {
      const int half = len >> 1;
      if (a.cu_q[lo + half] <= row) lo += half;
      len -= half;
    }
    if (lo >= a.R) return;
    t.req = lo;
    t.row0 = a.cu_q[lo];
    t.nq = a.cu_q[lo + 1] - t.row0;
  }
  t.end = tokens_of(a, t.req);
  const int lim = sees(a, t, row - t.row0);
  if (lim <= a.chunk) return;
  const int nc = (lim + a.chunk - 1) / a.chunk;
  const int sub = threadIdx.x % LPC, part = threadIdx.x / LPC;
  const float* ml = a.part_ml + at * a.chunks * 2;
  float m = kLowest, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int c = part; c < nc; c += CP) {
    const float m2 = ml[2 * c], l2 = ml[2 * c + 1];
    const f32x4 x = *reinterpret_cast<const f32x4*>(a.part + (at * a.chunks + c) * D + 4 * sub);
    const float nm = fmaxf(m, m2);
    const float f1 = __builtin_amdgcn_exp2f(m - nm), f2 = __builtin_amdgcn_exp2f(m2 - nm);
    m = nm;
    l = l * f1 + l2 * f2;
    o = o * f1 + x * f2;
  }
  so[threadIdx.x] = o;
  if (sub == 0) {
    sm[part] = m;
    sl[part] = l;
  }
  __syncthreads();
  if (threadIdx.x >= LPC) return;
#pragma unroll
  for (int c = 1; c < CP; ++c) {
    const float nm = fmaxf(m, sm[c]);
    const float f1 = __builtin_amdgcn_exp2f(m - nm), f2 = __builtin_amdgcn_exp2f(sm[c] - nm);
    m = nm;
    l = l * f1 + sl[c] * f2;
    o = o * f1 + so[c * LPC + sub] * f2;
  }
  const float f = l > 0.f ? 1.f / l : 0.f;
  uint2 w;
  w.x = pack2<DT>(o[0] * f, o[1] * f);
  w.y = pack2<DT>(o[2] * f, o[3] * f);
  *reinterpret_cast<uint2*>(a.out + at * D + 4 * sub) = w;
  if (sub == 0 && a.lse != nullptr)
    a.lse[at] = l > 0.f ? m * kLn2 + __logf(l) : -INFINITY;
}

template <typename F>
int by_shape(int dtype, int64_t D, F&& f) {
  auto with = [&](auto dt) {
    if (D == 64) return f(dt, std::integral_constant<int, 64>{});
    if (D == 128) return f(dt, std::integral_constant<int, 128>{});
    return f(dt, std::integral_constant<int, 256>{});
  };
  return dtype == FKC_F16 ? with(std::integral_constant<int, FKC_F16>{})
                          : with(std::integral_constant<int, FKC_BF16>{});
}

struct Plan {
  int nt;           // column tiles per workgroup
  int chunk;        // tokens per workgroup
  int chunks;
  int tiles_per_req;  // without cu_q
  int64_t tiles;      // of nt * 16 columns, over all requests (an upper bound)
};

Plan make_plan(const fkc_kv4_cache& c, int64_t H, int64_t T, int64_t R, int64_t max_seq,
               bool ragged) {
  Plan p;
  const int64_t G = H / c.heads;
  // Column tiles: as many as an average request fills, up to two.
  p.nt = R > 0 && T * G > 16 * R ? 2 : 1;
  const int64_t cols = 16 * p.nt;
  p.tiles_per_req = (int)((G + cols - 1) / cols);
  p.tiles = ragged ? T * G / cols + R + 1 : R * p.tiles_per_req;
  // Chunks: about four workgroups for each of the two places per CU.
  const int64_t want = 8 * (int64_t)device_shape().cus;
  const int64_t s = std::max<int64_t>(1, want / std::max<int64_t>(1, R * c.heads));
  int64_t chunk = (max_seq + s - 1) / s;
  chunk = std::min<int64_t>(std::max<int64_t>(chunk, 1024), 4096);
  p.chunk = (int)((chunk + 255) / 256 * 256);
  p.chunks = (int)std::max<int64_t>(1, (max_seq + p.chunk - 1) / p.chunk);
  return p;
}

template <int DT, int D, int NT, int WAVES>
int launch_split(const Args& a, const Plan& p, hipStream_t s) {
  const int bytes = kTable + std::max(WAVES / 2 * 32 * 4, p.chunk / 16 * 4);
  auto* kernel = &kv4_split_kernel<DT, D, NT, WAVES>;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return fail(FKC_ERR_LAUNCH, "kv4_attend: %d bytes of LDS refused", bytes);
  hipLaunchKernelGGL((kv4_split_kernel<DT, D, NT, WAVES>),
                     dim3((uint32_t)(p.tiles * a.heads * p.chunks)), dim3(WAVES * 64), bytes, s,
                     a);
  if (int rc = check_launch("kv4_attend")) return rc;
  if (p.chunks == 1) return FKC_OK;
  hipLaunchKernelGGL((kv4_join_kernel<DT, D>), dim3((uint32_t)a.T, (uint32_t)a.H), dim3(256), 0,
                     s, a);
  return check_launch("kv4_attend (join)");
}

}  // namespace

size_t kv4_attend_workspace_bytes(const fkc_kv4_cache& c, int64_t H, int64_t T, int64_t R,
                                  int64_t max_seq) {
  const Plan p = make_plan(c, H, T, R, max_seq, true);
  if (p.chunks == 1) return 0;
  Carve w(nullptr);
  w.take<float>((size_t)T * H * p.chunks * c.D);
  w.take<float>((size_t)T * H * p.chunks * 2);
  return w.used;
}

int launch_kv4_attend(const fkc_kv4_cache& c, const Kv4Attend& x, void* ws, size_t,
                      hipStream_t s) {
  const Plan p = make_plan(c, x.H, x.T, x.R, x.max_seq, x.cu_q != nullptr);
  if (p.tiles * c.heads > INT32_MAX / p.chunks)
    return fail(FKC_ERR_UNSUPPORTED, "kv4_attend: too many rows times chunks");
  const int G = (int)(x.H / c.heads);
  Args a{(const uint16_t*)x.q.p, x.q.token_stride, x.q.head_stride,
         (const uint8_t*)c.k_codes, (const uint8_t*)c.v_codes,
         (const uint16_t*)c.k_scales, (const uint16_t*)c.v_scales,
         (const uint16_t*)c.k_levels, (const uint16_t*)c.v_levels,
         x.tables, x.table_stride, x.seq, x.cu_q, (uint16_t*)x.out, x.lse, nullptr, nullptr,
         FastDiv((uint32_t)c.block_size), FastDiv((uint32_t)G), (uint32_t)c.num_blocks,
         (int)c.heads, (int)x.H, G, (int)x.T, (int)x.R, (int)x.max_seq, (int)x.causal,
         p.chunk, p.chunks, p.tiles_per_req, x.sm_scale * kLog2e};
  if (p.chunks > 1) {
    Carve w(ws);
    a.part = w.take<float>((size_t)x.T * x.H * p.chunks * c.D);
    a.part_ml = w.take<float>((size_t)x.T * x.H * p.chunks * 2);
  }
  return by_shape(c.dtype, c.D, [&](auto dt, auto d) {
    constexpr int DT = dt.value, DD = d.value;
    return p.nt == 1 ? launch_split<DT, DD, 1, DD == 256 ? 4 : 8>(a, p, s)
                     : launch_split<DT, DD, 2, 4>(a, p, s);
  });
}

}  // namespace fkc
