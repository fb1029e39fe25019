// Storing vectors in the 4-bit cache and reading them back.
//
// A vector x of one head is held as s = max |x_d| and, per element, the code of
// the level nearest to y_d = x_d * (1 / s): the assignment of the Lloyd loop
// with K = 16 and D = 1, in the same arithmetic whatever the path below (fp32
// quotient, fp32 distances, lowest index of equal ones).
//
// Bound by memory: 2 D bytes in and D / 2 + 2 out per vector, so the search
// has to cost less than the ~25 vector-ALU operations per element that the
// time of those bytes has room for.  Sixteen distances, compares and selects
// are 64, halving the sorted levels' 15 thresholds 33; one look into a table of
// y's CELLS cells, each with the one threshold that falls into it, is 10.
// Measured: 32768 tokens of 16 heads of 64 columns, bf16, keys and values, 48.7 us
// (170 MB, 3.5 TB/s; with sixteen distances 366 us) and reading them back 36.1
// (4.7 TB/s); 8191 tokens of 8 heads of 128, fp16, 14.5 and 10.7; 64 tokens 5.8
// and 3.6, of which the table's making (loads, sorting, a search) is about 3.
#include <algorithm>
#include <type_traits>

#include "device_util.hpp"
#include "fkc_internal.hpp"

namespace fkc {
namespace {

constexpr int LV = 16;           // levels per head
constexpr int KT = 512;          // threads per workgroup
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126

// Order-preserving map of finite floats to integers and back.
__device__ inline uint32_t float_key(float f) {
  const uint32_t b = __float_as_uint(f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ inline float key_float(uint32_t k) {
  return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}

// Cells of y, rising with y, as the byte offset of their entry: in the sum with
// 2^20 the last bit counts eighths of a cell.  Any y has one (NaN the first);
// quotients by the largest magnitude (|y| <= 1 + 2^-23) have their own.
constexpr int CELLS = 1024;
__device__ inline uint32_t cell_of(float y) {
  const float f = __builtin_fmaf(y, CELLS / 2 - 0.25f, 0x1p20f + CELLS / 2);
  return __float_as_uint(f) & (CELLS - 1) * 8u;
}
__device__ inline uint32_t cell_of_any(float y) { return cell_of(fminf(fmaxf(y, -1.f), 1.f)); }

// Fills the table of a head's levels, by the whole workgroup: cell c holds a
// threshold and the codes below it (4 bits) and from it on (the next 4).
// Returns whether the table describes the choice; if not, every level has to
// be compared.
//
// Between neighbours a < b the distances y - a and b - y, rounded, rise and
// fall with y, so the choice "b before a" (nearer, or as near with the lower
// index) turns once, at an exact fp32 threshold within a rounding of a distance
// of the middle; the four 16-lane rows of the first wave look for it, four
// places a round, lane j of a row for the one above the j-th smallest level.
// Farther levels cannot interfere while neighbours are so far apart that no
// rounded distance can make two of them equal: 2^-20 of the largest distance.
// Levels closer than that, not finite, or with two thresholds in one cell are
// left to the plain comparison; equal ones count as the one of lowest index.
struct Cells {
  uint2 at[CELLS];
  uint32_t cell[LV], code[LV];  // of threshold j; of the j-th smallest level
  int bad;
};

template <int DT>
__device__ inline bool fill_cells(const typename Elem<DT>::T* lv, Cells& t) {
#pragma clang fp contract(off)
  float thr = INFINITY;
  uint32_t cell = CELLS * 8, codes = 0;
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x, i = lane & 15;
    const float mine = Elem<DT>::load(lv[i]);
    int rank = 0, same = i;
#pragma unroll
    for (int c = LV - 1; c >= 0; --c) {
      const float other = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), c));
      const bool eq = other == mine;
      rank += other < mine || (eq && c < i);
      same = eq ? c : same;  // ends with the lowest
    }
    // (NaN, which ranks below nothing, sends several lanes to one place: bad.)
    const int to = ((lane & 48) | rank) * 4;
    const float a = __int_as_float(__builtin_amdgcn_ds_permute(to, __float_as_int(mine)));
    const int idx = __builtin_amdgcn_ds_permute(to, same);
    const int next = min(lane + 1, 63) * 4;
    const float b = __int_as_float(__builtin_amdgcn_ds_bpermute(next, __float_as_int(a)));
    const int idx_b = __builtin_amdgcn_ds_bpermute(next, idx);
    const float far =
        1.f + fmaxf(fabsf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), 0))),
                    fabsf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), LV - 1))));
    const bool pair = i + 1 < LV && b != a;  // this lane has a threshold to find
    bool bad = __any(!(fabsf(mine) < INFINITY) || (pair && !(b - a >= far * 0x1p-20f)));
    const float mid = 0.5f * a + 0.5f * b;
    const float e = (b - a) * 0x1p-22f + fabsf(mid) * 0x1p-22f;
    uint32_t lo = pair && !bad ? float_key(fmaxf(a, mid - e)) : 0;  // takes a
    uint32_t hi = pair && !bad ? float_key(fminf(b, mid + e)) : 1;  // takes b
    while (__any(hi - lo > 1)) {  // at most a fifth and four are left each round
      const uint32_t step = max((hi - lo) / 5, 1u);
      const float y = key_float(min(lo + step * (lane / 16 + 1), hi));
      const float da = y - a, db = b - y;
      const uint64_t m = __ballot(db < da || (db == da && idx_b < idx)) >> i;
      const uint32_t first =
          (m & 1) ? 0 : (m >> 16 & 1) ? 1 : (m >> 32 & 1) ? 2 : (m >> 48 & 1) ? 3 : 4;
      if (hi - lo > 1) {
        if (first < 4) hi = min(lo + step * (first + 1), hi);
        lo += step * first;
      }
    }
    if (pair && !bad) {
      thr = key_float(hi);
      cell = cell_of_any(thr);
    }
    codes = (uint32_t)idx | (uint32_t)idx_b << 4;
    uint32_t prev = CELLS * 8;
#pragma unroll
    for (int j = 0; j < LV - 1; ++j) {
      const uint32_t at = __builtin_amdgcn_readlane((int)cell, j);
      bad |= at < CELLS * 8 && at == prev;
      prev = at < CELLS * 8 ? at : prev;
    }
    if (lane < LV) {
      t.cell[lane] = cell / 8;
      t.code[lane] = (uint32_t)idx;
    }
    if (lane == 0) t.bad = bad;
  }
  __syncthreads();
  if (t.bad) return false;
  // Codes below the cells' thresholds: those from the last threshold of the
  // cells before on.
  uint32_t code[CELLS / KT];
#pragma unroll
  for (int c = 0; c < CELLS / KT; ++c) code[c] = t.code[0];
#pragma unroll
  for (int j = 0; j < LV - 1; ++j) {
    const uint32_t at = t.cell[j], id = t.code[j + 1];
#pragma unroll
    for (int c = 0; c < CELLS / KT; ++c)
      code[c] = at < threadIdx.x + c * KT ? id : code[c];
  }
#pragma unroll
  for (int c = 0; c < CELLS / KT; ++c)
    t.at[threadIdx.x + c * KT] = uint2{__float_as_uint(INFINITY), code[c]};
  __syncthreads();
  if (threadIdx.x < LV && cell < CELLS * 8)
    t.at[cell / 8] = uint2{__float_as_uint(thr), codes};
  __syncthreads();
  return true;
}

// NB passes of a workgroup over the rows of one head, D / 8 lanes per vector.
template <int D, int NB>
struct Batch {
  static constexpr int LPV = D / 8, VP = KT / LPV;
  uint4 x[NB];
  uint32_t slot[NB];
  __device__ inline void load(const uint16_t* base, int64_t token_stride,
                              const int32_t* slots, int tb, int t1, uint32_t num_slots) {
    const int first = tb + threadIdx.x / LPV;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int tok = first + i * VP;
      slot[i] = tok < t1 ? (uint32_t)slots[tok] : 0xffffffffu;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)  // a token that is not stored is not read either
      x[i] = slot[i] < num_slots ? *reinterpret_cast<const uint4*>(
                                       base + (int64_t)(first + i * VP) * token_stride)
                                 : uint4{0, 0, 0, 0};
  }
};

// The largest of v over the LPV lanes of a vector.
template <int LPV>
__device__ inline uint32_t vector_max(uint32_t v) {
#define FKC_DPP_MAX(CTRL) \
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true))
  FKC_DPP_MAX(0xB1);   // quad_perm [1,0,3,2]
  FKC_DPP_MAX(0x4E);   // quad_perm [2,3,0,1]
  FKC_DPP_MAX(0x141);  // row_half_mirror: 8 lanes
  if (LPV > 8) FKC_DPP_MAX(0x140);  // row_mirror: 16 lanes
#undef FKC_DPP_MAX
  if (LPV > 16) v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  return v;
}

template <int DT, int D, bool PLAIN, int NB>
__device__ inline void store_batch(const Batch<D, NB>& in, const Cells& t,
                                   const typename Elem<DT>::T* levels, uint32_t* codes,
                                   uint16_t* scales, int heads, int h, FastDiv bs,
                                   uint32_t num_slots) {
#pragma clang fp contract(off)
  using E = Elem<DT>;
  using T16 = typename E::T;
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  constexpr int LPV = D / 8;
  const int sub = threadIdx.x % LPV;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const uint32_t w[4] = {in.x[i].x, in.x[i].y, in.x[i].z, in.x[i].w};
    // Magnitudes of 16-bit floats order as their bits do, NaN on top.
    u16x2 two = {0, 0};
#pragma unroll
    for (int d = 0; d < 4; ++d)
      two = __builtin_elementwise_max(two, __builtin_bit_cast(u16x2, w[d] & 0x7fff7fffu));
    uint32_t top = vector_max<LPV>(max((uint32_t)two[0], (uint32_t)two[1]));
    float s = E::load(__builtin_bit_cast(T16, (uint16_t)top));
    if (s < kMinScale) {
      s = 0.f;
      top = 0;
    }
    const float inv = s > 0.f ? 1.f / s : 0.f;
    float y[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const uint16_t bits = (uint16_t)(w[d / 2] >> (16 * (d & 1)));
      y[d] = E::load(__builtin_bit_cast(T16, bits)) * inv;
    }
    uint32_t word = 0;
    if constexpr (PLAIN) {
      float best[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) best[d] = fabsf(y[d] - E::load(levels[0]));
#pragma unroll 1
      for (int c = 1; c < LV; ++c) {
        const float lv = E::load(levels[c]);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const float dist = fabsf(y[d] - lv);
          if (dist < best[d]) {
            best[d] = dist;
            word = (word & ~(15u << (4 * d))) | (uint32_t)c << (4 * d);
          }
        }
      }
    } else {
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const uint2 e = *reinterpret_cast<const uint2*>(
            reinterpret_cast<const char*>(t.at) + cell_of(y[d]));
        // the low four bits, on top of the word shifted down by four
        word = __builtin_amdgcn_alignbit(e.y >> (y[d] >= __uint_as_float(e.x) ? 4 : 0), word, 4);
      }
      // An element over an infinity or a NaN that is neither 0 takes level 0.
      if (__any(!(s < INFINITY))) {
#pragma unroll
        for (int d = 0; d < 8; ++d)
          if (y[d] != y[d]) word &= ~(15u << (4 * d));
      }
    }
    if (in.slot[i] < num_slots) {
      const uint32_t blk = bs.div(in.slot[i]);
      const int64_t row = ((int64_t)blk * heads + h) * bs.d + (in.slot[i] - blk * bs.d);
      codes[row * LPV + sub] = word;
      if (sub == 0) scales[row] = (uint16_t)top;
    }
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(KT, 8)
kv4_append_kernel(Kv4Rows kr, Kv4Rows vr, const int32_t* __restrict__ slots,
                  int T, int per_wg, uint32_t* __restrict__ k_codes,
                  uint32_t* __restrict__ v_codes, uint16_t* __restrict__ k_scales,
                  uint16_t* __restrict__ v_scales, const uint16_t* __restrict__ k_levels,
                  const uint16_t* __restrict__ v_levels, int heads, FastDiv bs,
                  uint32_t num_slots) {
  using T16 = typename Elem<DT>::T;
  constexpr int NB = 2;
  using B = Batch<D, NB>;
  __shared__ Cells t;
  const int h = blockIdx.y;
  const bool isv = blockIdx.z != 0;
  const Kv4Rows src = isv ? vr : kr;
  const T16* levels = reinterpret_cast<const T16*>(isv ? v_levels : k_levels) + h * LV;
  uint32_t* codes = isv ? v_codes : k_codes;
  uint16_t* scales = isv ? v_scales : k_scales;
  const uint16_t* base = static_cast<const uint16_t*>(src.p) + (int64_t)h * src.head_stride +
                         threadIdx.x % B::LPV * 8;
  const int t0 = blockIdx.x * per_wg;
  const int t1 = min(T, t0 + per_wg);
  // Rows are on their way while the table is made.
  B cur, nxt;
  cur.load(base, src.token_stride, slots, t0, t1, num_slots);
  const bool table = fill_cells<DT>(levels, t);
  for (int tb = t0; tb < t1; tb += NB * B::VP) {
    nxt.load(base, src.token_stride, slots, tb + NB * B::VP, t1, num_slots);
    if (table)
      store_batch<DT, D, false>(cur, t, levels, codes, scales, heads, h, bs, num_slots);
    else
      store_batch<DT, D, true>(cur, t, levels, codes, scales, heads, h, bs, num_slots);
    cur = nxt;
  }
}

// The reverse: eight elements per lane, levels in LDS once per bank so that
// 32 lanes of any codes read 32 banks.
template <int DT, int D>
__global__ void __launch_bounds__(KT)
kv4_read_kernel(const int32_t* __restrict__ slots, int T, int per_wg,
                const uint32_t* __restrict__ k_codes, const uint32_t* __restrict__ v_codes,
                const uint16_t* __restrict__ k_scales, const uint16_t* __restrict__ v_scales,
                const uint16_t* __restrict__ k_levels, const uint16_t* __restrict__ v_levels,
                int heads, FastDiv bs, uint32_t num_slots, uint16_t* __restrict__ k_out,
                uint16_t* __restrict__ v_out) {
  using E = Elem<DT>;
  using T16 = typename E::T;
  constexpr int LPV = D / 8, VP = KT / LPV, NB = 4;
  __shared__ float lv[LV * 32];
  const int h = blockIdx.y;
  const bool isv = blockIdx.z != 0;
  uint16_t* out = isv ? v_out : k_out;
  if (out == nullptr) return;
  const uint32_t* codes = isv ? v_codes : k_codes;
  const uint16_t* scales = isv ? v_scales : k_scales;
  const T16* levels = reinterpret_cast<const T16*>(isv ? v_levels : k_levels) + h * LV;
  for (int i = threadIdx.x; i < LV * 32; i += KT) lv[i] = E::load(levels[i / 32]);
  __syncthreads();
  const int sub = threadIdx.x % LPV, vec = threadIdx.x / LPV, bank = threadIdx.x & 31;
  const int t0 = blockIdx.x * per_wg;
  const int t1 = min(T, t0 + per_wg);
  for (int tb = t0; tb < t1; tb += NB * VP) {
    uint32_t word[NB], sc[NB];
    bool held[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int tok = tb + i * VP + vec;
      const uint32_t slot = tok < t1 ? (uint32_t)slots[tok] : 0xffffffffu;
      held[i] = slot < num_slots;
      const uint32_t blk = held[i] ? bs.div(slot) : 0;
      const int64_t row = ((int64_t)blk * heads + h) * bs.d + (slot - blk * bs.d);
      word[i] = held[i] ? codes[row * LPV + sub] : 0;
      sc[i] = held[i] ? scales[row] : 0;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int tok = tb + i * VP + vec;
      if (tok >= t1) continue;
      const float s = E::load(__builtin_bit_cast(T16, (uint16_t)sc[i]));
      uint32_t o[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const float a = s * lv[((word[i] >> (8 * d)) & 15u) * 32 + bank];
        const float b = s * lv[((word[i] >> (8 * d + 4)) & 15u) * 32 + bank];
        o[d] = (uint32_t)__builtin_bit_cast(uint16_t, E::store(a)) |
               (uint32_t)__builtin_bit_cast(uint16_t, E::store(b)) << 16;
      }
      if (!held[i]) o[0] = o[1] = o[2] = o[3] = 0;
      *reinterpret_cast<uint4*>(out + ((int64_t)tok * heads + h) * D + sub * 8) =
          uint4{o[0], o[1], o[2], o[3]};
    }
  }
}

// Tokens per workgroup: about four workgroups (all that fit) per CU over all
// heads, keys and values, in whole passes; at most 2^20, so that an int holds it
// for any T.
int tokens_per_wg(int64_t T, int64_t heads, int D) {
  const int64_t vp = KT / (D / 8);
  const int64_t passes = (T + vp - 1) / vp * heads * 2;
  const int64_t want = 4 * (int64_t)device_shape().cus;
  return (int)std::min<int64_t>(vp * std::max<int64_t>(1, (passes + want - 1) / want), 1 << 20);
}

}  // namespace

int launch_kv4_append(const fkc_kv4_cache& c, Kv4Rows k, Kv4Rows v,
                      const int32_t* slots, int64_t T, hipStream_t s) {
  if (c.num_blocks == 0) return FKC_OK;  // no slot is inside
  return kv4_by_shape(c.dtype, c.D, [&](auto dt, auto d) {
    const int per = tokens_per_wg(T, c.heads, d.value);
    const dim3 grid((uint32_t)((T + per - 1) / per), (uint32_t)c.heads, 2);
    hipLaunchKernelGGL((kv4_append_kernel<dt.value, d.value>), grid, dim3(KT), 0, s, k, v,
                       slots, (int)T, per, (uint32_t*)c.k_codes, (uint32_t*)c.v_codes,
                       (uint16_t*)c.k_scales, (uint16_t*)c.v_scales,
                       (const uint16_t*)c.k_levels, (const uint16_t*)c.v_levels,
                       (int)c.heads, FastDiv((uint32_t)c.block_size),
                       (uint32_t)(c.num_blocks * c.block_size));
    return check_launch("kv4_append");
  });
}

int launch_kv4_read(const fkc_kv4_cache& c, const int32_t* slots, int64_t T,
                    void* k_out, void* v_out, hipStream_t s) {
  return kv4_by_shape(c.dtype, c.D, [&](auto dt, auto d) {
    const int per = tokens_per_wg(T, c.heads, d.value);
    const dim3 grid((uint32_t)((T + per - 1) / per), (uint32_t)c.heads, 2);
    hipLaunchKernelGGL((kv4_read_kernel<dt.value, d.value>), grid, dim3(KT), 0, s, slots,
                       (int)T, per, (const uint32_t*)c.k_codes, (const uint32_t*)c.v_codes,
                       (const uint16_t*)c.k_scales, (const uint16_t*)c.v_scales,
                       (const uint16_t*)c.k_levels, (const uint16_t*)c.v_levels,
                       (int)c.heads, FastDiv((uint32_t)c.block_size),
                       (uint32_t)(c.num_blocks * c.block_size), (uint16_t*)k_out,
                       (uint16_t*)v_out);
    return check_launch("kv4_read");
  });
}

}  // namespace fkc
