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
// are 64; the sorted levels' thresholds halved four times are 23.
#include <algorithm>
#include <type_traits>

#include "device_util.hpp"
#include "fkc_internal.hpp"

namespace fkc {
namespace {

constexpr int LV = 16;           // levels per head
constexpr int KT = 256;          // threads per workgroup
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126

// Levels of one head, ready for the search.
struct Levels {
  float raw[LV];    // as stored
  float uniq[LV];   // ascending, without repeats
  int order[LV];    // index of uniq[j]: the lowest of equal levels
  int dup[LV];      // raw[i] repeats a level of lower index
  float thr[LV];    // smallest y that takes uniq[j + 1] before uniq[j]
  int n;            // distinct levels
  int plain;        // thresholds do not describe the search: compare them all
};

// Order-preserving map of finite floats to integers and back (+0 and -0
// apart, which compare equal: no threshold is between them).
__device__ inline int64_t float_key(float f) {
  const int32_t b = __float_as_int(f);
  return b < 0 ? -(int64_t)(b & 0x7fffffff) - 1 : (int64_t)b;
}
__device__ inline float key_float(int64_t k) {
  return k < 0 ? __int_as_float((int32_t)(-(k + 1)) | (int32_t)0x80000000)
               : __int_as_float((int32_t)k);
}

// Thresholds of the levels, by the whole workgroup.  Between neighbours a < b
// the distances y - a and b - y, rounded, rise and fall with y, so the choice
// "b before a" (nearer, or as near with the lower index) turns once, at an
// exact fp32 y within a few roundings of the middle; 16 lanes look for it,
// each round 16 places at once.  Farther levels cannot interfere while
// neighbours are so far apart that no rounded distance (|y| <= 1 + 2^-23) can
// make two of them equal: 2^-20 of the largest distance; levels closer than
// that, or not finite, are compared one by one instead.
template <int DT>
__device__ void prepare_levels(Levels& L, const typename Elem<DT>::T* lv) {
#pragma clang fp contract(off)
  const int t = threadIdx.x;
  if (t < LV) L.raw[t] = Elem<DT>::load(lv[t]);
  if (t == 0) L.plain = 0;
  __syncthreads();
  if (t < LV) {
    int dup = 0;
    for (int i = 0; i < t; ++i) dup |= L.raw[i] == L.raw[t];
    L.dup[t] = dup;
    L.thr[t] = INFINITY;
    L.uniq[t] = 0.f;
    L.order[t] = 0;
  }
  __syncthreads();
  if (t < LV && !L.dup[t]) {
    int rank = 0;
    for (int i = 0; i < LV; ++i) rank += !L.dup[i] && L.raw[i] < L.raw[t];
    L.uniq[rank] = L.raw[t];
    L.order[rank] = t;
  }
  if (t == 0) {
    int n = 0;
    for (int i = 0; i < LV; ++i) n += !L.dup[i];
    L.n = n;
  }
  __syncthreads();
  const int n = L.n;
  if (t < LV) {
    const float far = 1.f + fmaxf(fabsf(L.uniq[0]), fabsf(L.uniq[n - 1]));
    const bool ok = t + 1 < n ? L.uniq[t + 1] - L.uniq[t] >= far * 0x1p-20f
                              : fabsf(L.raw[t]) < INFINITY;
    if (!ok || !(fabsf(L.raw[t]) < INFINITY)) L.plain = 1;  // every writer stores 1
  }
  __syncthreads();
  const int j = t / 16, lane = t & 15;
  if (!L.plain && j + 1 < n) {
    const float a = L.uniq[j], b = L.uniq[j + 1];
    const bool lower = L.order[j + 1] < L.order[j];
    const float mid = 0.5f * a + 0.5f * b;
    const float e = (b - a) * 0x1p-20f + fabsf(mid) * 0x1p-22f;
    int64_t lo = float_key(fmaxf(a, mid - e)), hi = float_key(fminf(b, mid + e));
    // lo takes a, hi takes b; at most 9 rounds from the widest interval.
    while (hi - lo > 1) {
      const int64_t at = lo + (hi - lo) * (lane + 1) / 17;
      const float y = key_float(at);
      const float da = y - a, db = b - y;
      const bool takes_b = db < da || (db == da && lower);
      const uint64_t m = __ballot(takes_b) >> (threadIdx.x & 48);
      const int first = __builtin_ctz((uint32_t)m & 0xffffu | 0x10000u);
      const int64_t w = hi - lo;
      hi = first < 16 ? lo + w * (first + 1) / 17 : hi;
      lo = first > 0 ? lo + w * first / 17 : lo;
    }
    if (lane == 0) L.thr[j] = key_float(hi);
  }
  __syncthreads();
}

// The rows of one head that a workgroup stores: D / 8 lanes per vector.
template <int DT, int D>
__global__ void __launch_bounds__(KT)
kv4_append_kernel(Kv4Rows kr, Kv4Rows vr, const int32_t* __restrict__ slots,
                  int T, int per_wg, uint32_t* __restrict__ k_codes,
                  uint32_t* __restrict__ v_codes, uint16_t* __restrict__ k_scales,
                  uint16_t* __restrict__ v_scales, const uint16_t* __restrict__ k_levels,
                  const uint16_t* __restrict__ v_levels, int heads, FastDiv bs,
                  uint32_t num_slots) {
#pragma clang fp contract(off)
  using E = Elem<DT>;
  using T16 = typename E::T;
  constexpr int LPV = D / 8;        // lanes per vector, 8 elements each
  constexpr int VP = KT / LPV;      // vectors per pass of the workgroup
  constexpr int NB = 4;             // passes in flight
  __shared__ Levels L;
  const int h = blockIdx.y;
  const bool isv = blockIdx.z != 0;
  const Kv4Rows src = isv ? vr : kr;
  uint32_t* codes = isv ? v_codes : k_codes;
  uint16_t* scales = isv ? v_scales : k_scales;
  prepare_levels<DT>(L, reinterpret_cast<const T16*>(isv ? v_levels : k_levels) + h * LV);
  float thr[LV - 1];
#pragma unroll
  for (int i = 0; i < LV - 1; ++i) thr[i] = L.thr[i];
  uint64_t order = 0;
  for (int i = 0; i < LV; ++i) order |= (uint64_t)L.order[i] << (4 * i);
  const bool plain = L.plain != 0;

  const int sub = threadIdx.x % LPV, vec = threadIdx.x / LPV;
  const uint16_t* base = static_cast<const uint16_t*>(src.p) +
                         (int64_t)h * src.head_stride + sub * 8;
  const int t0 = blockIdx.x * per_wg;
  const int t1 = min(T, t0 + per_wg);
  for (int tb = t0; tb < t1; tb += NB * VP) {
    uint4 x[NB];
    uint32_t slot[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int tok = tb + i * VP + vec;
      slot[i] = tok < t1 ? (uint32_t)slots[tok] : 0xffffffffu;
      // a token that is not stored is not read either
      x[i] = slot[i] < num_slots
                 ? *reinterpret_cast<const uint4*>(base + (int64_t)tok * src.token_stride)
                 : uint4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      // Magnitudes of 16-bit floats order as their bits do, NaN on top.
      uint32_t top = 0;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        top = max(top, max(w[d] & 0x7fffu, (w[d] >> 16) & 0x7fffu));
#pragma unroll
      for (int off = 1; off < LPV; off <<= 1)
        top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
      float s = E::load(__builtin_bit_cast(T16, (uint16_t)top));
      if (s < kMinScale) {
        s = 0.f;
        top = 0;
      }
      const float inv = s > 0.f ? 1.f / s : 0.f;
      const bool finite = s < INFINITY;
      uint32_t word = 0;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const uint16_t bits = (uint16_t)(w[d / 2] >> (16 * (d & 1)));
        const float y = E::load(__builtin_bit_cast(T16, bits)) * inv;
        uint32_t code;
        if (!plain && finite) {
          // Thresholds below y: halve 15, 7, 3, 1 of them.
          float u[7], v[3];
          const bool c3 = y >= thr[7];
#pragma unroll
          for (int q = 0; q < 7; ++q) u[q] = c3 ? thr[8 + q] : thr[q];
          const bool c2 = y >= u[3];
#pragma unroll
          for (int q = 0; q < 3; ++q) v[q] = c2 ? u[4 + q] : u[q];
          const bool c1 = y >= v[1];
          const bool c0 = y >= (c1 ? v[2] : v[0]);
          const uint32_t rank = (c3 ? 8 : 0) + (c2 ? 4 : 0) + (c1 ? 2 : 0) + (c0 ? 1 : 0);
          code = (uint32_t)(order >> (4 * rank)) & 15u;
        } else {
          code = 0;
          float best = fabsf(y - L.raw[0]);
          for (int c = 1; c < LV; ++c) {
            const float dist = fabsf(y - L.raw[c]);
            if (dist < best) {
              best = dist;
              code = c;
            }
          }
        }
        word |= code << (4 * d);
      }
      if (slot[i] < num_slots) {
        const uint32_t blk = bs.div(slot[i]);
        const int64_t row = ((int64_t)blk * heads + h) * bs.d + (slot[i] - blk * bs.d);
        codes[row * LPV + sub] = word;
        if (sub == 0) scales[row] = (uint16_t)top;
      }
    }
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

// Tokens per workgroup: about eight workgroups per CU over all heads, keys
// and values, in whole passes.
int tokens_per_wg(int64_t T, int64_t heads, int D) {
  const int64_t vp = KT / (D / 8);
  const int64_t passes = (T + vp - 1) / vp * heads * 2;
  const int64_t want = 8 * (int64_t)device_shape().cus;
  return (int)(vp * std::max<int64_t>(1, (passes + want - 1) / want));
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

}  // namespace

int launch_kv4_append(const fkc_kv4_cache& c, Kv4Rows k, Kv4Rows v,
                      const int32_t* slots, int64_t T, hipStream_t s) {
  if (c.num_blocks == 0) return FKC_OK;  // no slot is inside
  return by_shape(c.dtype, c.D, [&](auto dt, auto d) {
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
  return by_shape(c.dtype, c.D, [&](auto dt, auto d) {
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
