// Attention over the 4-bit cache, the plain way: one workgroup per query and
// head, one thread per token of a 256-token tile for the scores, one thread
// per column for the weighted sum, with a running maximum and sum.
#include <type_traits>

#include "device_util.hpp"
#include "fkc_internal.hpp"

namespace fkc {
namespace {

constexpr int AT = 256;

template <int DT, int D>
__global__ void __launch_bounds__(AT)
kv4_attend_kernel(const uint16_t* __restrict__ q, int64_t q_ts, int64_t q_hs, int H,
                  const int32_t* __restrict__ tables, int64_t table_stride,
                  const int32_t* __restrict__ seq, const int32_t* __restrict__ cu_q,
                  int R, int max_seq, int causal, float sm_scale,
                  const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ v_codes,
                  const uint16_t* __restrict__ k_scales, const uint16_t* __restrict__ v_scales,
                  const uint16_t* __restrict__ k_levels, const uint16_t* __restrict__ v_levels,
                  int heads, uint32_t num_blocks, FastDiv bs, uint16_t* __restrict__ out,
                  float* __restrict__ lse, int T) {
  using E = Elem<DT>;
  using T16 = typename E::T;
  __shared__ float qs[D], kl[16], vl[16], p[AT], part[AT];
  __shared__ int64_t rows[AT];
  __shared__ float red[AT / 64];
  const int t = threadIdx.x, row = blockIdx.x, h = blockIdx.y, hc = h / (H / heads);
  int r = row, i = 0, nq = 1;
  if (cu_q != nullptr) {
    int lo = 0, len = R + 1;  // last r with cu_q[r] <= row
    while (len > 1) {
      const int half = len >> 1;
      if (cu_q[lo + half] <= row) lo += half;
      len -= half;
    }
    r = lo;
    if (r < R) {
      i = row - cu_q[r];
      nq = cu_q[r + 1] - cu_q[r];
    }
  }
  int end = r < R ? min(max(seq[r], 0), max_seq) : 0;
  if (causal) end = max(0, end - nq + 1 + i);
  if (t < 16) {
    kl[t] = E::load(__builtin_bit_cast(T16, k_levels[hc * 16 + t]));
    vl[t] = E::load(__builtin_bit_cast(T16, v_levels[hc * 16 + t]));
  }
  for (int d = t; d < D; d += AT)
    qs[d] = E::load(__builtin_bit_cast(T16, q[row * q_ts + h * q_hs + d])) * sm_scale;
  float m = -3.4e38f, l = 0.f, acc = 0.f;
  for (int t0 = 0; t0 < end; t0 += AT) {
    __syncthreads();
    float z = -INFINITY;
    int64_t at = -1;
    if (t0 + t < end) {
      const uint32_t b = bs.div(t0 + t);
      const uint32_t blk = (uint32_t)tables[(int64_t)r * table_stride + b];
      if (blk < num_blocks) {
        at = ((int64_t)blk * heads + hc) * bs.d + (t0 + t - b * bs.d);
        float s = 0.f;
        for (int d = 0; d < D / 2; ++d) {
          const int c = k_codes[at * (D / 2) + d];
          s += qs[2 * d] * kl[c & 15] + qs[2 * d + 1] * kl[c >> 4];
        }
        z = s * E::load(__builtin_bit_cast(T16, k_scales[at]));
      }
    }
    rows[t] = at;
    float mx = z;
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    if ((t & 63) == 0) red[t >> 6] = mx;
    __syncthreads();
    const float nm = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float w = __expf(z - nm), c = __expf(m - nm);
    m = nm;
    const float ws = wave_sum(w);
    __syncthreads();
    if ((t & 63) == 0) red[t >> 6] = ws;
    p[t] = at >= 0 ? w * E::load(__builtin_bit_cast(T16, v_scales[at])) : 0.f;
    __syncthreads();
    l = l * c + red[0] + red[1] + red[2] + red[3];
    acc *= c;
    const int d = t % D, step = AT / D;
    for (int j = t / D; j < AT; j += step)
      if (rows[j] >= 0) {
        const int cc = v_codes[rows[j] * (D / 2) + d / 2];
        acc += p[j] * vl[(d & 1) ? cc >> 4 : cc & 15];
      }
  }
  part[t] = acc;
  __syncthreads();
  if (t < D) {
    for (int j = t + D; j < AT; j += D) acc += part[j];
    out[((int64_t)row * H + h) * D + t] =
        __builtin_bit_cast(uint16_t, E::store(l > 0.f ? acc / l : 0.f));
  }
  if (t == 0 && lse != nullptr)
    lse[(int64_t)row * H + h] = l > 0.f ? m + __logf(l) : -INFINITY;
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

size_t kv4_attend_workspace_bytes(const fkc_kv4_cache&, int64_t, int64_t, int64_t, int64_t) {
  return 0;
}

int launch_kv4_attend(const fkc_kv4_cache& c, const Kv4Attend& a, void*, size_t,
                      hipStream_t s) {
  return by_shape(c.dtype, c.D, [&](auto dt, auto d) {
    hipLaunchKernelGGL((kv4_attend_kernel<dt.value, d.value>),
                       dim3((uint32_t)a.T, (uint32_t)a.H), dim3(AT), 0, s,
                       (const uint16_t*)a.q.p, a.q.token_stride, a.q.head_stride, (int)a.H,
                       a.tables, a.table_stride, a.seq, a.cu_q, (int)a.R, (int)a.max_seq,
                       (int)a.causal, a.sm_scale, (const uint8_t*)c.k_codes,
                       (const uint8_t*)c.v_codes, (const uint16_t*)c.k_scales,
                       (const uint16_t*)c.v_scales, (const uint16_t*)c.k_levels,
                       (const uint16_t*)c.v_levels, (int)c.heads, (uint32_t)c.num_blocks,
                       FastDiv((uint32_t)c.block_size), (uint16_t*)a.out, a.lse, (int)a.T);
    return check_launch("kv4_attend");
  });
}

}  // namespace fkc
