// extern "C" boundary of the 4-bit key/value cache: argument checks.
// Pointers and strides are the caller's contract; everything that a kernel's
// indexing or grid assumes of the sizes is checked here, before any launch.
#include <hip/hip_runtime.h>

#include <limits>

#include "fkc_internal.hpp"

namespace fkc {
namespace {

constexpr int64_t kI32 = std::numeric_limits<int32_t>::max();

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int cache_ok(const fkc_kv4_cache* c, const char* what) {
  if (!c) return fail(FKC_ERR_INVALID, "%s: null cache", what);
  if (c->dtype != FKC_F16 && c->dtype != FKC_BF16)
    return fail(c->dtype == FKC_F32 ? FKC_ERR_UNSUPPORTED : FKC_ERR_INVALID,
                "%s: dtype %d is not fp16 or bf16", what, c->dtype);
  if (c->D != 64 && c->D != 128 && c->D != 256)
    return fail(c->D < 1 ? FKC_ERR_INVALID : FKC_ERR_UNSUPPORTED,
                "%s: D = %lld is not 64, 128 or 256", what, (long long)c->D);
  if (c->block_size < 16 || c->block_size % 16 || c->block_size > (1 << 20))
    return fail(FKC_ERR_INVALID,
                "%s: block_size %lld is not a multiple of 16 up to 2^20", what,
                (long long)c->block_size);
  if (c->heads < 1 || c->heads > 16384 || c->num_blocks < 0 ||
      c->num_blocks > kI32 / c->block_size)
    return fail(FKC_ERR_INVALID,
                "%s: need 1 <= heads <= 16384 and num_blocks * block_size < 2^31",
                what);
  // The kernels number the cache's 16-slot groups over all heads in 32 bits.
  if (c->num_blocks * (c->block_size / 16) > kI32 / c->heads)
    return fail(FKC_ERR_UNSUPPORTED, "%s: slots * heads reaches 2^35", what);
  const void* ps[] = {c->k_codes,  c->v_codes,  c->k_scales,
                      c->v_scales, c->k_levels, c->v_levels};
  if (!c->k_levels || !c->v_levels)
    return fail(FKC_ERR_INVALID, "%s: null levels", what);
  for (const void* p : ps) {
    if (!p && c->num_blocks > 0)  // an empty cache has no codes or scales
      return fail(FKC_ERR_INVALID, "%s: null cache pointer", what);
    if (!aligned16(p))
      return fail(FKC_ERR_INVALID, "%s: cache pointer not 16-byte aligned", what);
  }
  return FKC_OK;
}

// Rows that kernels load 16 bytes at a time.
int rows_ok(const void* p, int64_t ts, int64_t hs, const char* name,
            const char* what) {
  if (!p) return fail(FKC_ERR_INVALID, "%s: null pointer argument", what);
  if (!aligned16(p) || ts % 8 || hs % 8)
    return fail(FKC_ERR_INVALID, "%s: rows of %s not 16-byte aligned", what, name);
  return FKC_OK;
}

int attend_sizes_ok(const fkc_kv4_cache& c, int64_t H, int64_t T, int64_t R,
                    int64_t max_seq, const char* what) {
  if (H < 1 || H > 16384 || H % c.heads)
    return fail(FKC_ERR_INVALID,
                "%s: H = %lld is not a multiple (up to 16384) of the cache's %lld heads",
                what, (long long)H, (long long)c.heads);
  if (T < 0 || R < 0 || max_seq < 0 || T > kI32 / H || R > kI32 / H ||
      max_seq > kI32 - 65536)
    return fail(FKC_ERR_INVALID, "%s: T * H, R * H or max_seq out of range", what);
  return FKC_OK;
}

}  // namespace
}  // namespace fkc

using namespace fkc;

extern "C" {

int fkc_block_tables(const int32_t* seq_lens, const int32_t* new_lens, int64_t R,
                     int32_t* tables, int64_t table_stride, int64_t max_blocks,
                     const int32_t* free_blocks, int64_t num_free,
                     int64_t block_size, int64_t num_tokens, int32_t* slots,
                     int32_t* cu_new, int32_t* taken, fkc_stream_t stream) {
  clear_error();
  if (R < 0 || R > kI32 - 1 || num_free < 0 || num_tokens < 0 ||
      num_tokens > kI32 || max_blocks < 0 || max_blocks > kI32 ||
      block_size < 1 || block_size > (1 << 20))
    return fail(FKC_ERR_INVALID, "block_tables: size out of range");
  if (table_stride < max_blocks)
    return fail(FKC_ERR_INVALID, "block_tables: rows of tables overlap");
  if (!cu_new || !taken || (R && (!seq_lens || !new_lens)) ||
      (R && max_blocks && !tables) || (num_free && !free_blocks) ||
      (num_tokens && !slots))
    return fail(FKC_ERR_INVALID, "block_tables: null pointer argument");
  return launch_block_tables(seq_lens, new_lens, (int)R, tables, table_stride,
                             (int)max_blocks, free_blocks, num_free,
                             (int)block_size, num_tokens, slots, cu_new, taken,
                             reinterpret_cast<hipStream_t>(stream));
}

int fkc_kv4_append(const fkc_kv4_cache* cache, const void* k,
                   int64_t k_token_stride, int64_t k_head_stride, const void* v,
                   int64_t v_token_stride, int64_t v_head_stride,
                   const int32_t* slots, int64_t T, fkc_stream_t stream) {
  clear_error();
  if (int rc = cache_ok(cache, "kv4_append")) return rc;
  if (T < 0 || T > (1 << 30)) return fail(FKC_ERR_INVALID, "kv4_append: T out of range");
  if (T == 0) return FKC_OK;
  if (int rc = rows_ok(k, k_token_stride, k_head_stride, "k", "kv4_append")) return rc;
  if (int rc = rows_ok(v, v_token_stride, v_head_stride, "v", "kv4_append")) return rc;
  if (!slots) return fail(FKC_ERR_INVALID, "kv4_append: null pointer argument");
  return launch_kv4_append(*cache, {k, k_token_stride, k_head_stride},
                           {v, v_token_stride, v_head_stride}, slots, T,
                           reinterpret_cast<hipStream_t>(stream));
}

int fkc_kv4_read(const fkc_kv4_cache* cache, const int32_t* slots, int64_t T,
                 void* k_out, void* v_out, fkc_stream_t stream) {
  clear_error();
  if (int rc = cache_ok(cache, "kv4_read")) return rc;
  if (T < 0 || T > (1 << 30)) return fail(FKC_ERR_INVALID, "kv4_read: T out of range");
  if (T == 0 || (!k_out && !v_out)) return FKC_OK;
  if (!slots) return fail(FKC_ERR_INVALID, "kv4_read: null pointer argument");
  if (!aligned16(k_out) || !aligned16(v_out))
    return fail(FKC_ERR_INVALID, "kv4_read: outputs not 16-byte aligned");
  return launch_kv4_read(*cache, slots, T, k_out, v_out,
                         reinterpret_cast<hipStream_t>(stream));
}

size_t fkc_kv4_attend_workspace_bytes(const fkc_kv4_cache* cache, int64_t H,
                                      int64_t T, int64_t R, int64_t max_seq) {
  clear_error();
  if (cache_ok(cache, "kv4_attend_workspace_bytes") ||
      attend_sizes_ok(*cache, H, T, R, max_seq, "kv4_attend_workspace_bytes"))
    return 0;
  return kv4_attend_workspace_bytes(*cache, H, T, R, max_seq);
}

int fkc_kv4_attend(const fkc_kv4_cache* cache, const void* q,
                   int64_t q_token_stride, int64_t q_head_stride, int64_t H,
                   int64_t T, const int32_t* tables, int64_t table_stride,
                   int64_t max_blocks, const int32_t* seq_lens,
                   const int32_t* cu_q, int64_t R, int64_t max_seq, int causal,
                   float sm_scale, void* out, float* lse, void* workspace,
                   size_t workspace_bytes, fkc_stream_t stream) {
  clear_error();
  if (int rc = cache_ok(cache, "kv4_attend")) return rc;
  if (int rc = attend_sizes_ok(*cache, H, T, R, max_seq, "kv4_attend")) return rc;
  if (!cu_q && T != R)
    return fail(FKC_ERR_INVALID, "kv4_attend: one query per request needs T == R");
  if (max_blocks < 0 || table_stride < max_blocks)
    return fail(FKC_ERR_INVALID, "kv4_attend: rows of tables overlap");
  if (max_seq > 0 && (max_seq - 1) / cache->block_size >= max_blocks)
    return fail(FKC_ERR_INVALID,
                "kv4_attend: max_seq %lld is longer than %lld blocks of %lld",
                (long long)max_seq, (long long)max_blocks,
                (long long)cache->block_size);
  if (T == 0) return FKC_OK;
  if (int rc = rows_ok(q, q_token_stride, q_head_stride, "q", "kv4_attend"))
    return rc;
  if (!out || (R && !seq_lens) || (R && max_seq && !tables))
    return fail(FKC_ERR_INVALID, "kv4_attend: null pointer argument");
  if (!aligned16(out))
    return fail(FKC_ERR_INVALID, "kv4_attend: out not 16-byte aligned");
  const size_t need = kv4_attend_workspace_bytes(*cache, H, T, R, max_seq);
  if (need && (!workspace || workspace_bytes < need))
    return fail(FKC_ERR_WORKSPACE, "kv4_attend: workspace %zu < %zu bytes",
                workspace_bytes, need);
  if (need && reinterpret_cast<uintptr_t>(workspace) % kWorkspaceAlign)
    return fail(FKC_ERR_WORKSPACE, "kv4_attend: workspace not %d-byte aligned",
                kWorkspaceAlign);
  const Kv4Attend a{{q, q_token_stride, q_head_stride},
                    H, T, tables, table_stride, seq_lens, cu_q, R, max_seq,
                    causal != 0, sm_scale, out, lse};
  return launch_kv4_attend(*cache, a, workspace, workspace_bytes,
                           reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
