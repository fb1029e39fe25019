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

int attend_ok(const fkc_kv4_cache& c, const Kv4Attend& a, int64_t max_blocks) {
  if (int rc = attend_sizes_ok(c, a.H, a.T, a.R, a.max_seq, "kv4_attend")) return rc;
  if (!a.cu_q && a.T != a.R)
    return fail(FKC_ERR_INVALID, "kv4_attend: one query per request needs T == R");
  if (max_blocks < 0 || a.table_stride < max_blocks)
    return fail(FKC_ERR_INVALID, "kv4_attend: rows of tables overlap");
  if (a.max_seq > 0 && (a.max_seq - 1) / c.block_size >= max_blocks)
    return fail(FKC_ERR_INVALID,
                "kv4_attend: max_seq %lld is longer than %lld blocks of %lld",
                (long long)a.max_seq, (long long)max_blocks, (long long)c.block_size);
  if (a.T == 0) return FKC_OK;
  if (int rc = rows_ok(a.q.p, a.q.token_stride, a.q.head_stride, "q", "kv4_attend"))
    return rc;
  if (!a.out || (a.R && !a.seq) || (a.R && a.max_seq && !a.tables))
    return fail(FKC_ERR_INVALID, "kv4_attend: null pointer argument");
  if (!aligned16(a.out))
    return fail(FKC_ERR_INVALID, "kv4_attend: out not 16-byte aligned");
  return FKC_OK;
}

int scores_ok(const fkc_kv4_scores* x, const char* what) {
  if (!x) return fail(FKC_ERR_INVALID, "%s: null scores", what);
  // (beyond these factors of it leave fp32's range)
  if (x->softcap != 0.f && !(x->softcap >= 1e-30f && x->softcap <= 1e30f))
    return fail(FKC_ERR_INVALID, "%s: softcap is not between 1e-30 and 1e30", what);
  if (x->window < 0 || x->window > kI32)
    return fail(FKC_ERR_INVALID, "%s: window out of range", what);
  return FKC_OK;
}

bool plain(const fkc_kv4_scores& x) {
  return x.softcap == 0.f && !x.slopes && x.window == 0 && !x.starts && !x.prefix_lens;
}

Kv4Scores inner(const fkc_kv4_scores& x) {
  return {x.softcap, x.slopes, x.window, x.starts, x.prefix_lens};
}

int tables_ok(const int32_t* tables, int64_t stride, int64_t max_blocks,
              const int32_t* seq, int64_t R, const char* what) {
  if (R < 0 || R > kI32 || max_blocks < 0 || max_blocks > kI32)
    return fail(FKC_ERR_INVALID, "%s: size out of range", what);
  if (stride < max_blocks)
    return fail(FKC_ERR_INVALID, "%s: rows of tables overlap", what);
  // The kernels number the entries in 32 bits.
  if (max_blocks && R >= (int64_t)UINT32_MAX / max_blocks)
    return fail(FKC_ERR_UNSUPPORTED, "%s: 2^32 table entries and more", what);
  if (R && (!seq || (max_blocks && !tables)))
    return fail(FKC_ERR_INVALID, "%s: null pointer argument", what);
  return FKC_OK;
}

int workspace_ok(const void* ws, size_t bytes, size_t need, const char* what) {
  if (need && (!ws || bytes < need))
    return fail(FKC_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", what, bytes, need);
  if (need && reinterpret_cast<uintptr_t>(ws) % kWorkspaceAlign)
    return fail(FKC_ERR_WORKSPACE, "%s: workspace not %d-byte aligned", what,
                kWorkspaceAlign);
  return FKC_OK;
}

// Blocks of one cache fit the other.
int alike(const fkc_kv4_cache& a, const fkc_kv4_cache& b, const char* what) {
  if (a.heads != b.heads || a.block_size != b.block_size || a.D != b.D || a.dtype != b.dtype)
    return fail(FKC_ERR_INVALID,
                "%s: the caches differ in heads, block_size, D or dtype", what);
  // The kernels count the 16-byte units of a block in 32 bits.
  if (a.block_size * a.heads > kI32 / (a.D + 4))
    return fail(FKC_ERR_UNSUPPORTED, "%s: blocks of 2^31 bytes and more", what);
  return FKC_OK;
}

bool overlap(const fkc_kv4_cache& a, const fkc_kv4_cache& b) {
  const int64_t vectors = a.heads * a.block_size;
  auto part = [&](const fkc_kv4_cache& c, int i, uintptr_t* lo) {
    const void* p[] = {c.k_codes, c.v_codes, c.k_scales, c.v_scales};
    *lo = reinterpret_cast<uintptr_t>(p[i]);
    return *lo + (uintptr_t)(c.num_blocks * vectors * (i < 2 ? c.D / 2 : 2));
  };
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      uintptr_t lo, lo2;
      const uintptr_t hi = part(a, i, &lo), hi2 = part(b, j, &lo2);
      if (lo < hi2 && lo2 < hi) return true;
    }
  return false;
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
  const Kv4Attend a{{q, q_token_stride, q_head_stride},
                    H, T, tables, table_stride, seq_lens, cu_q, R, max_seq,
                    causal != 0, sm_scale, out, lse};
  if (int rc = attend_ok(*cache, a, max_blocks)) return rc;
  if (T == 0) return FKC_OK;
  if (int rc = workspace_ok(workspace, workspace_bytes,
                            kv4_attend_workspace_bytes(*cache, H, T, R, max_seq),
                            "kv4_attend"))
    return rc;
  return launch_kv4_attend(*cache, a, workspace, workspace_bytes,
                           reinterpret_cast<hipStream_t>(stream));
}

size_t fkc_kv4_attend_scored_workspace_bytes(const fkc_kv4_cache* cache, int64_t H,
                                             int64_t T, int64_t R, int64_t max_seq,
                                             int causal, const fkc_kv4_scores* scores) {
  clear_error();
  if (cache_ok(cache, "kv4_attend_scored_workspace_bytes") ||
      attend_sizes_ok(*cache, H, T, R, max_seq, "kv4_attend_scored_workspace_bytes") ||
      scores_ok(scores, "kv4_attend_scored_workspace_bytes"))
    return 0;
  if (plain(*scores)) return kv4_attend_workspace_bytes(*cache, H, T, R, max_seq);
  return kv4_attend_scored_workspace_bytes(*cache, H, T, R, max_seq, causal != 0,
                                           inner(*scores));
}

int fkc_kv4_attend_scored(const fkc_kv4_cache* cache, const void* q,
                          int64_t q_token_stride, int64_t q_head_stride, int64_t H,
                          int64_t T, const int32_t* tables, int64_t table_stride,
                          int64_t max_blocks, const int32_t* seq_lens,
                          const int32_t* cu_q, int64_t R, int64_t max_seq, int causal,
                          float sm_scale, const fkc_kv4_scores* scores, void* out,
                          float* lse, void* workspace, size_t workspace_bytes,
                          fkc_stream_t stream) {
  clear_error();
  if (int rc = cache_ok(cache, "kv4_attend")) return rc;
  if (int rc = scores_ok(scores, "kv4_attend")) return rc;
  const Kv4Attend a{{q, q_token_stride, q_head_stride},
                    H, T, tables, table_stride, seq_lens, cu_q, R, max_seq,
                    causal != 0, sm_scale, out, lse};
  if (int rc = attend_ok(*cache, a, max_blocks)) return rc;
  if (T == 0) return FKC_OK;
  const Kv4Scores x = inner(*scores);
  const bool without = plain(*scores);
  const size_t need =
      without ? kv4_attend_workspace_bytes(*cache, H, T, R, max_seq)
              : kv4_attend_scored_workspace_bytes(*cache, H, T, R, max_seq, causal != 0, x);
  if (int rc = workspace_ok(workspace, workspace_bytes, need, "kv4_attend")) return rc;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return without ? launch_kv4_attend(*cache, a, workspace, workspace_bytes, s)
                 : launch_kv4_attend_scored(*cache, a, x, workspace, s);
}

size_t fkc_free_blocks_workspace_bytes(int64_t num_blocks) {
  clear_error();
  if (num_blocks < 0 || num_blocks > kI32) {
    fail(FKC_ERR_INVALID, "free_blocks_workspace_bytes: size out of range");
    return 0;
  }
  return free_blocks_workspace_bytes(num_blocks);
}

int fkc_free_blocks(const int32_t* tables, int64_t table_stride, int64_t max_blocks,
                    const int32_t* seq_lens, int64_t R, int64_t block_size,
                    int64_t num_blocks, int32_t* free_blocks, int32_t* count,
                    void* workspace, size_t workspace_bytes, fkc_stream_t stream) {
  clear_error();
  if (int rc = tables_ok(tables, table_stride, max_blocks, seq_lens, R, "free_blocks"))
    return rc;
  if (block_size < 1 || block_size > (1 << 20) || num_blocks < 0 || num_blocks > kI32)
    return fail(FKC_ERR_INVALID, "free_blocks: size out of range");
  if (!count || (num_blocks && !free_blocks))
    return fail(FKC_ERR_INVALID, "free_blocks: null pointer argument");
  if (int rc = workspace_ok(workspace, workspace_bytes,
                            free_blocks_workspace_bytes(num_blocks), "free_blocks"))
    return rc;
  return launch_free_blocks({tables, table_stride, max_blocks, seq_lens, R}, block_size,
                            num_blocks, free_blocks, count, workspace,
                            reinterpret_cast<hipStream_t>(stream));
}

size_t fkc_kv4_fork_workspace_bytes(const fkc_kv4_cache* cache, int64_t F) {
  clear_error();
  if (cache_ok(cache, "kv4_fork_workspace_bytes") ||
      alike(*cache, *cache, "kv4_fork_workspace_bytes"))
    return 0;
  if (F < 0 || F > kI32) {
    fail(FKC_ERR_INVALID, "kv4_fork_workspace_bytes: F out of range");
    return 0;
  }
  return kv4_fork_workspace_bytes(*cache, F);
}

int fkc_kv4_fork(const fkc_kv4_cache* cache, const int32_t* tables, int64_t table_stride,
                 int64_t max_blocks, const int32_t* seq_lens, int64_t R,
                 const int32_t* parents, int64_t F, const int32_t* free_blocks,
                 int64_t num_free, int32_t* new_tables, int32_t* new_seq, int32_t* taken,
                 void* workspace, size_t workspace_bytes, fkc_stream_t stream) {
  clear_error();
  if (int rc = cache_ok(cache, "kv4_fork")) return rc;
  if (int rc = alike(*cache, *cache, "kv4_fork")) return rc;
  if (int rc = tables_ok(tables, table_stride, max_blocks, seq_lens, R, "kv4_fork"))
    return rc;
  if (F < 0 || F > kI32 || num_free < 0)
    return fail(FKC_ERR_INVALID, "kv4_fork: size out of range");
  if (max_blocks && F >= (int64_t)UINT32_MAX / max_blocks)
    return fail(FKC_ERR_UNSUPPORTED, "kv4_fork: 2^32 table entries and more");
  // (a workgroup of 256 for each, and a launch has less than 2^32 threads)
  if (F >= 1 << 24) return fail(FKC_ERR_UNSUPPORTED, "kv4_fork: 2^24 children and more");
  if (!taken || (F && (!parents || !new_seq || (max_blocks && !new_tables))) ||
      (num_free && !free_blocks))
    return fail(FKC_ERR_INVALID, "kv4_fork: null pointer argument");
  if (int rc = workspace_ok(workspace, workspace_bytes, kv4_fork_workspace_bytes(*cache, F),
                            "kv4_fork"))
    return rc;
  return launch_kv4_fork(*cache, {tables, table_stride, max_blocks, seq_lens, R}, parents, F,
                         free_blocks, num_free, new_tables, new_seq, taken, workspace,
                         reinterpret_cast<hipStream_t>(stream));
}

size_t fkc_kv4_compact_workspace_bytes(const fkc_kv4_cache* cache) {
  clear_error();
  return cache_ok(cache, "kv4_compact_workspace_bytes") ? 0
                                                        : kv4_compact_workspace_bytes(*cache);
}

int fkc_kv4_compact(const fkc_kv4_cache* cache, const int32_t* tables, int64_t table_stride,
                    int64_t max_blocks, const int32_t* seq_lens, int64_t R,
                    const fkc_kv4_cache* into, int32_t* new_tables, int32_t* used,
                    void* workspace, size_t workspace_bytes, fkc_stream_t stream) {
  clear_error();
  if (int rc = cache_ok(cache, "kv4_compact")) return rc;
  if (int rc = cache_ok(into, "kv4_compact")) return rc;
  if (int rc = alike(*cache, *into, "kv4_compact")) return rc;
  if (overlap(*cache, *into))
    return fail(FKC_ERR_INVALID, "kv4_compact: the caches share memory");
  if (int rc = tables_ok(tables, table_stride, max_blocks, seq_lens, R, "kv4_compact"))
    return rc;
  if (!used || (R && max_blocks && !new_tables))
    return fail(FKC_ERR_INVALID, "kv4_compact: null pointer argument");
  if (int rc = workspace_ok(workspace, workspace_bytes, kv4_compact_workspace_bytes(*cache),
                            "kv4_compact"))
    return rc;
  return launch_kv4_compact(*cache, {tables, table_stride, max_blocks, seq_lens, R}, *into,
                            new_tables, used, workspace,
                            reinterpret_cast<hipStream_t>(stream));
}

int fkc_kv4_copy_blocks(const fkc_kv4_cache* cache, const int32_t* src,
                        const fkc_kv4_cache* into, const int32_t* dst, int64_t n,
                        fkc_stream_t stream) {
  clear_error();
  if (int rc = cache_ok(cache, "kv4_copy_blocks")) return rc;
  if (int rc = cache_ok(into, "kv4_copy_blocks")) return rc;
  if (int rc = alike(*cache, *into, "kv4_copy_blocks")) return rc;
  if (n < 0 || n > kI32) return fail(FKC_ERR_INVALID, "kv4_copy_blocks: n out of range");
  if (n == 0 || cache->num_blocks == 0 || into->num_blocks == 0) return FKC_OK;
  if (!src || !dst) return fail(FKC_ERR_INVALID, "kv4_copy_blocks: null pointer argument");
  return launch_kv4_copy_blocks(*cache, src, *into, dst, n,
                                reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
