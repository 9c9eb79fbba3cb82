// C ABI of the attention entry points: host-side checks before any launch.
#include <math.h>

#include "attn.h"

using namespace dsk;

namespace {

constexpr int64_t kMostBlocks = 1 << 23;   // a launch counts its threads in 32 bits

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int check_heads(const char* fn, int heads, int kv_heads, int head_dim) {
  if (head_dim != 64 && head_dim != 128)
    return fail(DSK_EUNSUPPORTED, "%s: head_dim=%d, 64 and 128 are built", fn, head_dim);
  if (kv_heads < 1 || kv_heads > 1024) return fail(DSK_EINVAL, "%s: kv_heads=%d must be in [1, 1024]", fn, kv_heads);
  if (heads < 1 || heads > 1024 || heads % kv_heads || heads / kv_heads > 64)
    return fail(DSK_EINVAL, "%s: heads=%d must be 1 to 64 times kv_heads=%d, at most 1024", fn, heads, kv_heads);
  return DSK_OK;
}

constexpr int64_t kMostStride = int64_t{1} << 40;

// Strides of `what`: rows of 16-byte pieces, `unit` elements each.
int check_strides(const char* fn, const char* what, int64_t token, int64_t head, int unit) {
  if (token % unit || head % unit)
    return fail(DSK_EALIGN, "%s: strides of %s (%lld, %lld) must be multiples of %d elements", fn, what,
                static_cast<long long>(token), static_cast<long long>(head), unit);
  if (token < 0 || head < 0 || token > kMostStride || head > kMostStride)
    return fail(DSK_EINVAL, "%s: strides of %s (%lld, %lld) out of range", fn, what, static_cast<long long>(token),
                static_cast<long long>(head));
  return DSK_OK;
}

// Rows that are written: no two heads or tokens may share elements.
int check_out(const char* fn, const char* what, int64_t token, int64_t head, int64_t tokens, int heads, int head_dim) {
  const bool in_range = token >= 0 && head >= 0 && token <= kMostStride && head <= kMostStride;   // else refused below
  bool apart = !in_range || ((tokens == 1 || token >= head_dim) && (heads == 1 || head >= head_dim));
  if (in_range && apart && tokens > 1 && heads > 1 && token < head * (heads - 1) + head_dim) {
    // a token's heads do not lie together: the tokens next to a distance of i heads, before and behind it
    for (int64_t i = 1; i < heads && apart; ++i) {
      const int64_t before = i * head / token, rest = i * head % token;
      apart = (before >= tokens || rest >= head_dim) && (before + 1 >= tokens || token - rest >= head_dim);
    }
  }
  if (!apart)
    return fail(DSK_EINVAL, "%s: rows of %s overlap (strides %lld, %lld)", fn, what, static_cast<long long>(token),
                static_cast<long long>(head));
  return check_strides(fn, what, token, head, 8);
}

int check_cache(const char* fn, const dsk_kv_cache* c) {
  if (!c) return fail(DSK_EINVAL, "%s: cache is NULL", fn);
  const int p = c->page_size;
  if (p != 16 && p != 32 && p != 64 && p != 128 && p != 256)
    return fail(DSK_EINVAL, "%s: page_size=%d must be 16, 32, 64, 128 or 256", fn, p);
  if (c->n_pages < 1 || c->n_seqs < 1 || c->max_pages < 1)
    return fail(DSK_EINVAL, "%s: n_pages=%d, n_seqs=%d, max_pages=%d must be >= 1", fn, c->n_pages, c->n_seqs, c->max_pages);
  if (static_cast<int64_t>(c->max_pages) * p >= (int64_t{1} << 30))
    return fail(DSK_EUNSUPPORTED, "%s: a sequence of %lld positions exceeds 2^30", fn, static_cast<long long>(c->max_pages) * p);
  if (c->table_stride < c->max_pages && c->n_seqs > 1)
    return fail(DSK_EINVAL, "%s: table_stride=%lld is less than max_pages=%d", fn, static_cast<long long>(c->table_stride), c->max_pages);
  return DSK_OK;
}

int check_cache_pointers(const char* fn, const void* k, const void* v, const int32_t* table) {
  if (!k || !v || !table) return fail(DSK_EINVAL, "%s: k_cache, v_cache or table is NULL", fn);
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(DSK_EALIGN, "%s: the cache must be 16-byte aligned", fn);
  if (!aligned(table, 4)) return fail(DSK_EALIGN, "%s: the page table must be 4-byte aligned", fn);
  return DSK_OK;
}

int check_qk(const char* fn, const dsk_qk_desc* d, const void* q, const void* k, const int32_t* positions,
             const double* freq, const float* q_gamma, const float* k_gamma, void* q_out) {
  if (!d) return fail(DSK_EINVAL, "%s: desc is NULL", fn);
  if (d->tokens < 1) return fail(DSK_EINVAL, "%s: tokens=%d must be >= 1", fn, d->tokens);
  if (d->tokens > kMostBlocks) return fail(DSK_EUNSUPPORTED, "%s: tokens=%d exceeds 2^23", fn, d->tokens);
  if (d->head_dim != 64 && d->head_dim != 128)
    return fail(DSK_EUNSUPPORTED, "%s: head_dim=%d, 64 and 128 are built", fn, d->head_dim);
  if (d->heads < 0 || d->heads > 1024 || d->kv_heads < 1 || d->kv_heads > 1024)
    return fail(DSK_EINVAL, "%s: heads=%d must be in [0, 1024], kv_heads=%d in [1, 1024]", fn, d->heads, d->kv_heads);
  if (d->dtype != DSK_DTYPE_BF16 && d->dtype != DSK_DTYPE_F32)
    return fail(DSK_EINVAL, "%s: dtype %d must be BF16 or F32", fn, d->dtype);
  if (!k || !positions || (d->heads > 0 && (!q || !q_out)) || (d->heads == 0 && (q || q_out)))
    return fail(DSK_EINVAL, "%s: NULL pointer argument, or queries without heads", fn);
  if (d->rot_dim < 0 || d->rot_dim % 16 || d->rot_first < 0 || d->rot_first % 8 ||
      d->rot_dim > d->head_dim || d->rot_first > d->head_dim - d->rot_dim)
    return fail(DSK_EINVAL, "%s: rot_dim=%d must be a multiple of 16 and rot_first=%d one of 8, inside head_dim=%d", fn,
                d->rot_dim, d->rot_first, d->head_dim);
  if (d->rot_dim > 0 && !freq) return fail(DSK_EINVAL, "%s: freq is NULL", fn);
  if (!(d->eps >= 0.0f) || !isfinite(d->eps) || !isfinite(d->mscale))
    return fail(DSK_EINVAL, "%s: eps must be >= 0, eps and mscale finite", fn);
  if (!d->norm && (q_gamma || k_gamma)) return fail(DSK_EINVAL, "%s: gamma without the norm", fn);
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(q_out, 16))
    return fail(DSK_EALIGN, "%s: q, k and q_out must be 16-byte aligned", fn);
  if (!aligned(positions, 4) || !aligned(freq, 8) || !aligned(q_gamma, 4) || !aligned(k_gamma, 4))
    return fail(DSK_EALIGN, "%s: positions, freq and the gammas must be aligned to their type", fn);
  const int unit = d->dtype == DSK_DTYPE_BF16 ? 8 : 4;
  int rc = d->heads ? check_strides(fn, "q", d->q_token, d->q_head, unit) : DSK_OK;
  if (!rc) rc = check_strides(fn, "k", d->k_token, d->k_head, unit);
  if (!rc && d->heads) rc = check_out(fn, "q_out", d->qo_token, d->qo_head, d->tokens, d->heads, d->head_dim);
  return rc;
}

}  // namespace

extern "C" {

int dsk_qk_norm_rope(const dsk_qk_desc* d, const void* q, const void* k, const int32_t* positions, const double* freq,
                     const float* q_gamma, const float* k_gamma, void* q_out, void* k_out, void* stream) {
  const char* fn = "dsk_qk_norm_rope";
  int rc = check_qk(fn, d, q, k, positions, freq, q_gamma, k_gamma, q_out);
  if (rc) return rc;
  if (!k_out) return fail(DSK_EINVAL, "%s: k_out is NULL", fn);
  if (!aligned(k_out, 16)) return fail(DSK_EALIGN, "%s: k_out must be 16-byte aligned", fn);
  rc = check_out(fn, "k_out", d->ko_token, d->ko_head, d->tokens, d->kv_heads, d->head_dim);
  if (rc) return rc;
  return hip_check(launch_qk(*d, q, k, nullptr, positions, nullptr, freq, q_gamma, k_gamma, nullptr, q_out, k_out,
                             static_cast<hipStream_t>(stream)), fn);
}

int dsk_kv_append(const dsk_qk_desc* d, const dsk_kv_cache* cache, const void* q, const void* k, const void* v,
                  const int32_t* positions, const int32_t* seq, const double* freq, const float* q_gamma,
                  const float* k_gamma, void* k_cache, void* v_cache, const int32_t* table, void* q_out, void* k_out,
                  void* stream) {
  const char* fn = "dsk_kv_append";
  int rc = check_qk(fn, d, q, k, positions, freq, q_gamma, k_gamma, q_out);
  if (rc) return rc;
  if (!v || !seq) return fail(DSK_EINVAL, "%s: v or seq is NULL", fn);
  if (!aligned(v, 16) || !aligned(k_out, 16)) return fail(DSK_EALIGN, "%s: v and k_out must be 16-byte aligned", fn);
  if (!aligned(seq, 4)) return fail(DSK_EALIGN, "%s: seq must be 4-byte aligned", fn);
  if (d->prefix_len < 0) return fail(DSK_EINVAL, "%s: prefix_len=%d must be >= 0", fn, d->prefix_len);
  rc = check_cache(fn, cache);
  if (!rc) rc = check_cache_pointers(fn, k_cache, v_cache, table);
  if (!rc) rc = check_strides(fn, "v", d->v_token, d->v_head, d->dtype == DSK_DTYPE_BF16 ? 8 : 4);
  if (!rc && k_out) rc = check_out(fn, "k_out", d->ko_token, d->ko_head, d->tokens, d->kv_heads, d->head_dim);
  if (rc) return rc;
  const CacheView view = cache_view(*cache, k_cache, v_cache, table);
  return hip_check(launch_qk(*d, q, k, v, positions, seq, freq, q_gamma, k_gamma, &view, q_out, k_out,
                             static_cast<hipStream_t>(stream)), fn);
}

int dsk_prompt_attention(const dsk_prompt_desc* d, const void* q, const void* k, const void* v, const int32_t* cu_q,
                         const int32_t* cu_k, void* out, void* stream) {
  const char* fn = "dsk_prompt_attention";
  if (!d) return fail(DSK_EINVAL, "%s: desc is NULL", fn);
  int rc = check_heads(fn, d->heads, d->kv_heads, d->head_dim);
  if (rc) return rc;
  if (d->tokens < 1 || d->kv_tokens < 1) return fail(DSK_EINVAL, "%s: tokens=%d, kv_tokens=%d must be >= 1", fn, d->tokens, d->kv_tokens);
  if (d->n_seqs < 1 || d->n_seqs > 65535) return fail(DSK_EINVAL, "%s: n_seqs=%d must be in [1, 65535]", fn, d->n_seqs);
  if (static_cast<int64_t>(d->tokens) * d->heads >= (int64_t{1} << 30) || d->kv_tokens >= (1 << 30))
    return fail(DSK_EUNSUPPORTED, "%s: tokens * heads and kv_tokens must stay below 2^30", fn);
  if (static_cast<int64_t>(d->n_seqs) * d->kv_heads > kMostBlocks)
    return fail(DSK_EUNSUPPORTED, "%s: n_seqs * kv_heads exceeds 2^23", fn);
  if (!(d->scale > 0.0f) || !isfinite(d->scale)) return fail(DSK_EINVAL, "%s: scale must be positive and finite", fn);
  if (!q || !k || !v || !cu_q || !cu_k || !out) return fail(DSK_EINVAL, "%s: NULL pointer argument", fn);
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
    return fail(DSK_EALIGN, "%s: q, k, v and out must be 16-byte aligned", fn);
  if (!aligned(cu_q, 4) || !aligned(cu_k, 4)) return fail(DSK_EALIGN, "%s: cu_q and cu_k must be 4-byte aligned", fn);
  rc = check_strides(fn, "q", d->q_token, d->q_head, 8);
  if (!rc) rc = check_strides(fn, "k", d->k_token, d->k_head, 8);
  if (!rc) rc = check_strides(fn, "v", d->v_token, d->v_head, 8);
  if (!rc) rc = check_out(fn, "out", d->o_token, d->o_head, d->tokens, d->heads, d->head_dim);
  if (!rc && (d->k_token >= (1 << 26) || d->v_token >= (1 << 26)))
    rc = fail(DSK_EUNSUPPORTED, "%s: token strides of k and v must stay below 2^26", fn);
  if (rc) return rc;
  return hip_check(launch_prompt(*d, q, k, v, cu_q, cu_k, out, static_cast<hipStream_t>(stream)), fn);
}

static int check_paged(const char* fn, const dsk_paged_desc* d, const dsk_kv_cache* cache) {
  if (!d) return fail(DSK_EINVAL, "%s: desc is NULL", fn);
  int rc = check_heads(fn, d->heads, d->kv_heads, d->head_dim);
  if (!rc) rc = check_cache(fn, cache);
  if (rc) return rc;
  if (d->batch < 1 || d->batch > 65535 || cache->n_seqs != d->batch)
    return fail(DSK_EINVAL, "%s: batch=%d must be in [1, 65535] and the table's rows (%d)", fn, d->batch, cache->n_seqs);
  if (d->q_len < 1 || d->q_len > 16 || d->q_len * (d->heads / d->kv_heads) > 64)
    return fail(DSK_EUNSUPPORTED, "%s: q_len=%d must be in [1, 16] and q_len * heads / kv_heads at most 64", fn, d->q_len);
  if (static_cast<int64_t>(d->batch) * d->q_len * d->heads > kMostBlocks)
    return fail(DSK_EUNSUPPORTED, "%s: batch * q_len * heads exceeds 2^23", fn);
  const int64_t keys = static_cast<int64_t>(cache->max_pages) * cache->page_size;
  if (static_cast<int64_t>(d->batch) * d->kv_heads * (keys / 128 + 1) >= INT32_MAX)
    return fail(DSK_EUNSUPPORTED, "%s: batch * kv_heads * the keys of a table row exceed 2^38", fn);
  if (d->prefix_len < 0 || d->prefix_len >= (1 << 30))
    return fail(DSK_EINVAL, "%s: prefix_len=%d must be in [0, 2^30)", fn, d->prefix_len);
  if (!(d->scale > 0.0f) || !isfinite(d->scale)) return fail(DSK_EINVAL, "%s: scale must be positive and finite", fn);
  rc = check_strides(fn, "q", d->q_token, d->q_head, 8);
  if (!rc) rc = check_out(fn, "out", d->o_token, d->o_head, static_cast<int64_t>(d->batch) * d->q_len, d->heads, d->head_dim);
  return rc;
}

int dsk_paged_attention_workspace_size(const dsk_paged_desc* d, const dsk_kv_cache* cache, size_t* bytes) {
  const char* fn = "dsk_paged_attention_workspace_size";
  int rc = check_paged(fn, d, cache);
  if (rc) return rc;
  if (!bytes) return fail(DSK_EINVAL, "%s: bytes is NULL", fn);
  *bytes = paged_workspace(*d, *cache);
  return DSK_OK;
}

int dsk_paged_attention(const dsk_paged_desc* d, const dsk_kv_cache* cache, const void* q, const void* k_cache,
                        const void* v_cache, const int32_t* table, const int32_t* lens, const int32_t* prefix,
                        void* out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "dsk_paged_attention";
  int rc = check_paged(fn, d, cache);
  if (rc) return rc;
  rc = check_cache_pointers(fn, k_cache, v_cache, table);
  if (rc) return rc;
  if (!q || !lens || !out || !workspace || (d->prefix_len > 0 && !prefix))
    return fail(DSK_EINVAL, "%s: NULL pointer argument", fn);
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 256))
    return fail(DSK_EALIGN, "%s: q and out must be 16-byte, the workspace 256-byte aligned", fn);
  if (!aligned(lens, 4) || !aligned(prefix, 4)) return fail(DSK_EALIGN, "%s: lens and prefix must be 4-byte aligned", fn);
  if (workspace_bytes < paged_workspace(*d, *cache))
    return fail(DSK_ESPACE, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, paged_workspace(*d, *cache));
  const CacheView view = cache_view(*cache, const_cast<void*>(k_cache), const_cast<void*>(v_cache), table);
  return hip_check(launch_paged(*d, *cache, q, view, lens, prefix, out, workspace, static_cast<hipStream_t>(stream)), fn);
}

}  // extern "C"
