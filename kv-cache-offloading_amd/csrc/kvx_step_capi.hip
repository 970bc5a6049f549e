// C ABI of the operators around an e4m3 KV cache: argument checks, then one
// launcher each. Nothing here allocates, so no C++ exception can leave it.
#include <algorithm>

#include "kvx_step.h"

namespace kvx {
namespace {

constexpr int64_t kMostSpan = int64_t{1} << 40;  // bytes, as elsewhere in the library
constexpr int64_t kMostGrid = (int64_t{1} << 24) - 1;  // workgroups of 256 (1024) threads that a launch may have

bool spans(int64_t a, int64_t b, int64_t c, int64_t d) {
  int64_t p = a;
  return a >= 0 && b >= 0 && c >= 0 && d >= 0 && !__builtin_mul_overflow(p, b, &p) && p <= kMostSpan &&
         !__builtin_mul_overflow(p, c, &p) && p <= kMostSpan && !__builtin_mul_overflow(p, d, &p) && p <= kMostSpan;
}

int check_dtype(int32_t dtype, bool fp32) {
  if (dtype == KVX_DTYPE_BF16 || dtype == KVX_DTYPE_FP16) return KVX_OK;
  if (dtype == KVX_DTYPE_FP32) {
    if (fp32) return KVX_OK;
    return set_error(KVX_E_UNSUPPORTED, "queries of an e4m3 cache are bf16 or fp16");
  }
  return set_error(KVX_E_INVALID, "unknown element type %d", dtype);
}

int bytes_of(int32_t dtype) { return dtype == KVX_DTYPE_FP32 ? 4 : 2; }

// Rows of `heads` * head_dim elements that start on 16 bytes, `stride` elements apart.
int check_rows(const char* what, const void* p, int64_t stride, int64_t count, int64_t row, int32_t dtype) {
  if (count == 0) return KVX_OK;
  if (!p) return set_error(KVX_E_INVALID, "%s is NULL", what);
  if (stride < 0 || !spans(count, stride > row ? stride : row, bytes_of(dtype), 1))
    return set_error(KVX_E_INVALID, "%s: bad stride, or more than 2^40 bytes", what);
  if ((uintptr_t)p % 16 || (count > 1 && stride * bytes_of(dtype) % 16))
    return set_error(KVX_E_INVALID, "%s: rows must start on 16 bytes", what);
  return KVX_OK;
}

int check_cache(const kvx_fp8_cache* c, bool need_v, Fp8Cache* out) {
  if (!c) return set_error(KVX_E_INVALID, "cache is NULL");
  if (c->num_blocks < 0 || c->block_size <= 0 || c->group_size <= 0 || c->num_heads <= 0 || c->head_dim <= 0)
    return set_error(KVX_E_INVALID, "cache sizes must be positive (blocks %d, block size %d, group %d, heads %d, "
                     "head_dim %d)", c->num_blocks, c->block_size, c->group_size, c->num_heads, c->head_dim);
  if (c->block_size % c->group_size)
    return set_error(KVX_E_INVALID, "a group of %d tokens does not divide a block of %d", c->group_size, c->block_size);
  if (c->group_size % 16 || c->group_size > kMaxGroup)
    return set_error(KVX_E_UNSUPPORTED, "groups are multiples of 16 tokens, up to %d (got %d)", kMaxGroup, c->group_size);
  if (c->head_dim % 16 || c->head_dim > kMaxHeadDim)
    return set_error(KVX_E_UNSUPPORTED, "head_dim is a multiple of 16, up to %d (got %d)", kMaxHeadDim, c->head_dim);
  if (c->num_heads > 32767) return set_error(KVX_E_UNSUPPORTED, "more than 32767 KV heads");
  if (!spans(c->num_blocks, c->block_size, c->num_heads, c->head_dim))
    return set_error(KVX_E_UNSUPPORTED, "the cache spans more than 2^40 bytes");
  if (c->num_blocks > 0) {
    if (!c->k_codes || !c->k_scales || (need_v && (!c->v_codes || !c->v_scales)))
      return set_error(KVX_E_INVALID, "NULL cache pointer");
    if ((uintptr_t)c->k_codes % 16 || (need_v && (uintptr_t)c->v_codes % 16))
      return set_error(KVX_E_INVALID, "cache codes must start on 16 bytes");
    if ((uintptr_t)c->k_scales % 4 || (need_v && (uintptr_t)c->v_scales % 4))
      return set_error(KVX_E_INVALID, "cache scales must start on 4 bytes");
  }
  out->k = (uint8_t*)c->k_codes;
  out->v = (uint8_t*)c->v_codes;
  out->k_scale = c->k_scales;
  out->v_scale = c->v_scales;
  out->num_blocks = c->num_blocks;
  out->block_size = c->block_size;
  out->group = c->group_size;
  out->heads = c->num_heads;
  out->head_dim = c->head_dim;
  out->block_of = FastDiv((uint32_t)c->block_size);
  out->group_of = FastDiv((uint32_t)c->group_size);
  return KVX_OK;
}

int check_batch(const kvx_paged_batch* b, const Fp8Cache& c, PagedBatch* out, bool need_lens = true) {
  if (!b) return set_error(KVX_E_INVALID, "batch is NULL");
  if (b->num_seqs < 0 || b->num_tokens < 0 || b->table_width < 0 || b->max_seqlen < 0 || b->table_stride < 0)
    return set_error(KVX_E_INVALID, "batch sizes must be non-negative");
  if (b->num_seqs > 65535) return set_error(KVX_E_UNSUPPORTED, "more than 65535 sequences in one call");
  if ((int64_t)b->table_width * c.block_size > (int64_t)INT32_MAX - 2048)
    return set_error(KVX_E_UNSUPPORTED, "block tables reach past 2^31 positions");
  if (b->num_seqs > 0 && ((need_lens && !b->context_lens) || (b->table_width > 0 && !b->block_tables)))
    return set_error(KVX_E_INVALID, "NULL batch pointer");
  if (!b->cu_seqlens && b->num_tokens != b->num_seqs && b->num_tokens != 0)
    return set_error(KVX_E_INVALID, "without cu_seqlens there is one query row a sequence (%d rows, %d sequences)",
                     b->num_tokens, b->num_seqs);
  out->tables = b->block_tables;
  out->context_lens = b->context_lens;
  out->cu_seqlens = b->cu_seqlens;
  out->table_stride = b->table_stride;
  out->table_width = b->table_width;
  out->num_seqs = b->num_seqs;
  out->max_seqlen = b->cu_seqlens ? std::max(1, std::min(b->max_seqlen, b->num_tokens)) : 1;
  out->num_tokens = b->num_tokens;
  return KVX_OK;
}

int check_queries(const Fp8Cache& c, const PagedBatch& b, int32_t q_heads, const void* query, int64_t q_stride,
                  int32_t dtype, float softmax_scale) {
  int rc = check_dtype(dtype, false);
  if (rc) return rc;
  if (q_heads <= 0 || q_heads % c.heads)
    return set_error(KVX_E_INVALID, "%d query heads are not a multiple of %d KV heads", q_heads, c.heads);
  if (!(softmax_scale > 0.0f && softmax_scale < INFINITY))
    return set_error(KVX_E_INVALID, "softmax_scale must be positive and finite");
  if ((int64_t)b.num_tokens * q_heads > int64_t{1} << 30)
    return set_error(KVX_E_UNSUPPORTED, "more than 2^30 query rows");
  return check_rows("query", query, q_stride, b.num_tokens, (int64_t)q_heads * c.head_dim, dtype);
}

}  // namespace
}  // namespace kvx

using namespace kvx;

extern "C" {

int kvx_rotary_embed(const void* query, int64_t query_stride, const void* key, int64_t key_stride, void* query_out,
                     int64_t query_out_stride, void* key_out, int64_t key_out_stride, const void* positions,
                     int32_t position_bytes, const double* frequencies, int64_t num_tokens, int32_t query_heads,
                     int32_t key_heads, int32_t head_dim, int32_t rotary_dim, int32_t interleaved, float magnitude,
                     int32_t dtype, void* stream) {
  int rc = check_dtype(dtype, true);
  if (rc) return rc;
  if (num_tokens < 0 || query_heads < 0 || key_heads < 0 || head_dim <= 0)
    return set_error(KVX_E_INVALID, "sizes must be non-negative, head_dim positive");
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return set_error(KVX_E_INVALID, "rotary_dim must be even and within head_dim (%d of %d)", rotary_dim, head_dim);
  if (rotary_dim > 4096) return set_error(KVX_E_UNSUPPORTED, "rotary_dim exceeds 4096");
  if (position_bytes != 4 && position_bytes != 8) return set_error(KVX_E_INVALID, "positions are int32 or int64");
  if (query_stride < 0 || key_stride < 0 || query_out_stride < 0 || key_out_stride < 0)
    return set_error(KVX_E_INVALID, "strides must be non-negative");
  if (num_tokens == 0 || query_heads + (int64_t)key_heads == 0) return KVX_OK;
  if (num_tokens > kMostGrid || (query_heads + (int64_t)key_heads) * head_dim > INT32_MAX)
    return set_error(KVX_E_UNSUPPORTED, "too many tokens or heads for one launch");
  if (!positions || !frequencies || (query_heads && (!query || !query_out)) || (key_heads && (!key || !key_out)))
    return set_error(KVX_E_INVALID, "NULL tensor pointer");
  RotaryArgs a{};
  a.query = query;
  a.key = key;
  a.query_out = query_out;
  a.key_out = key_out;
  a.q_stride = query_stride;
  a.k_stride = key_stride;
  a.q_out_stride = query_out_stride;
  a.k_out_stride = key_out_stride;
  a.positions = positions;
  a.frequencies = frequencies;
  a.num_tokens = num_tokens;
  a.q_heads = query_heads;
  a.k_heads = key_heads;
  a.head_dim = head_dim;
  a.rotary_dim = rotary_dim;
  a.long_positions = position_bytes == 8;
  a.interleaved = interleaved != 0;
  a.magnitude = magnitude;
  return hip_status(launch_rotary(a, dtype, (hipStream_t)stream), "rotary_embed launch");
}

int kvx_store_kvcache_fp8(const kvx_fp8_cache* cache, const void* key, int64_t key_stride, const void* value,
                          int64_t value_stride, int32_t dtype, const int32_t* slot_mapping, int64_t num_tokens,
                          void* stream) {
  Fp8Cache c;
  int rc = check_cache(cache, true, &c);
  if (!rc) rc = check_dtype(dtype, true);
  if (rc) return rc;
  if (num_tokens < 0) return set_error(KVX_E_INVALID, "negative token count");
  if (num_tokens == 0 || c.num_blocks == 0) return KVX_OK;
  if (!slot_mapping) return set_error(KVX_E_INVALID, "slot_mapping is NULL");
  // Workgroups of 16 tokens, the smallest group; where there are few, of fewer.
  if (num_tokens > INT32_MAX - 2048 || slices_grid(num_tokens / 16 + 1, 2 * c.heads) > kMostGrid)
    return set_error(KVX_E_UNSUPPORTED, "too many tokens for one launch");
  const int64_t row = (int64_t)c.heads * c.head_dim;
  if ((rc = check_rows("key", key, key_stride, num_tokens, row, dtype))) return rc;
  if ((rc = check_rows("value", value, value_stride, num_tokens, row, dtype))) return rc;
  return hip_status(launch_store_fp8(c, key, key_stride, value, value_stride, dtype, slot_mapping, (int32_t)num_tokens,
                                     (hipStream_t)stream),
                    "store_kvcache_fp8 launch");
}

int kvx_attention_fp8_workspace(const kvx_fp8_cache* cache, const kvx_paged_batch* batch, int32_t query_heads,
                                int64_t* bytes) {
  Fp8Cache c;
  PagedBatch b;
  int rc = check_cache(cache, true, &c);
  if (!rc) rc = check_batch(batch, c, &b);
  if (rc) return rc;
  if (!bytes) return set_error(KVX_E_INVALID, "bytes is NULL");
  if (query_heads <= 0 || query_heads % c.heads)
    return set_error(KVX_E_INVALID, "%d query heads are not a multiple of %d KV heads", query_heads, c.heads);
  *bytes = b.num_seqs == 0 || b.num_tokens == 0
               ? 0
               : attention_workspace(attention_plan(c, b, query_heads).splits, b.num_tokens, query_heads, c.head_dim);
  return KVX_OK;
}

int kvx_attention_fp8(const kvx_fp8_cache* cache, const kvx_paged_batch* batch, const void* query,
                      int64_t query_stride, int32_t query_heads, int32_t dtype, float softmax_scale, void* out,
                      float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  AttentionArgs a{};
  int rc = check_cache(cache, true, &a.cache);
  if (!rc) rc = check_batch(batch, a.cache, &a.batch);
  if (!rc) rc = check_queries(a.cache, a.batch, query_heads, query, query_stride, dtype, softmax_scale);
  if (rc) return rc;
  if (a.batch.num_seqs == 0 || a.batch.num_tokens == 0) return KVX_OK;
  if (!out) return set_error(KVX_E_INVALID, "out is NULL");
  if ((uintptr_t)out % 16 || (uintptr_t)lse % 4) return set_error(KVX_E_INVALID, "out must start on 16 bytes, lse on 4");
  a.query = query;
  a.q_stride = query_stride;
  a.q_heads = query_heads;
  a.per_kv = query_heads / a.cache.heads;
  a.per_kv_of = FastDiv((uint32_t)a.per_kv);
  a.scale = softmax_scale * 1.4426950408889634f;
  a.out = out;
  a.lse = lse;
  const AttentionPlan plan = attention_plan(a.cache, a.batch, query_heads);
  a.splits = plan.splits;
  a.split_steps = plan.split_steps;
  a.row_tiles = plan.row_tiles;
  const int64_t need = attention_workspace(a.splits, a.batch.num_tokens, query_heads, a.cache.head_dim);
  if (need > workspace_bytes || (need > 0 && (!workspace || (uintptr_t)workspace % 16)))
    return set_error(KVX_E_INVALID, "attention needs %lld bytes of workspace on 16 bytes (got %lld)", (long long)need,
                     (long long)workspace_bytes);
  a.partial = (float*)workspace;
  if (slices_grid((int64_t)a.batch.num_seqs * a.splits * a.row_tiles, a.cache.heads) > kMostGrid / 2)
    return set_error(KVX_E_UNSUPPORTED, "too many sequences, heads and queries for one launch");
  return hip_status(launch_attention(a, dtype, (hipStream_t)stream), "attention_fp8 launch");
}

int kvx_attention_weights_fp8(const kvx_fp8_cache* cache, const kvx_paged_batch* batch, const void* query,
                              int64_t query_stride, int32_t query_heads, int32_t dtype, float softmax_scale,
                              const float* lse, const float* weights, float* out, int64_t width, void* stream) {
  WeightsArgs a{};
  int rc = check_cache(cache, false, &a.cache);
  if (!rc) rc = check_batch(batch, a.cache, &a.batch);
  if (!rc) rc = check_queries(a.cache, a.batch, query_heads, query, query_stride, dtype, softmax_scale);
  if (rc) return rc;
  if (width < 0 || width > (int64_t)INT32_MAX - 2048) return set_error(KVX_E_INVALID, "bad width of the weights");
  if (a.batch.num_seqs == 0 || width == 0) return KVX_OK;
  if (!out || (a.batch.num_tokens > 0 && !lse)) return set_error(KVX_E_INVALID, "NULL tensor pointer");
  if (!spans(a.batch.num_seqs, a.cache.heads, width, 4) ||
      slices_grid((int64_t)a.batch.num_seqs * (width / 128 + 1), a.cache.heads) > kMostGrid)
    return set_error(KVX_E_UNSUPPORTED, "too many weights for one launch");
  a.query = query;
  a.q_stride = query_stride;
  a.q_heads = query_heads;
  a.per_kv = query_heads / a.cache.heads;
  a.per_kv_of = FastDiv((uint32_t)a.per_kv);
  a.scale = softmax_scale * 1.4426950408889634f;
  a.lse = lse;
  a.weights = weights;
  a.out = out;
  a.width = (int32_t)width;
  return hip_status(launch_attention_weights(a, dtype, (hipStream_t)stream), "attention_weights_fp8 launch");
}

int kvx_select_tokens(const float* weights, const int32_t* context_lens, int32_t num_seqs, int32_t num_heads,
                      int64_t width, int32_t keep, int32_t recent, int32_t* indices, int32_t* counts, float* kept,
                      void* stream) {
  if (num_seqs < 0 || num_heads <= 0 || width < 0 || keep < 0 || recent < 0)
    return set_error(KVX_E_INVALID, "sizes must be non-negative");
  if (width > (int64_t)INT32_MAX - 2048 || keep > INT32_MAX - 2048 || !spans(num_seqs, num_heads, width, 4) ||
      !spans(num_seqs, num_heads, keep, 4) || (int64_t)num_seqs * num_heads > kMostGrid / 4)
    return set_error(KVX_E_UNSUPPORTED, "too many weights for one launch");
  if (num_seqs == 0) return KVX_OK;
  if (!context_lens || !counts || (width > 0 && !weights) || (keep > 0 && (!indices || !kept)))
    return set_error(KVX_E_INVALID, "NULL tensor pointer");
  return hip_status(launch_select(weights, num_seqs * num_heads, num_heads, (int32_t)width, context_lens, keep,
                                  recent < keep ? recent : keep, indices, counts, kept, (hipStream_t)stream),
                    "select_tokens launch");
}

int kvx_compact_kvcache_fp8(const kvx_fp8_cache* cache, const kvx_paged_batch* from, const int32_t* indices,
                            const int32_t* counts, int32_t keep, const int32_t* to_tables, int64_t to_stride,
                            int32_t to_width, void* stream) {
  Fp8Cache c;
  PagedBatch b;
  int rc = check_cache(cache, true, &c);
  if (!rc) rc = check_batch(from, c, &b, false);
  if (rc) return rc;
  if (keep < 0 || to_stride < 0 || to_width < 0) return set_error(KVX_E_INVALID, "sizes must be non-negative");
  if (b.num_seqs == 0 || keep == 0 || c.num_blocks == 0) return KVX_OK;
  if (!indices || !counts || !to_tables) return set_error(KVX_E_INVALID, "NULL tensor pointer");
  if ((int64_t)to_width * c.block_size < keep)
    return set_error(KVX_E_RANGE, "%d blocks of %d tokens do not hold %d", to_width, c.block_size, keep);
  if (keep > INT32_MAX - 2048 || !spans(b.num_seqs, c.heads, keep, 4) ||
      slices_grid(((int64_t)keep / c.group + 1) * b.num_seqs, 2 * c.heads) > kMostGrid)
    return set_error(KVX_E_UNSUPPORTED, "too many tokens for one launch");
  return hip_status(launch_compact(c, b, indices, counts, keep, to_tables, to_stride, to_width, (hipStream_t)stream),
                    "compact_kvcache_fp8 launch");
}

}  // extern "C"
