// C entry points over a paged 8-bit KV cache, and sampling: argument checks in the
// order of the other entries (dimensions, bounds, overflow, buffers, uint32 ranges),
// then one launch function each.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "context_internal.hpp"
#include "paged_q8_internal.hpp"

using namespace kraken;

namespace {

constexpr size_t kInt32Max = 0x7fffffffu;
// Limits that keep a launch's workgroups of 256 threads within a grid: pairs of a sequence
// and a KV head, and rows (tokens x heads), four of which share a workgroup of the join.
constexpr size_t kMaxPairs = size_t{1} << 20;
constexpr size_t kMaxRows = size_t{1} << 26;

int refuse(const char* w, const char* what) { return invalid(std::string("HIP ") + w + what); }

// The cache's checks; `w` begins the messages.
int cache_args(const kraken_paged_q8_cache* cache, const char* w, PagedQ8Args& c) {
  if (cache == nullptr) {
    return refuse(w, " cache must not be null");
  }
  if (cache->pages == 0 || cache->page_tokens == 0 || cache->kv_heads == 0 ||
      cache->head_dim == 0) {
    return refuse(w, " dimensions must be positive");
  }
  uint32_t shift = 0;
  switch (cache->page_tokens) {
    case 16: shift = 4; break;
    case 32: shift = 5; break;
    case 64: shift = 6; break;
    case 128: shift = 7; break;
    default: return refuse(w, " supports pages of 16/32/64/128 tokens");
  }
  if (cache->head_dim != 64 && cache->head_dim != 128 && cache->head_dim != 256) {
    return refuse(w, " supports head_dim 64/128/256");
  }
  if (cache->pages > kInt32Max) {
    return refuse(w, " page count exceeds int32 range");
  }
  size_t scales = 0, tokens = 0, bytes = 0;
  if (!checked_mul(cache->pages, cache->kv_heads, scales) ||
      !checked_mul(scales, cache->page_tokens, tokens) ||
      !checked_mul(tokens, cache->head_dim, bytes)) {
    return refuse(w, " value count overflow");
  }
  KRAKEN_TRY(validate_buffer(cache->key_pages, bytes, 1u, w, " key pages"));
  KRAKEN_TRY(validate_buffer(cache->value_pages, bytes, 1u, w, " value pages"));
  KRAKEN_TRY(validate_f32(cache->key_scales, scales, w, " key scales"));
  KRAKEN_TRY(validate_f32(cache->value_scales, scales, w, " value scales"));
  if (((uintptr_t)cache->key_pages.data | (uintptr_t)cache->value_pages.data) & 15u) {
    return refuse(w, " pages must be 16-byte aligned");
  }
  if (cache->kv_heads > kMaxPairs) {
    return refuse(w, " takes up to 1048576 kv_heads");
  }
  c.keys = static_cast<int8_t*>(cache->key_pages.data);
  c.values = static_cast<int8_t*>(cache->value_pages.data);
  c.key_scales = static_cast<float*>(cache->key_scales.data);
  c.value_scales = static_cast<float*>(cache->value_scales.data);
  c.pages = (uint32_t)cache->pages;
  c.page_shift = shift;
  c.kv_heads = (uint32_t)cache->kv_heads;
  c.head_dim = (uint32_t)cache->head_dim;
  return KRAKEN_OK;
}

int batch_args(const kraken_paged_batch* batch, size_t kv_heads, const char* w,
               PagedBatchArgs& b) {
  if (batch == nullptr) {
    return refuse(w, " batch must not be null");
  }
  if (batch->sequences == 0 || batch->table_width == 0 || batch->tokens == 0 ||
      batch->max_query == 0 || batch->max_keys == 0) {
    return refuse(w, " batch dimensions must be positive");
  }
  if (batch->tokens > kInt32Max || batch->max_keys > kInt32Max) {
    return refuse(w, " batch exceeds int32 range");
  }
  if (batch->sequences > kMaxPairs / kv_heads) {
    return refuse(w, " takes up to 1048576 pairs of a sequence and a KV head");
  }
  size_t entries = 0;
  if (!checked_mul(batch->sequences, batch->table_width, entries)) {
    return refuse(w, " value count overflow");
  }
  KRAKEN_TRY(validate_buffer(batch->page_table, entries, sizeof(int32_t), w, " page table"));
  KRAKEN_TRY(validate_buffer(batch->query_starts, batch->sequences + 1u, sizeof(uint32_t), w,
                             " query starts"));
  KRAKEN_TRY(validate_buffer(batch->lengths, batch->sequences, sizeof(uint32_t), w, " lengths"));
  KRAKEN_TRY(check_u32(batch->table_width, w, " table width"));
  b.table = static_cast<const int32_t*>(batch->page_table.data);
  b.starts = static_cast<const uint32_t*>(batch->query_starts.data);
  b.lengths = static_cast<const uint32_t*>(batch->lengths.data);
  b.sequences = (uint32_t)batch->sequences;
  b.width = (uint32_t)batch->table_width;
  b.tokens = (uint32_t)batch->tokens;
  b.max_keys = (uint32_t)batch->max_keys;
  // No sequence can bring more than either.
  b.max_query = (uint32_t)std::min({batch->max_query, batch->tokens, batch->max_keys});
  return KRAKEN_OK;
}

int finish(kraken_hip_context* ctx, hipError_t e, const char* w) {
  if (e != hipSuccess) {
    return internal(std::string("HIP ") + w + " launch failed: " + hipGetErrorString(e));
  }
  return finish_launch(ctx, "HIP ", w, " command failed: ");
}

int paged_attention_entry(kraken_hip_context* ctx, const kraken_buffer& query,
                          const kraken_buffer& gate, const kraken_paged_q8_cache* cache,
                          const kraken_paged_batch* batch, size_t heads,
                          const kraken_buffer& output, bool f16) {
  const char* w = "paged attention";
  KRAKEN_TRY(check_context(ctx));
  PagedAttentionArgs a{};
  if (heads == 0) {
    return invalid("HIP paged attention dimensions must be positive");
  }
  KRAKEN_TRY(cache_args(cache, w, a.cache));
  if (heads % cache->kv_heads != 0) {
    return invalid("HIP paged attention heads must be divisible by kv_heads");
  }
  KRAKEN_TRY(batch_args(batch, cache->kv_heads, w, a.batch));
  size_t rows = 0, values = 0;
  if (!checked_mul(batch->tokens, heads, rows) || !checked_mul(rows, cache->head_dim, values)) {
    return invalid("HIP paged attention value count overflow");
  }
  if (rows > kMaxRows) {
    return invalid("HIP paged attention takes up to 67108864 query rows");
  }
  const size_t element = f16 ? sizeof(uint16_t) : sizeof(float);
  KRAKEN_TRY(validate_buffer(query, values, element, w, " query"));
  if (gate.data != nullptr) {
    KRAKEN_TRY(validate_f32(gate, values, w, " gate"));
  }
  KRAKEN_TRY(validate_buffer(output, values, element, w, " output"));
  if (((uintptr_t)query.data | (uintptr_t)gate.data | (uintptr_t)output.data) & 15u) {
    return invalid("HIP paged attention buffers must be 16-byte aligned");
  }
  a.query = query.data;
  a.gate = static_cast<const float*>(gate.data);
  a.output = output.data;
  a.heads = (uint32_t)heads;
  a.f16 = f16;
  KRAKEN_TRY(begin_launch(ctx));
  KRAKEN_TRY(ensure_workspace(ctx, attention_paged_q8_workspace_bytes(a, ctx->cu_count)));
  return finish(ctx, launch_attention_paged_q8(a, ctx->cu_count, ctx->workspace, ctx->stream), w);
}

}  // namespace

extern "C" {

KRAKEN_API int kraken_hip_qwen35_attention_prologue_paged_q8_kv(
  kraken_hip_context* ctx, kraken_buffer q_gate, kraken_buffer key, kraken_buffer value,
  kraken_buffer q_norm, kraken_buffer k_norm, kraken_buffer positions,
  const kraken_paged_q8_cache* cache, const kraken_paged_batch* batch, size_t heads,
  size_t n_dims, size_t section_0, size_t section_1, size_t section_2, size_t section_3,
  float theta, float eps, kraken_buffer query_out, kraken_buffer gate_out) {
  const char* w = "paged attention prologue";
  KRAKEN_TRY(check_context(ctx));
  PagedPrologueArgs a{};
  if (heads == 0) {
    return invalid("HIP paged attention prologue dimensions must be positive");
  }
  KRAKEN_TRY(cache_args(cache, w, a.cache));
  if (heads % cache->kv_heads != 0) {
    return invalid("HIP paged attention prologue heads must be divisible by kv_heads");
  }
  if (n_dims == 0 || n_dims > cache->head_dim || n_dims % 2u != 0) {
    return invalid("HIP MRoPE dimensions are invalid");
  }
  size_t sections = 0;
  if (!checked_add(section_0, section_1, sections) ||
      !checked_add(sections, section_2, sections) ||
      !checked_add(sections, section_3, sections)) {
    return invalid("HIP MRoPE sections overflow");
  }
  if (sections == 0) {
    return invalid("HIP MRoPE sections must not all be zero");
  }
  if (!(theta > 0.0f) || std::isinf(theta)) {
    return invalid("HIP MRoPE theta must be positive and finite");
  }
  KRAKEN_TRY(batch_args(batch, cache->kv_heads, w, a.batch));
  const size_t tokens = batch->tokens;
  size_t rows = 0, query_values = 0, joint_values = 0, kv_rows = 0, kv_values = 0;
  if (!checked_mul(tokens, heads, rows) || !checked_mul(rows, cache->head_dim, query_values) ||
      !checked_mul(query_values, 2u, joint_values) ||
      !checked_mul(tokens, cache->kv_heads, kv_rows) ||
      !checked_mul(kv_rows, cache->head_dim, kv_values)) {
    return invalid("HIP paged attention prologue value count overflow");
  }
  KRAKEN_TRY(validate_f32(q_gate, joint_values, w, " q_gate"));
  KRAKEN_TRY(validate_f32(key, kv_values, w, " key"));
  KRAKEN_TRY(validate_f32(value, kv_values, w, " value"));
  KRAKEN_TRY(validate_f32(q_norm, cache->head_dim, w, " q_norm"));
  KRAKEN_TRY(validate_f32(k_norm, cache->head_dim, w, " k_norm"));
  if (positions.data != nullptr) {
    KRAKEN_TRY(validate_buffer(positions, 4u * tokens, sizeof(int32_t), w, " positions"));
  }
  KRAKEN_TRY(validate_f32(query_out, query_values, w, " query output"));
  KRAKEN_TRY(validate_f32(gate_out, query_values, w, " gate output"));
  KRAKEN_TRY(check_u32(heads, w, " heads"));
  KRAKEN_TRY(check_u32(sections, "MRoPE", " sections"));
  a.q_gate = static_cast<const float*>(q_gate.data);
  a.key = static_cast<const float*>(key.data);
  a.value = static_cast<const float*>(value.data);
  a.q_norm = static_cast<const float*>(q_norm.data);
  a.k_norm = static_cast<const float*>(k_norm.data);
  a.positions = static_cast<const int32_t*>(positions.data);
  a.query_out = static_cast<float*>(query_out.data);
  a.gate_out = static_cast<float*>(gate_out.data);
  a.heads = (uint32_t)heads;
  a.n_dims = (uint32_t)n_dims;
  a.s0 = (uint32_t)section_0;
  a.s1 = (uint32_t)section_1;
  a.s2 = (uint32_t)section_2;
  a.s3 = (uint32_t)section_3;
  a.log2_theta = std::log2((double)theta);
  a.eps = eps;
  KRAKEN_TRY(begin_launch(ctx));
  return finish(ctx, launch_prologue_paged_q8(a, ctx->stream), w);
}

KRAKEN_API int kraken_hip_attention_f32_paged_q8_kv(
  kraken_hip_context* ctx, kraken_buffer query, kraken_buffer gate,
  const kraken_paged_q8_cache* cache, const kraken_paged_batch* batch, size_t heads,
  kraken_buffer output) {
  return paged_attention_entry(ctx, query, gate, cache, batch, heads, output, false);
}

KRAKEN_API int kraken_hip_attention_f16q_paged_q8_kv(
  kraken_hip_context* ctx, kraken_buffer query, const kraken_paged_q8_cache* cache,
  const kraken_paged_batch* batch, size_t heads, kraken_buffer output) {
  return paged_attention_entry(ctx, query, kraken_buffer{nullptr, 0}, cache, batch, heads, output,
                               true);
}

KRAKEN_API int kraken_hip_dequantize_kv_pages_q8_f16(
  kraken_hip_context* ctx, const kraken_paged_q8_cache* cache, kraken_buffer page_ids,
  size_t count, kraken_buffer key_rows, kraken_buffer value_rows) {
  const char* w = "KV page dequantize";
  KRAKEN_TRY(check_context(ctx));
  if (count == 0) {
    return invalid("HIP KV page dequantize dimensions must be positive");
  }
  PagedQ8Args c{};
  KRAKEN_TRY(cache_args(cache, w, c));
  size_t heads = 0, tokens = 0, values = 0;
  if (!checked_mul(count, cache->kv_heads, heads) ||
      !checked_mul(heads, cache->page_tokens, tokens) ||
      !checked_mul(tokens, cache->head_dim, values)) {
    return invalid("HIP KV page dequantize value count overflow");
  }
  if (heads > kInt32Max / 256u) {
    return invalid("HIP KV page dequantize takes too many pages at once");
  }
  KRAKEN_TRY(validate_buffer(page_ids, count, sizeof(int32_t), w, " page ids"));
  KRAKEN_TRY(validate_buffer(key_rows, values, sizeof(uint16_t), w, " key rows"));
  KRAKEN_TRY(validate_buffer(value_rows, values, sizeof(uint16_t), w, " value rows"));
  if (((uintptr_t)key_rows.data | (uintptr_t)value_rows.data) & 15u) {
    return invalid("HIP KV page dequantize rows must be 16-byte aligned");
  }
  KRAKEN_TRY(begin_launch(ctx));
  return finish(ctx,
                launch_dequantize_pages_q8(c, static_cast<const int32_t*>(page_ids.data),
                                           (uint32_t)count, key_rows.data, value_rows.data,
                                           ctx->stream),
                w);
}

KRAKEN_API int kraken_hip_sample_f32_i32(kraken_hip_context* ctx, kraken_buffer logits,
                                         size_t rows, size_t size, size_t row_stride,
                                         kraken_buffer temperature, kraken_buffer top_k,
                                         kraken_buffer top_p, kraken_buffer min_p,
                                         kraken_buffer uniforms, kraken_buffer token_output,
                                         kraken_buffer probability_output) {
  const char* w = "sample";
  KRAKEN_TRY(check_context(ctx));
  if (rows == 0 || size == 0) {
    return invalid("HIP sample dimensions must be positive");
  }
  if (row_stride < size) {
    return invalid("HIP sample row stride must be at least the row size");
  }
  size_t values = 0;
  if (!checked_mul(rows - 1u, row_stride, values) || !checked_add(values, size, values)) {
    return invalid("HIP sample value count overflow");
  }
  if (size > (size_t{1} << 22) || rows > 65535u) {
    return invalid("HIP sample takes rows of up to 4194304 logits, and 65535 of them");
  }
  KRAKEN_TRY(validate_f32(logits, values, w, " logits"));
  const struct {
    const kraken_buffer& buffer;
    const char* name;
  } optional[] = {{temperature, " temperature"},
                  {top_k, " top_k"},
                  {top_p, " top_p"},
                  {min_p, " min_p"},
                  {probability_output, " probability output"}};
  for (const auto& o : optional) {
    if (o.buffer.data != nullptr) {
      KRAKEN_TRY(validate_buffer(o.buffer, rows, 4u, w, o.name));
    }
  }
  KRAKEN_TRY(validate_f32(uniforms, rows, w, " uniforms"));
  KRAKEN_TRY(validate_buffer(token_output, rows, sizeof(int32_t), w, " token output"));
  SampleArgs a{};
  a.logits = static_cast<const float*>(logits.data);
  a.temperature = static_cast<const float*>(temperature.data);
  a.top_k = static_cast<const int32_t*>(top_k.data);
  a.top_p = static_cast<const float*>(top_p.data);
  a.min_p = static_cast<const float*>(min_p.data);
  a.uniforms = static_cast<const float*>(uniforms.data);
  a.tokens = static_cast<int32_t*>(token_output.data);
  a.probabilities = static_cast<float*>(probability_output.data);
  a.row_stride = row_stride;
  a.rows = (uint32_t)rows;
  a.size = (uint32_t)size;
  KRAKEN_TRY(begin_launch(ctx));
  KRAKEN_TRY(ensure_workspace(ctx, sample_workspace_bytes(a)));
  return finish(ctx, launch_sample(a, ctx->workspace, ctx->stream), w);
}

}  // extern "C"
