// Arguments of the kernels over a paged 8-bit KV cache, and the parts they share:
// which rows of a batch a sequence has, and which page holds a position.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace kraken {

// The least scale of a page that is not all zeros: the prologue holds rows that need less
// as zeros, and the attention takes a lesser value scale, zero too, as this one.  A key
// then adds up to 2^(11 + 4 + 70) to a softmax's sum (attention_paged_q8_common.hpp), 2^31
// of them 2^116, below f32's largest; and beside values whose scale is up to 2^30, a key of
// such a page is lost to f32's least normal number only 37 octaves below the top score.
constexpr float kLeastScale = 0x1p-70f;

// kraken_paged_q8_cache with device pointers; page_tokens = 1 << page_shift.
struct PagedQ8Args {
  int8_t* keys;         // [pages][kv_heads][page_tokens][head_dim]
  int8_t* values;       // [pages][kv_heads][page_tokens / 8][head_dim][8]
  float* key_scales;    // [pages][kv_heads]
  float* value_scales;  // [pages][kv_heads]
  uint32_t pages, page_shift, kv_heads, head_dim;
};

// kraken_paged_batch with device pointers.
struct PagedBatchArgs {
  const int32_t* table;    // [sequences][width]
  const uint32_t* starts;  // [sequences + 1]
  const uint32_t* lengths; // [sequences]
  uint32_t sequences, width, tokens, max_query, max_keys;
};

struct PagedPrologueArgs {
  const float* q_gate;
  const float* key;
  const float* value;
  const float* q_norm;
  const float* k_norm;
  const int32_t* positions;  // [4][tokens] or null
  float* query_out;
  float* gate_out;
  PagedQ8Args cache;
  PagedBatchArgs batch;
  uint32_t heads, n_dims, s0, s1, s2, s3;
  double log2_theta;
  float eps;
};

struct PagedAttentionArgs {
  const void* query;  // f32, or f16 with f16 set
  const float* gate;  // nullable
  void* output;       // as the query
  PagedQ8Args cache;
  PagedBatchArgs batch;
  uint32_t heads;
  bool f16;
};

struct SampleArgs {
  const float* logits;
  const float* temperature;  // nullable, as the next three
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniforms;
  int32_t* tokens;
  float* probabilities;  // nullable
  size_t row_stride;
  uint32_t rows, size;
};

// kraken_shared_prefixes with device pointers.
struct SharedPrefixArgs {
  const uint32_t* starts;   // [groups + 1]
  const uint32_t* lengths;  // [groups]
  uint32_t groups, max_rows, max_prefix;
};

struct KeyWeightsArgs {
  PagedAttentionArgs rows;  // without gate and output
  uint32_t window;          // rows of a sequence that count
  float decay;
  float* weights;     // [sequences][kv_heads][row_stride]
  size_t row_stride;
  uint32_t stride;    // row_stride, as far as a length goes
};

struct SelectKeysArgs {
  const float* weights;  // [sequences][kv_heads][weight_stride]
  const uint32_t* lengths;
  const uint32_t* keep;
  int32_t* kept;  // [sequences][kv_heads][kept_stride]
  uint32_t* kept_lengths;
  size_t weight_stride, kept_stride;
  uint32_t sequences, kv_heads, max_keys, first, last;
};

struct GatherPagesArgs {
  PagedQ8Args cache;
  const int32_t* table;         // [sequences][width]
  const int32_t* target_table;  // [sequences][target_width]
  const int32_t* kept;          // [sequences][kv_heads][kept_stride]
  const uint32_t* kept_lengths;
  const float* weights;   // [sequences][kv_heads][weight_stride] or null
  float* weights_output;  // alike
  size_t kept_stride, weight_stride;
  uint32_t sequences, width, target_width;
};

constexpr uint32_t kMaxTopLogprobs = 32;

struct LogprobsArgs {
  const float* logits;
  const float* temperature;  // nullable, as the next and the outputs
  const int32_t* tokens;
  float* logprobs;
  int32_t* ranks;
  float* entropies;
  int32_t* top_tokens;
  float* top_logprobs;
  size_t row_stride;
  uint32_t rows, size, top;
};

hipError_t launch_prologue_paged_q8(const PagedPrologueArgs& a, hipStream_t stream);
hipError_t launch_dequantize_pages_q8(const PagedQ8Args& c, const int32_t* ids, uint32_t count,
                                      void* key_rows, void* value_rows, hipStream_t stream);
size_t attention_paged_q8_workspace_bytes(const PagedAttentionArgs& a, int cu_count);
hipError_t launch_attention_paged_q8(const PagedAttentionArgs& a, int cu_count, void* workspace,
                                     hipStream_t stream);
size_t attention_shared_q8_workspace_bytes(const PagedAttentionArgs& a, const SharedPrefixArgs& p,
                                           int cu_count);
hipError_t launch_attention_shared_q8(const PagedAttentionArgs& a, const SharedPrefixArgs& p,
                                      int cu_count, void* workspace, hipStream_t stream);
size_t key_weights_workspace_bytes(const KeyWeightsArgs& a, int cu_count);
hipError_t launch_key_weights(const KeyWeightsArgs& a, int cu_count, void* workspace,
                              hipStream_t stream);
hipError_t launch_select_keys(const SelectKeysArgs& a, hipStream_t stream);
hipError_t launch_gather_pages(const GatherPagesArgs& a, hipStream_t stream);
size_t token_logprobs_workspace_bytes(const LogprobsArgs& a);
hipError_t launch_token_logprobs(const LogprobsArgs& a, void* workspace, hipStream_t stream);
size_t sample_workspace_bytes(const SampleArgs& a);
hipError_t launch_sample(const SampleArgs& a, void* workspace, hipStream_t stream);

// A sequence's rows of the batch and its length; count 0 where it brings none or
// breaks a bound of the batch (it is then left out).
struct PagedSequence {
  uint32_t start, count, length;
};

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatchArgs& b, uint32_t sequence,
                                                        uint32_t page_shift) {
  const uint32_t start = b.starts[sequence], end = b.starts[sequence + 1];
  const uint32_t length = b.lengths[sequence];
  const uint32_t count = end - start;
  const bool fits = start <= end && end <= b.tokens && count <= b.max_query && count <= length &&
                    length <= b.max_keys && (uint64_t)length <= (uint64_t)b.width << page_shift;
  return {start, fits ? count : 0u, fits ? length : 0u};
}

// The sequence that row `token` of the batch belongs to, looked for by a wave, 64
// sequences at a time; count 0 where none has it.
struct PagedRow {
  PagedSequence sequence;
  uint32_t index;
};

__device__ __forceinline__ PagedRow paged_row(const PagedBatchArgs& b, uint32_t token,
                                              uint32_t page_shift) {
  const uint32_t lane = threadIdx.x & 63u;
  for (uint32_t at = 0; at < b.sequences; at += 64) {
    const uint32_t i = at + lane;
    PagedSequence s{0u, 0u, 0u};
    if (i < b.sequences) {
      s = paged_sequence(b, i, page_shift);
    }
    const uint64_t has = __ballot(token - s.start < s.count);
    if (has != 0) {
      const int from = __builtin_ctzll(has);
      return {{(uint32_t)__builtin_amdgcn_readlane((int)s.start, from),
               (uint32_t)__builtin_amdgcn_readlane((int)s.count, from),
               (uint32_t)__builtin_amdgcn_readlane((int)s.length, from)},
              at + (uint32_t)from};
    }
  }
  return {{0u, 0u, 0u}, 0u};
}

// Sum over a wave's lanes up to each (row_shr within 16 lanes, then the rows before).
__device__ __forceinline__ uint32_t wave_prefix(uint32_t x) {
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, true);
  return x;
}

// Item `want` of a batch whose sequences have count(sequence) items each, looked for by
// every wave of a workgroup, 64 sequences at a time: its sequence (index and rows; count 0
// past the last item) and its number there.
struct PagedItem {
  PagedSequence sequence;
  uint32_t index, item;
};

template <class Count>
__device__ __forceinline__ PagedItem paged_item(const PagedBatchArgs& b, uint32_t want,
                                                uint32_t page_shift, Count count) {
  const uint32_t lane = threadIdx.x & 63u;
  for (uint32_t at = 0; at < b.sequences; at += 64) {
    const uint32_t i = at + lane;
    PagedSequence s{0u, 0u, 0u};
    uint32_t items = 0;
    if (i < b.sequences) {
      s = paged_sequence(b, i, page_shift);
      items = s.count != 0 ? count(s) : 0u;
    }
    const uint32_t upto = wave_prefix(items);
    const uint64_t past = __ballot(upto > want);
    if (past != 0) {
      const int from = __builtin_ctzll(past);
      return {{(uint32_t)__builtin_amdgcn_readlane((int)s.start, from),
               (uint32_t)__builtin_amdgcn_readlane((int)s.count, from),
               (uint32_t)__builtin_amdgcn_readlane((int)s.length, from)},
              at + (uint32_t)from,
              want - (uint32_t)__builtin_amdgcn_readlane((int)(upto - items), from)};
    }
    want -= (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  }
  return {{0u, 0u, 0u}, 0u, 0u};
}

}  // namespace kraken
