// What the two forms of key weights share (key_weights_q8.hip: many rows, the keys' scores
// formed twice; key_weights_few_q8.hip: few rows, their scores kept).
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "attention_paged_q8_common.hpp"

namespace kraken {

// Rows of a sequence and KV head up to which its scores are kept: a block of the matrix
// cores' 16 columns.
constexpr uint32_t kFewRows = 16;

// A sequence's rows that count, by KV head, over all groups of rows; 0 if it is left out.
__device__ __forceinline__ uint32_t counted_rows(const KeyWeightsArgs& a, const PagedSequence& s,
                                                 uint32_t group) {
  return s.length > a.stride ? 0u : min(s.count, a.window) * group;
}

// What a key has when sums are added to it: its earlier weight, if it had one, decayed.
__device__ __forceinline__ float decayed_weight(const KeyWeightsArgs& a, const float* at,
                                                bool had) {
  return a.decay > 0.0f && had ? a.decay * *at : 0.0f;
}

// A key's scale, NaN if it is infinite: the scores that it made -inf would vanish.
__device__ __forceinline__ float finite_or_nan(float x) { return fabsf(x) < INFINITY ? x : NAN; }

// What a length cannot pass.
inline uint32_t longest_length(const KeyWeightsArgs& a) {
  const uint64_t table = (uint64_t)a.rows.batch.width << a.rows.cache.page_shift;
  uint64_t keys = a.rows.batch.max_keys < a.stride ? a.rows.batch.max_keys : a.stride;
  keys = table < keys ? table : keys;
  return (uint32_t)keys;
}

// Whether sequences of up to kFewRows rows have their scores kept, and the bytes of that
// (0: no).
size_t few_weights_bytes(const KeyWeightsArgs& a, int cu_count);
void launch_few_weights(const KeyWeightsArgs& a, int cu_count, void* workspace,
                        hipStream_t stream);

}  // namespace kraken
