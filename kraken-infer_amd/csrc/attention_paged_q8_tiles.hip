// Causal attention of a ragged batch over 8-bit KV pages.
#include <hip/hip_runtime.h>

#include "attention_paged_q8_common.hpp"
#include "device_common.hpp"

namespace kraken {
namespace {

// The plain form: a wave per row and head, one key at a time, softmax with a running
// maximum and sum.
template <class T, int kRegs>
__global__ __launch_bounds__(64) void attention_paged_q8_plain(PagedAttentionArgs a) {
  const int lane = threadIdx.x;
  const uint32_t head = blockIdx.x % a.heads, row = blockIdx.x / a.heads;
  const uint32_t d_head = a.cache.head_dim, shift = a.cache.page_shift;
  uint32_t b = 0;
  for (uint32_t at = 1; at <= a.batch.sequences; at += 64) {
    const uint32_t i = at + lane;
    b += (uint32_t)__popcll(__ballot(i <= a.batch.sequences && a.batch.starts[i] <= row));
  }
  if (b >= a.batch.sequences) {
    return;
  }
  const PagedSequence s = paged_sequence(a.batch, b, shift);
  if (row < s.start || row >= s.start + s.count) {
    return;
  }
  if (s.count * (a.heads / a.cache.kv_heads) <= kDecodeRows) {
    return;
  }
  const uint32_t keys = s.length - s.count + (row - s.start) + 1u;
  const uint32_t kv_head = head / (a.heads / a.cache.kv_heads);
  const size_t at = ((size_t)row * a.heads + head) * d_head;
  float q[kRegs], o[kRegs];
  const float scale = 1.0f / sqrtf((float)d_head);
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    q[i] = (float)static_cast<const T*>(a.query)[at + lane + 64 * i] * scale;
    o[i] = 0.0f;
  }
  float m = -1e30f, l = 0.0f;
  for (uint32_t j = 0; j < keys; ++j) {
    const int32_t page = a.batch.table[(size_t)b * a.batch.width + (j >> shift)];
    if (page < 0 || (uint32_t)page >= a.cache.pages) {
      continue;
    }
    const uint32_t slot = j & ((1u << shift) - 1u);
    const size_t page_head = (size_t)page * a.cache.kv_heads + kv_head;
    const int8_t* k = a.cache.keys + ((page_head << shift) + slot) * d_head;
    const int8_t* v = a.cache.values + (page_head << shift) * d_head +
                      (size_t)(slot >> 3) * d_head * 8u + (slot & 7u);
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      dot = fmaf(q[i], (float)k[lane + 64 * i], dot);
    }
    dot = wave_sum(dot) * a.cache.key_scales[page_head];
    const float top = fmaxf(m, dot);
    const float keep = expf(m - top), w = expf(dot - top);
    m = top;
    l = l * keep + w;
    const float wv = w * a.cache.value_scales[page_head];
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      o[i] = o[i] * keep + wv * (float)v[(size_t)(lane + 64 * i) * 8u];
    }
  }
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    float x = l > 0.0f || l != l ? o[i] / l : 0.0f;
    if (a.gate != nullptr) {
      x *= 1.0f / (1.0f + expf(-a.gate[at + lane + 64 * i]));
    }
    static_cast<T*>(a.output)[at + lane + 64 * i] = static_cast<T>(x);
  }
}

template <class T>
void launch_plain(const PagedAttentionArgs& a, hipStream_t stream) {
  const dim3 grid(a.batch.tokens * a.heads);
  if (a.cache.head_dim == 256u) {
    attention_paged_q8_plain<T, 4><<<grid, 64, 0, stream>>>(a);
  } else if (a.cache.head_dim == 128u) {
    attention_paged_q8_plain<T, 2><<<grid, 64, 0, stream>>>(a);
  } else {
    attention_paged_q8_plain<T, 1><<<grid, 64, 0, stream>>>(a);
  }
}

}  // namespace

hipError_t launch_attention_paged_q8_tiles(const PagedAttentionArgs& a, const PagedSplit&,
                                           hipStream_t stream) {
  if (a.f16) {
    launch_plain<half_t>(a, stream);
  } else {
    launch_plain<float>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace kraken
