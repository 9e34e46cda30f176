// The attention weight that cached keys receive from a batch's rows.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention_paged_q8_common.hpp"
#include "context_internal.hpp"
#include "device_common.hpp"

namespace kraken {
namespace {

constexpr uint32_t kThreads = 256;

// A sequence as the weights take it: its last rows within the window, count 0 if it is
// left out.
struct WeightRows {
  PagedSequence sequence;
  uint32_t first;  // row of the sequence
};

__device__ __forceinline__ WeightRows weight_rows(const KeyWeightsArgs& a, uint32_t sequence) {
  WeightRows r{paged_sequence(a.rows.batch, sequence, a.rows.cache.page_shift), 0u};
  if (r.sequence.length > a.stride) {
    r.sequence.count = 0;
  }
  r.first = r.sequence.count - min(r.sequence.count, a.window);
  return r;
}

template <class T>
__device__ __forceinline__ float score_of(const KeyWeightsArgs& a, const T* query,
                                          uint32_t kv_head, const int32_t* table, uint32_t key) {
  const PagedQ8Args& c = a.rows.cache;
  const int32_t page = table[key >> c.page_shift];
  if (page < 0 || (uint32_t)page >= c.pages) {
    return -INFINITY;
  }
  const size_t page_head = (size_t)page * c.kv_heads + kv_head;
  const int8_t* codes =
    c.keys + ((page_head << c.page_shift) + (key & ((1u << c.page_shift) - 1u))) * c.head_dim;
  float sum = 0.0f;
  for (uint32_t i = 0; i < c.head_dim; ++i) {
    sum = fmaf((float)query[i], (float)codes[i], sum);
  }
  return sum * (kLog2e / sqrtf((float)c.head_dim)) * c.key_scales[page_head];
}

// Each row's largest score and sum: log2 of the sum of 2^score, one workgroup a row.
template <class T>
__global__ __launch_bounds__(kThreads) void weight_row_kernel(KeyWeightsArgs a, float* logs) {
  __shared__ float s[kThreads / 64u];
  const uint32_t token = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  const uint32_t group = a.rows.heads / a.rows.cache.kv_heads, d = a.rows.cache.head_dim;
  const PagedRow row = paged_row(a.rows.batch, token, a.rows.cache.page_shift);
  if (row.sequence.count == 0) {
    return;
  }
  const uint32_t visible =
    row.sequence.length - row.sequence.count + (token - row.sequence.start) + 1u;
  const T* query = static_cast<const T*>(a.rows.query) + ((size_t)token * a.rows.heads + head) * d;
  const int32_t* table = a.rows.batch.table + (size_t)row.index * a.rows.batch.width;
  float top = kLowestMax, sum = 0.0f;
  for (uint32_t key = tid; key < visible; key += kThreads) {
    const float x = score_of(a, query, head / group, table, key);
    const float up = fmaxf(top, x);
    sum = sum * exp2f(top - up) + exp2f(x - up);
    top = up;
  }
  const float mine = halves_max(across8_max(reduce8_max(top)));
  __syncthreads();
  if ((tid & 63u) == 0) {
    s[tid >> 6] = mine;
  }
  __syncthreads();
  float most = s[0];
  for (uint32_t i = 1; i < kThreads / 64u; ++i) {
    most = fmaxf(most, s[i]);
  }
  sum = wave_sum(sum * exp2f(top - most));
  __syncthreads();
  if ((tid & 63u) == 0) {
    s[tid >> 6] = sum;
  }
  __syncthreads();
  if (tid == 0) {
    sum = 0.0f;
    for (uint32_t i = 0; i < kThreads / 64u; ++i) {
      sum += s[i];
    }
    // A row without a key gives nothing: its scores are -inf.
    logs[(size_t)token * a.rows.heads + head] = sum == 0.0f ? 0.0f : most + log2f(sum);
  }
}

// A thread a key.
template <class T>
__global__ __launch_bounds__(kThreads) void weight_key_kernel(KeyWeightsArgs a,
                                                              const float* logs) {
  const uint32_t pair = blockIdx.x, kv_heads = a.rows.cache.kv_heads;
  const uint32_t sequence = pair / kv_heads, kv_head = pair % kv_heads;
  const uint32_t group = a.rows.heads / kv_heads, d = a.rows.cache.head_dim;
  const WeightRows r = weight_rows(a, sequence);
  const PagedSequence s = r.sequence;
  const int32_t* table = a.rows.batch.table + (size_t)sequence * a.rows.batch.width;
  if (s.count == 0) {
    return;
  }
  for (uint32_t key = blockIdx.y * kThreads + threadIdx.x; key < s.length;
       key += gridDim.y * kThreads) {
    float* at = a.weights + (size_t)pair * a.row_stride + key;
    const uint32_t before = s.length - s.count;
    float sum = 0.0f;
    for (uint32_t i = r.first; i < s.count; ++i) {
      if (key > before + i) {
        continue;
      }
      for (uint32_t g = 0; g < group; ++g) {
        const size_t row = (size_t)(s.start + i) * a.rows.heads + kv_head * group + g;
        sum += exp2f(score_of(a, static_cast<const T*>(a.rows.query) + row * d, kv_head, table,
                              key) - logs[row]);
      }
    }
    *at = a.decay > 0.0f && key < before ? sum + a.decay * *at : sum;
  }
}

template <class T>
void launch_type(const KeyWeightsArgs& a, float* logs, hipStream_t stream) {
  weight_row_kernel<T><<<dim3(a.rows.batch.tokens, a.rows.heads), kThreads, 0, stream>>>(a, logs);
  const uint32_t across = std::min((a.rows.batch.max_keys + kThreads - 1u) / kThreads, 1024u);
  weight_key_kernel<T>
    <<<dim3(a.rows.batch.sequences * a.rows.cache.kv_heads, across), kThreads, 0, stream>>>(a,
                                                                                          logs);
}

}  // namespace

size_t key_weights_workspace_bytes(const KeyWeightsArgs& a, int) {
  return (size_t)a.rows.batch.tokens * a.rows.heads * sizeof(float);
}

hipError_t launch_key_weights(const KeyWeightsArgs& a, int, void* workspace, hipStream_t stream) {
  float* logs = static_cast<float*>(workspace);
  if (a.rows.f16) {
    launch_type<half_t>(a, logs, stream);
  } else {
    launch_type<float>(a, logs, stream);
  }
  return hipGetLastError();
}

}  // namespace kraken
