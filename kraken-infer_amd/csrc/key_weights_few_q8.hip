// The attention weight that cached keys receive: the sequences of few rows (the single
// tokens of a decode step).  Their keys pass through the matrix cores once, and the scores,
// 4 bytes for each row and key beside the key's own head_dim, are kept until the rows' sums
// are known.
//
// The first launch is the score half of the attention's decode kernel
// (attention_paged_q8.hip): a workgroup takes one KV head of one sequence and a run of its
// keys, its four waves 32-key steps in turn, S^T = K Q^T (16x16x32), the f32 query's two
// f16 parts in one product's columns up to 8 rows.  It leaves the scores in log2 units as
// [step][row][32] and each row's maximum and sum.  The second joins those and adds
// 2^(score - log2 of the row's sum) over the rows of each key.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "context_internal.hpp"
#include "device_common.hpp"
#include "key_weights_internal.hpp"

namespace kraken {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = 4;
constexpr uint32_t kSumKeys = 1024;  // of a workgroup of the second launch
constexpr size_t kMostBytes = size_t{1} << 30;

struct FewPlan {
  uint32_t group;      // query heads of a KV head
  uint32_t rows;       // most of a sequence
  uint32_t part_keys;  // of a workgroup of the first launch
  uint32_t parts;      // most of a sequence
  uint32_t steps;      // of 32 keys, most of a sequence
  float* scores;       // [sequences][kv_heads][steps][rows][32]
  float2* stats;       // [sequences][kv_heads][parts][rows]
};

__device__ __forceinline__ bool takes_few(uint32_t rows) { return rows != 0 && rows <= kFewRows; }

template <int D, class T, bool kStacked>
__global__ __launch_bounds__(kThreads, 3) void few_scores_kernel(KeyWeightsArgs a, FewPlan p) {
  constexpr uint32_t kRows = kStacked ? 8 : 16;
  constexpr bool kTwo = !kStacked && std::is_same<T, float>::value;
  constexpr int kLoads = D / 64;  // 16-byte loads of a key row per lane and row tile
  __shared__ float2 joined[kWaves][kRows];

  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t n = lane & 15u, g = lane >> 4;
  const uint32_t shift = a.rows.cache.page_shift, kv_heads = a.rows.cache.kv_heads;
  const uint32_t kv_head = blockIdx.x % kv_heads;
  const PagedItem found =
    paged_item(a.rows.batch, blockIdx.x / kv_heads, shift, [&](const PagedSequence& q) {
      return takes_few(counted_rows(a, q, p.group))
               ? (q.length + p.part_keys - 1u) / p.part_keys
               : 0u;
    });
  const PagedSequence s = found.sequence;
  if (s.count == 0) {
    return;
  }
  const uint32_t rows = counted_rows(a, s, p.group), part = found.item;
  const uint32_t begin = part * p.part_keys, end = min(s.length, begin + p.part_keys);
  const uint32_t steps = (end - begin + 31u) / 32u;
  const size_t pair = (size_t)found.index * kv_heads + kv_head;
  const int32_t* table = a.rows.batch.table + (size_t)found.index * a.rows.batch.width;
  auto page_of = [&](uint32_t key) {
    return table[min(key >> shift, a.rows.batch.width - 1u)];
  };
  auto first_key = [&](uint32_t step) { return begin + step * 32u; };
  // Of the lane's key rows (run n / 4 of the step's four) and of its scores' run g.
  auto place_k = [&](uint32_t step) { return first_key(step) + 8u * (n >> 2) + (n & 3u); };

  u32x4_t k[2][kLoads];
  auto load_k = [&](uint32_t step, int32_t page) {
    const uint32_t held = page >= 0 && (uint32_t)page < a.rows.cache.pages ? (uint32_t)page : 0u;
    const int8_t* at = a.rows.cache.keys +
                       ((((size_t)held * kv_heads + kv_head) << shift) +
                        (place_k(step) & ((1u << shift) - 1u))) * D + 16u * g;
#pragma unroll
    for (int i = 0; i < 2 * kLoads; ++i) {
      k[i / kLoads][i % kLoads] = __builtin_nontemporal_load(
        reinterpret_cast<const u32x4_t*>(at + i / kLoads * 4 * D + 64 * (i % kLoads)));
    }
  };
  float key_scale = 0.0f;
  bool inside = false;
  auto load_scale = [&](int32_t page) {
    inside = page >= 0 && (uint32_t)page < a.rows.cache.pages;
    key_scale = a.rows.cache.key_scales[(size_t)(inside ? page : 0) * kv_heads + kv_head];
  };
  int32_t page_k = page_of(place_k(wave)), page_s = page_of(first_key(wave) + 8u * g);

  // This lane's query row and the keys that it sees.
  const uint32_t row = kStacked ? n & 7u : n;
  const bool real = row < rows;
  const uint32_t token = s.count - min(s.count, a.window) + (real ? row / p.group : 0u);
  const uint32_t visible = s.length - s.count + token + 1u;
  const T* query = static_cast<const T*>(a.rows.query) +
                   ((size_t)(s.start + token) * a.rows.heads + kv_head * p.group +
                    (real ? row % p.group : 0u)) * D + 16u * g;
  half8_t q_hi[2 * kLoads], q_lo[kTwo ? 2 * kLoads : 1];
  float row_factor;
  {
    float x[kLoads][16], largest = 0.0f;
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        load4(query + 64 * c + 4 * i, &x[c][4 * i]);
      }
    }
    if (wave < steps) {
      load_k(wave, page_k);
      load_scale(page_s);
    }
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[c][i] = real ? x[c][i] : 0.0f;
        largest = fmaxf(largest, fabsf(x[c][i]));
      }
    }
    largest = xor32_max(xor16_max(largest));
    const int e = query_exponent(largest);
    // 1 / sqrt(D) in log2 units, over the row's power of two.
    row_factor = ldexpf(kLog2e / (D == 64 ? 8.0f : D == 256 ? 16.0f : 11.313708498984761f), -e);
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        half8_t hi, lo;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          half2_t u, w;
          split_pair(ldexpf(x[c][8 * h + i], e), ldexpf(x[c][8 * h + i + 1], e), u, w);
          hi[i] = u[0];
          hi[i + 1] = u[1];
          lo[i] = w[0];
          lo[i + 1] = w[1];
        }
        if constexpr (kStacked) {
          q_hi[2 * c + h] = n < 8u ? hi : lo;
        } else {
          q_hi[2 * c + h] = hi;
          if constexpr (kTwo) {
            q_lo[2 * c + h] = lo;
          }
        }
      }
    }
  }

  float top = kLowestMax, sum = 0.0f;
  for (uint32_t step = wave; step < steps; step += kWaves) {
    const uint32_t next = step + kWaves;
    if (next < steps) {
      page_k = page_of(place_k(next));
      page_s = page_of(first_key(next) + 8u * g);
    }
    float4_t score[2] = {float4_t{0.0f, 0.0f, 0.0f, 0.0f}, float4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
          const half8_t x = codes_to_f16(k[tile][c][2 * h], k[tile][c][2 * h + 1]);
          score[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q_hi[2 * c + h], score[tile],
                                                               0, 0, 0);
          if constexpr (kTwo) {
            score[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q_lo[2 * c + h],
                                                                 score[tile], 0, 0, 0);
          }
        }
      }
    }
    const float factor = inside ? row_factor * key_scale : 0.0f;
    const float offset = inside ? 0.0f : -INFINITY;
    if (next < steps) {
      load_k(next, page_k);
      load_scale(page_s);
    }
    const uint32_t key = first_key(step) + 8u * g;
    float w[8], largest = kLowestMax;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = score[i / 4][i % 4];
      if constexpr (kStacked) {
        x += dpp<kDppRowRor8>(x);
      }
      w[i] = fmaf(x, factor, offset);
      w[i] = key + i < visible ? w[i] : -INFINITY;
      largest = fmaxf(largest, w[i]);
    }
    if (real && n < kRows) {
      float* at = p.scores + ((pair * p.steps + begin / 32u + step) * p.rows + row) * 32u + 8u * g;
      *reinterpret_cast<float4_t*>(at) = float4_t{w[0], w[1], w[2], w[3]};
      *reinterpret_cast<float4_t*>(at + 4) = float4_t{w[4], w[5], w[6], w[7]};
    }
    const float up = fmaxf(top, largest);
    sum *= fast_exp2(top - up);
    top = up;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum += fast_exp2(w[i] - top);
    }
  }
  // The four runs of a step, then the waves.
  {
    const float up = xor32_max(xor16_max(top));
    sum = xor32_sum(xor16_sum(sum * fast_exp2(top - up)));
    top = up;
  }
  if (g == 0 && n < kRows) {
    joined[wave][n] = make_float2(top, sum);
  }
  __syncthreads();
  if (threadIdx.x < rows) {
    float2 all = joined[0][threadIdx.x];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) {
      const float2 x = joined[w][threadIdx.x];
      const float up = fmaxf(all.x, x.x);
      all.y = all.y * fast_exp2(all.x - up) + x.y * fast_exp2(x.x - up);
      all.x = up;
    }
    p.stats[(pair * p.parts + part) * p.rows + threadIdx.x] = all;
  }
}

__global__ __launch_bounds__(kThreads) void few_sums_kernel(KeyWeightsArgs a, FewPlan p) {
  __shared__ float logs[kFewRows];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t kv_heads = a.rows.cache.kv_heads, kv_head = blockIdx.x % kv_heads;
  const PagedItem found = paged_item(
    a.rows.batch, blockIdx.x / kv_heads, a.rows.cache.page_shift, [&](const PagedSequence& q) {
      return takes_few(counted_rows(a, q, p.group)) ? (q.length + kSumKeys - 1u) / kSumKeys : 0u;
    });
  const PagedSequence s = found.sequence;
  if (s.count == 0) {
    return;
  }
  const uint32_t rows = counted_rows(a, s, p.group);
  const size_t pair = (size_t)found.index * kv_heads + kv_head;
  const uint32_t parts = (s.length + p.part_keys - 1u) / p.part_keys;
  // log2 of each row's sum; infinity, which makes its weights zero, without any key.
  for (uint32_t row = wave; row < rows; row += kWaves) {
    float top = kLowestMax, sum = 0.0f;
    for (uint32_t i = lane; i < parts; i += 64u) {
      const float2 x = p.stats[(pair * p.parts + i) * p.rows + row];
      const float up = fmaxf(top, x.x);
      sum = sum * fast_exp2(top - up) + x.y * fast_exp2(x.x - up);
      top = up;
    }
    const float up = halves_max(across8_max(reduce8_max(top)));
    sum = wave_sum(sum * fast_exp2(top - up));
    if (lane == 0) {
      logs[row] = sum == 0.0f ? INFINITY : up + log2f(sum);
    }
  }
  __syncthreads();
  const uint32_t before = s.length - s.count;
#pragma unroll
  for (uint32_t i = 0; i < kSumKeys / kThreads; ++i) {
    const uint32_t key = found.item * kSumKeys + i * kThreads + threadIdx.x;
    if (key < s.length) {
      const float* scores =
        p.scores + (pair * p.steps + key / 32u) * p.rows * 32u + key % 32u;
      float sum = 0.0f;
      for (uint32_t row = 0; row < rows; ++row) {
        sum += fast_exp2(scores[row * 32u] - logs[row]);
      }
      float* at = a.weights + pair * a.row_stride + key;
      *at = sum + decayed_weight(a, at, key < before);
    }
  }
}

FewPlan plan_of(const KeyWeightsArgs& a, int cu_count, size_t& bytes, void* workspace) {
  FewPlan p{};
  p.group = a.rows.heads / a.rows.cache.kv_heads;
  const uint64_t rows = (uint64_t)std::min(a.window, a.rows.batch.max_query) * p.group;
  p.rows = (uint32_t)std::min<uint64_t>(rows, kFewRows);
  const uint64_t pairs = (uint64_t)a.rows.batch.sequences * a.rows.cache.kv_heads;
  const uint32_t keys = longest_length(a);
  p.steps = (keys + 31u) / 32u;
  // Parts as the attention's decode kernel has them.
  const uint64_t most = 11u * (uint64_t)cu_count;
  uint64_t per = (pairs * keys + most - 1u) / most;
  per = std::min<uint64_t>((std::max<uint64_t>(per, 128u) + 127u) / 128u * 128u, 4096u);
  p.part_keys = (uint32_t)per;
  p.parts = (keys + p.part_keys - 1u) / p.part_keys;
  const double scores = (double)pairs * p.steps * p.rows * 128.0;
  const double stats = (double)pairs * p.parts * p.rows * sizeof(float2);
  // (A single sequence of more rows is not worth a second pair of launches for where it brings
  // fewer: 8192 keys, 128 rows 33.9 us with them, 29.8 without.)
  if (p.group > kFewRows || scores + stats > (double)kMostBytes ||
      (a.rows.batch.sequences == 1u && rows > kFewRows)) {
    bytes = 0;
    return p;
  }
  p.scores = static_cast<float*>(workspace);
  p.stats = reinterpret_cast<float2*>(p.scores + pairs * p.steps * p.rows * 32u);
  bytes = (size_t)(scores + stats);
  return p;
}

template <int D, class T>
void launch_for(const KeyWeightsArgs& a, const FewPlan& p, hipStream_t stream) {
  const uint32_t pairs = a.rows.batch.sequences * a.rows.cache.kv_heads;
  if (p.rows <= 8u) {
    few_scores_kernel<D, T, true><<<dim3(pairs * p.parts), kThreads, 0, stream>>>(a, p);
  } else {
    few_scores_kernel<D, T, false><<<dim3(pairs * p.parts), kThreads, 0, stream>>>(a, p);
  }
  const uint32_t blocks = (p.steps * 32u + kSumKeys - 1u) / kSumKeys;
  few_sums_kernel<<<dim3(pairs * blocks), kThreads, 0, stream>>>(a, p);
}

template <class T>
void launch_type(const KeyWeightsArgs& a, const FewPlan& p, hipStream_t stream) {
  if (a.rows.cache.head_dim == 256u) {
    launch_for<256, T>(a, p, stream);
  } else if (a.rows.cache.head_dim == 128u) {
    launch_for<128, T>(a, p, stream);
  } else {
    launch_for<64, T>(a, p, stream);
  }
}

}  // namespace

size_t few_weights_bytes(const KeyWeightsArgs& a, int cu_count) {
  size_t bytes;
  plan_of(a, cu_count, bytes, nullptr);
  return bytes;
}

void launch_few_weights(const KeyWeightsArgs& a, int cu_count, void* workspace,
                        hipStream_t stream) {
  size_t bytes;
  const FewPlan p = plan_of(a, cu_count, bytes, workspace);
  if (a.rows.f16) {
    launch_type<half_t>(a, p, stream);
  } else {
    launch_type<float>(a, p, stream);
  }
}

}  // namespace kraken
