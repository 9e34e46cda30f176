// Eviction from a paged 8-bit cache: which positions of each sequence and KV head stay,
// and their move into fresh pages.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "context_internal.hpp"
#include "device_common.hpp"
#include "paged_q8_internal.hpp"
#include "row_order.hpp"

namespace kraken {
namespace {

constexpr uint32_t kSelectThreads = 1024;
constexpr uint32_t kSelectWaves = kSelectThreads / 64u;
constexpr uint32_t kGatherThreads = 256;

// Sum over the workgroup's threads before this one, and the whole.
__device__ __forceinline__ uint32_t block_before(uint32_t x, uint32_t& all, uint32_t* s) {
  const uint32_t upto = wave_scan(x, Sum{});
  __syncthreads();
  if ((threadIdx.x & 63u) == 63u) {
    s[threadIdx.x >> 6] = upto;
  }
  __syncthreads();
  uint32_t before = 0;
  all = 0;
  for (uint32_t i = 0; i < kSelectWaves; ++i) {
    before += i < threadIdx.x >> 6 ? s[i] : 0u;
    all += s[i];
  }
  return before + upto - x;
}

// One workgroup a sequence and KV head: the least key that is kept, found eight bits at a
// time from the top by counts, then the kept positions in order, of those equal to it the
// first few.
__global__ __launch_bounds__(kSelectThreads) void select_keys_kernel(SelectKeysArgs a) {
  __shared__ uint32_t bins[256], s[kSelectWaves];
  __shared__ uint32_t digit, above;
  const uint32_t pair = blockIdx.x, sequence = pair / a.kv_heads, tid = threadIdx.x;
  const uint32_t length = a.lengths[sequence];
  if (length > a.max_keys) {
    return;
  }
  const uint32_t k = min(a.keep[sequence], length);
  if (k > a.kept_stride) {
    return;
  }
  if (pair % a.kv_heads == 0 && tid == 0) {
    a.kept_lengths[sequence] = k;
  }
  // Positions [0, first) and [end, length) are kept, and `most` of those between.
  const uint32_t last = min(a.last, k), first = min(min(a.first, k - last), length - last);
  const uint32_t end = length - last;
  const uint32_t most = k - last - first;
  const float* weights = a.weights + (size_t)pair * a.weight_stride;
  int32_t* kept = a.kept + (size_t)pair * a.kept_stride;
  for (uint32_t i = tid; i < first; i += kSelectThreads) {
    kept[i] = (int32_t)i;
  }
  for (uint32_t i = tid; i < last; i += kSelectThreads) {
    kept[k - last + i] = (int32_t)(end + i);
  }
  if (most == 0) {
    return;
  }
  uint32_t least = 0, want = most;  // `want` of those whose high digits are those of `least`
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256u) {
      bins[tid] = 0;
    }
    __syncthreads();
    for (uint32_t i = first + tid; i < end; i += kSelectThreads) {
      const uint32_t key = key_of(weights[i]);
      if (shift == 24 || key >> (shift + 8) == least >> (shift + 8)) {
        atomicAdd(&bins[key >> shift & 255u], 1u);
      }
    }
    __syncthreads();
    // From the largest digit down.
    const uint32_t mine = tid < 256u ? bins[255u - tid] : 0u;
    uint32_t all;
    const uint32_t before = block_before(mine, all, s);
    if (before < want && want <= before + mine) {
      digit = 255u - tid;
      above = before;
    }
    __syncthreads();
    least |= digit << shift;
    want -= above;
  }
  uint32_t at = first, ties = 0;
  for (uint32_t base = first; base < end; base += kSelectThreads) {
    const uint32_t i = base + tid;
    const uint32_t key = i < end ? key_of(weights[i]) : 0u;
    const bool equal = i < end && key == least;
    uint32_t all;
    const uint32_t tie = ties + block_before(equal ? 1u : 0u, all, s);
    ties += all;
    const bool keep = i < end && (key > least || (equal && tie < want));
    const uint32_t place = at + block_before(keep ? 1u : 0u, all, s);
    at += all;
    if (keep) {
      kept[place] = (int32_t)i;
    }
  }
}

// A kept token's place in the source pages; page -1 where there is none.
struct Source {
  int32_t page;
  uint32_t slot;
};

__device__ __forceinline__ Source source_of(const GatherPagesArgs& a, uint32_t sequence,
                                            int32_t position) {
  const uint32_t shift = a.cache.page_shift;
  if (position < 0 || (uint32_t)position >> shift >= a.width) {
    return {-1, 0u};
  }
  const int32_t page = a.table[(size_t)sequence * a.width + ((uint32_t)position >> shift)];
  return {page >= 0 && (uint32_t)page < a.cache.pages ? page : -1,
          (uint32_t)position & ((1u << shift) - 1u)};
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// One workgroup a target page and KV head.
__global__ __launch_bounds__(kGatherThreads) void gather_pages_kernel(GatherPagesArgs a,
                                                                      uint64_t items) {
  __shared__ Source sources[128];
  __shared__ float scales[2][128], ratio[2][128];
  __shared__ float page_scale[2];
  const PagedQ8Args& c = a.cache;
  const uint32_t tid = threadIdx.x, page_tokens = 1u << c.page_shift, d = c.head_dim;
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    __syncthreads();
    const uint32_t head = (uint32_t)(item % c.kv_heads);
    const uint64_t rest = item / c.kv_heads;
    const uint32_t p = (uint32_t)(rest % a.target_width);
    const uint32_t sequence = (uint32_t)(rest / a.target_width);
    const uint64_t pair = (uint64_t)sequence * c.kv_heads + head;
    const uint32_t n = a.kept_lengths[sequence];
    const uint64_t begin = (uint64_t)p << c.page_shift;
    if (begin >= n || n > a.kept_stride || n > (uint64_t)a.target_width << c.page_shift ||
        (a.weights != nullptr && n > a.weight_stride)) {
      continue;
    }
    if (tid < page_tokens) {
      Source from{-1, 0u};
      if (begin + tid < n) {
        const int32_t position = a.kept[pair * a.kept_stride + begin + tid];
        from = source_of(a, sequence, position);
        if (a.weights != nullptr) {
          const float* weights = a.weights + pair * a.weight_stride;
          a.weights_output[pair * a.weight_stride + begin + tid] =
            position >= 0 && (uint32_t)position < a.weight_stride ? weights[position] : 0.0f;
        }
      }
      sources[tid] = from;
      const size_t at = (size_t)max(from.page, 0) * c.kv_heads + head;
      scales[0][tid] = from.page >= 0 ? c.key_scales[at] : 0.0f;
      scales[1][tid] = from.page >= 0 ? c.value_scales[at] : 0.0f;
    }
    __syncthreads();
    const int32_t target = a.target_table[(size_t)sequence * a.target_width + p];
    if (target < 0 || (uint32_t)target >= c.pages) {
      continue;
    }
    const size_t page_head = (size_t)target * c.kv_heads + head;
    if (tid < 2u) {
      float most = 0.0f;
      bool all = true;
      for (uint32_t i = 0; i < page_tokens; ++i) {
        most = fmaxf(most, scales[tid][i]);
        all = all && finite(scales[tid][i]);
      }
      page_scale[tid] = all ? most : NAN;
      (tid == 0 ? c.key_scales : c.value_scales)[page_head] = page_scale[tid];
    }
    __syncthreads();
    if (tid < page_tokens) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // Of a NaN page, and of equal scales (zeros too), the codes stay.
        const float to = page_scale[i], from = scales[i][tid];
        ratio[i][tid] = from == to || !finite(to) ? 1.0f : from / to;
      }
    }
    __syncthreads();
    int8_t* keys = c.keys + (page_head << c.page_shift) * d;
    int8_t* values = c.values + (page_head << c.page_shift) * d;
    for (uint32_t e = tid; e < page_tokens * d; e += kGatherThreads) {
      const uint32_t t = e / d, dim = e % d;
      const Source from = sources[t];
      int key = 0, value = 0;
      if (from.page >= 0) {
        const size_t base = (((size_t)from.page * c.kv_heads + head) << c.page_shift) * d;
        key = c.keys[base + (size_t)from.slot * d + dim];
        value = c.values[base + ((size_t)(from.slot / 8u) * d + dim) * 8u + from.slot % 8u];
      }
      keys[e] = (int8_t)rintf((float)key * ratio[0][t]);
      values[((size_t)(t / 8u) * d + dim) * 8u + t % 8u] =
        (int8_t)rintf((float)value * ratio[1][t]);
    }
  }
}

}  // namespace

hipError_t launch_select_keys(const SelectKeysArgs& a, hipStream_t stream) {
  select_keys_kernel<<<dim3(a.sequences * a.kv_heads), kSelectThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_gather_pages(const GatherPagesArgs& a, hipStream_t stream) {
  const uint64_t items = (uint64_t)a.sequences * a.cache.kv_heads * a.target_width;
  const uint32_t blocks = (uint32_t)std::min<uint64_t>(items, uint64_t{1} << 20);
  gather_pages_kernel<<<dim3(blocks), kGatherThreads, 0, stream>>>(a, items);
  return hipGetLastError();
}

}  // namespace kraken
