// One token a row from logits, with temperature, top-k, top-p and min-p, by a given
// uniform number.
//
// Every filter keeps a prefix of the order of falling logits, so what is kept is a
// threshold: the logits above it and, of those equal to it, the first few by index.
// Logits are ordered by 32-bit keys.  A weight w = exp((l - max) / T) is formed in 64
// bits and held as an integer of 2^-shift, with room for `size` of the largest: the
// sums are exact whatever their order, so that atomics give one result, and close
// enough to the real numbers (3e-11 of the sum over 250000 tokens) that a cut or a
// draw falls on their side of a border.
//
// One workgroup per row: the threshold by radix selection over 8-bit digits of the
// key, by counts for top-k and by weights for top-p, then the draw by a scan in order
// of index.
#include <hip/hip_runtime.h>

#include "context_internal.hpp"
#include "device_common.hpp"
#include "paged_q8_internal.hpp"

namespace kraken {
namespace {

constexpr uint32_t kThreads = 1024;

// Keys order as the logits do; 0 for NaN, which is below -inf's, and -0 as +0.
__device__ __forceinline__ uint32_t key_of(float logit) {
  if (logit != logit) {
    return 0u;
  }
  const uint32_t bits = __float_as_uint(logit + 0.0f);
  return bits ^ ((bits >> 31) != 0u ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) != 0u ? 0x80000000u : 0xffffffffu));
}

constexpr uint32_t kMinusInfKey = 0x007fffffu;

// What a row is drawn by.
struct RowRule {
  bool greedy;
  double inverse_temperature, top_p, min_p, uniform;
  uint32_t top_k;  // 0: all
};

__device__ __forceinline__ RowRule row_rule(const SampleArgs& a, uint32_t row) {
  RowRule r;
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  r.greedy = !(t > 0.0f);
  r.inverse_temperature = 1.0 / (double)t;
  const int32_t k = a.top_k != nullptr ? a.top_k[row] : 0;
  r.top_k = k > 0 && (uint32_t)k < a.size ? (uint32_t)k : 0u;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  r.top_p = p < 1.0f ? (double)p : 1.0;  // NaN: 1
  const float m = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  r.min_p = m > 0.0f ? (double)m : 0.0;  // NaN: 0
  const float u = a.uniforms[row];
  r.uniform = u > 0.0f ? (u < 1.0f ? (double)u : 1.0) : 0.0;
  return r;
}

// The weight of a key; `top` is the largest.
__device__ __forceinline__ double weight_of(uint32_t key, uint32_t top, double inverse) {
  if (key == top) {
    return 1.0;
  }
  if (key <= kMinusInfKey) {
    return 0.0;
  }
  return exp(((double)logit_of(key) - (double)logit_of(top)) * inverse);
}

__device__ __forceinline__ uint64_t fixed(double w, int shift) {
  return (uint64_t)__double2ll_rn(ldexp(w, shift));
}

struct Scratch {
  uint64_t sums[256];
  uint32_t counts[256];
  uint64_t wave_sum[16];
  uint32_t wave_count[16];
  uint64_t found_sum;
  uint32_t found, found_count;
};

__device__ __forceinline__ uint64_t block_sum(uint64_t x, Scratch& s) {
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    x += (uint64_t)__shfl_xor((long long)x, step, 64);
  }
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) {
    s.wave_sum[threadIdx.x >> 6] = x;
  }
  __syncthreads();
  uint64_t all = 0;
  for (uint32_t i = 0; i < kThreads / 64u; ++i) {
    all += s.wave_sum[i];
  }
  return all;
}

// Exclusive prefix sums of a (weight, count) pair over the workgroup, and the totals.
__device__ __forceinline__ void block_scan(uint64_t& x, uint32_t& n, uint64_t& all, uint32_t& all_n,
                                           Scratch& s) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint64_t own = x;
  const uint32_t own_n = n;
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const uint64_t y = (uint64_t)__shfl_up((long long)x, step, 64);
    const uint32_t m = (uint32_t)__shfl_up((int)n, step, 64);
    if (lane >= (uint32_t)step) {
      x += y;
      n += m;
    }
  }
  __syncthreads();
  if (lane == 63u) {
    s.wave_sum[wave] = x;
    s.wave_count[wave] = n;
  }
  __syncthreads();
  all = 0;
  all_n = 0;
  uint64_t before = 0;
  uint32_t before_n = 0;
  for (uint32_t i = 0; i < kThreads / 64u; ++i) {
    before += i < wave ? s.wave_sum[i] : 0u;
    before_n += i < wave ? s.wave_count[i] : 0u;
    all += s.wave_sum[i];
    all_n += s.wave_count[i];
  }
  x = x - own + before;
  n = n - own_n + before_n;
}

// The kept set: keys above `key`, and the first `ties` by index of those equal to it.
struct Cut {
  uint32_t key, ties;
};

// Radix selection over the row.  by_weight false: the key of rank `count`, ties such
// that `count` keys are kept.  by_weight true: among the keys that `within` keeps, the
// lowest one before which less than `target` lies, ties likewise; at least one.
__device__ Cut select_cut(const float* logits, uint32_t size, uint32_t top, double inverse, int shift,
                          bool by_weight, uint32_t count, double target, Cut within, Scratch& s) {
  uint32_t prefix = 0;
  uint64_t above = 0;    // weight of the keys above the prefix
  uint32_t above_n = 0;  // and their number
  for (int level = 0; level < 4; ++level) {
    const int at = 24 - 8 * level;
    __syncthreads();
    if (threadIdx.x < 256u) {
      s.sums[threadIdx.x] = 0;
      s.counts[threadIdx.x] = 0;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
      const uint32_t key = key_of(logits[i]);
      if (level != 0 && (key >> (at + 8)) != prefix) {
        continue;
      }
      const uint32_t digit = (key >> at) & 255u;
      if (!by_weight) {
        atomicAdd(&s.counts[digit], 1u);
      } else if (key > within.key) {
        atomicAdd((unsigned long long*)&s.sums[digit], fixed(weight_of(key, top, inverse), shift));
        atomicAdd(&s.counts[digit], 1u);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      if (by_weight && within.ties != 0 && (level == 0 || (within.key >> (at + 8)) == prefix)) {
        const uint32_t digit = (within.key >> at) & 255u;
        s.sums[digit] += within.ties * fixed(weight_of(within.key, top, inverse), shift);
        s.counts[digit] += within.ties;
      }
      uint64_t sum = above;
      uint32_t n = above_n, digit = 0;
      uint64_t found_sum = sum;
      uint32_t found_n = n;
      bool any = false;
      for (int d = 255; d >= 0; --d) {
        if (s.counts[d] == 0) {
          continue;
        }
        const bool reaches = by_weight ? !any || (double)sum < target : n < count;
        if (!reaches) {
          break;
        }
        any = true;
        digit = (uint32_t)d;
        found_sum = sum;
        found_n = n;
        sum += s.sums[d];
        n += s.counts[d];
      }
      s.found = digit;
      s.found_sum = found_sum;
      s.found_count = found_n;
      s.counts[0] = s.counts[digit];
    }
    __syncthreads();
    prefix = prefix << 8 | s.found;
    above = s.found_sum;
    above_n = s.found_count;
  }
  const uint32_t here = s.counts[0];  // keys equal to the prefix, of those in question
  Cut cut{prefix, 0};
  if (!by_weight) {
    cut.ties = count - above_n;
  } else {
    const uint64_t w = fixed(weight_of(prefix, top, inverse), shift);
    // The i-th tie is kept where above + i w < target.
    uint32_t ties = here;
    if (w != 0) {
      const double need = ceil((target - (double)above) / (double)w);
      ties = need < (double)here ? (need > 1.0 ? (uint32_t)need : 1u) : here;
    }
    cut.ties = ties;
  }
  return cut;
}

__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a, int shift) {
  __shared__ Scratch s;
  __shared__ uint32_t wave_top[16], wave_index[16];
  const uint32_t row = blockIdx.x, size = a.size;
  const float* logits = a.logits + (size_t)row * a.row_stride;
  const RowRule rule = row_rule(a, row);

  // The largest key and its first index.
  uint32_t top = 0, index = size;
  for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
    const uint32_t key = key_of(logits[i]);
    if (key > top) {
      top = key;
      index = i;
    }
  }
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const uint32_t k = (uint32_t)__shfl_xor((int)top, step, 64);
    const uint32_t j = (uint32_t)__shfl_xor((int)index, step, 64);
    index = k > top || (k == top && j < index) ? j : index;
    top = max(top, k);
  }
  if ((threadIdx.x & 63u) == 0) {
    wave_top[threadIdx.x >> 6] = top;
    wave_index[threadIdx.x >> 6] = index;
  }
  __syncthreads();
  for (uint32_t i = 0; i < kThreads / 64u; ++i) {
    const uint32_t k = wave_top[i], j = wave_index[i];
    index = k > top || (k == top && j < index) ? j : index;
    top = max(top, k);
  }
  if (rule.greedy || rule.min_p > 1.0 || top <= kMinusInfKey) {
    if (threadIdx.x == 0) {
      a.tokens[row] = (int32_t)index;
      if (a.probabilities != nullptr) {
        a.probabilities[row] = top > kMinusInfKey ? 1.0f : 0.0f;
      }
    }
    return;
  }

  const double inverse = rule.inverse_temperature;
  Cut cut{0u, 0u};  // every key but NaN's
  if (rule.top_k != 0) {
    cut = select_cut(logits, size, top, inverse, shift, false, rule.top_k, 0.0, cut, s);
  }
  if (rule.top_p < 1.0) {
    uint64_t sum = 0;
    for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
      const uint32_t key = key_of(logits[i]);
      sum += key > cut.key ? fixed(weight_of(key, top, inverse), shift) : 0u;
    }
    sum = block_sum(sum, s);
    sum += cut.ties * fixed(weight_of(cut.key, top, inverse), shift);
    cut = select_cut(logits, size, top, inverse, shift, true, 0u, rule.top_p * (double)sum, cut, s);
  }

  // The whole sum of what is kept, then the tile in which the draw falls.
  const uint32_t per = 4u * kThreads;
  auto kept_weight = [&](uint32_t key) {
    if (key < cut.key || key == 0u) {
      return (uint64_t)0;
    }
    const double w = weight_of(key, top, inverse);
    return w >= rule.min_p ? fixed(w, shift) : (uint64_t)0;
  };
  const uint64_t tie_weight = kept_weight(cut.key);
  uint64_t sum = 0;
  for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
    const uint32_t key = key_of(logits[i]);
    sum += key > cut.key ? kept_weight(key) : 0u;
  }
  const uint64_t total = block_sum(sum, s) + cut.ties * tie_weight;
  const double target = rule.uniform * (double)total;
  uint64_t before = 0;
  uint32_t ties_before = 0;
  __shared__ uint32_t chosen, last_kept;
  if (threadIdx.x == 0) {
    chosen = size;
    last_kept = index;
  }
  for (uint32_t base = 0; base < size; base += per) {
    uint64_t w[4], x = 0;
    uint32_t tie[4], n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t i = base + 4u * threadIdx.x + k;
      const uint32_t key = i < size ? key_of(logits[i]) : 0u;
      tie[k] = i < size && key == cut.key ? 1u : 0u;
      w[k] = i < size && key > cut.key ? kept_weight(key) : 0u;
      x += w[k];
      n += tie[k];
    }
    uint64_t all;
    uint32_t all_n;
    block_scan(x, n, all, all_n, s);
    // Ties before this thread's run, and how many of them are kept.
    uint64_t at = before + x + (uint64_t)(min(ties_before + n, cut.ties) -
                                          min(ties_before, cut.ties)) * tie_weight;
    uint32_t seen = ties_before + n;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (tie[k] != 0u) {
        w[k] = seen < cut.ties ? tie_weight : 0u;
        ++seen;
      }
      at += w[k];
      if (w[k] != 0u) {
        const uint32_t i = base + 4u * threadIdx.x + k;
        if ((double)at > target) {
          atomicMin(&chosen, i);
        } else {
          atomicMax(&last_kept, i);
        }
      }
    }
    before += all + (uint64_t)(min(ties_before + all_n, cut.ties) - min(ties_before, cut.ties)) *
                      tie_weight;
    ties_before += all_n;
    __syncthreads();
    if (chosen != size) {
      break;  // uniform: read after the barrier, written before it
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const uint32_t token = chosen != size ? chosen : last_kept;
    a.tokens[row] = (int32_t)token;
    if (a.probabilities != nullptr) {
      const double w = weight_of(key_of(logits[token]), top, inverse);
      a.probabilities[row] = (float)(ldexp(w, shift) / (double)total);
    }
  }
}

}  // namespace

size_t sample_workspace_bytes(const SampleArgs&) { return 0; }

hipError_t launch_sample(const SampleArgs& a, void*, hipStream_t stream) {
  int shift = 62;
  for (uint64_t n = a.size; n > 1u; n = (n + 1u) / 2u) {
    --shift;
  }
  sample_row_kernel<<<dim3(a.rows), kThreads, 0, stream>>>(a, shift);
  return hipGetLastError();
}

}  // namespace kraken
