// One token a row from logits, with temperature, top-k, top-p and min-p, by a given
// uniform number.
//
// Every filter keeps a prefix of the order of falling logits, so what is kept is a
// threshold: the logits above it and, of those equal to it, the first few by index.
// Nothing is sorted.  Logits are ordered by 32-bit keys.  A weight w = exp((l - max) / T)
// is formed in 64 bits and held as an integer of 2^-shift, with room for `size` of the
// largest: the sums are exact whatever their order, so that atomics give one result, and
// close enough to the real numbers (6e-11 of the largest weight over 250000 tokens) that
// a cut or a draw falls on their side of a border.
//
// Four launches, the first three with a workgroup for each chunk of a row:
//   top     the largest key of the chunk and its first index
//   bins    the row's histogram over 1/8 octaves of weight: how many and how much, and
//           each chunk's own weights by bin
//   gather  the histogram says which bins a threshold can lie in (one, or a few where
//           top-p depends on a top-k that is not resolved yet): their elements go to a
//           list, and what lies above them is summed by chunk from the chunk's bins
//   draw    one workgroup a row: the threshold by radix selection in the list, then the
//           chunk in which the draw falls, and the token by a scan of that chunk alone.
// So a row is read three times, from memory once (the rest from the caches), and
// exponentials are formed once.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "context_internal.hpp"
#include "device_common.hpp"
#include "paged_q8_internal.hpp"

namespace kraken {
namespace {

constexpr uint32_t kThreads = 256;       // of the chunk kernels
constexpr uint32_t kDrawThreads = 1024;  // of the draw
constexpr uint32_t kBins = 512;          // 1/8 octave each; the last takes all below 2^-63
constexpr uint32_t kMaxChunks = 4096;
constexpr uint32_t kMinusInfKey = 0x007fffffu;

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

// No draw: the first of the largest logits.
__device__ __forceinline__ bool takes_top(const RowRule& rule, uint32_t top) {
  return rule.greedy || rule.min_p > 1.0 || top <= kMinusInfKey;
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

// The bin of a key: falling weights fall into rising bins (each step of it is
// monotone).  `scale` is 8 log2(e) / T.
__device__ __forceinline__ uint32_t bin_of(uint32_t key, uint32_t top, float scale) {
  const float z = (logit_of(top) - logit_of(key)) * scale;
  return key == top ? 0u : (uint32_t)fminf(z, (float)(kBins - 1u));  // NaN: the last
}

// A row's place in the workspace.
struct RowWork {
  uint64_t* bin_weight;   // [kBins]
  uint32_t* bin_count;    // [kBins]
  uint32_t* listed;       // number of entries of the list
  uint64_t* chunk_weight; // [chunks]: of what is kept whatever the threshold
  uint64_t* chunk_top;    // [chunks]: key << 32 | ~index
  uint64_t* chunk_bins;   // [chunks][kBins]
  uint64_t* list;         // [size]: key << 32 | index
};

struct Plan {
  uint32_t chunk, chunks;  // logits per chunk, chunks per row
  int shift;
  uint64_t* work;
  size_t row_words;  // 8-byte words of the workspace per row
};

__host__ __device__ __forceinline__ size_t words_per_row(uint32_t chunks, uint32_t size) {
  return kBins + kBins / 2u + 1u + (size_t)chunks * (2u + kBins) + size;
}

__device__ __forceinline__ RowWork row_work(const Plan& p, uint32_t row) {
  RowWork w;
  w.bin_weight = p.work + (size_t)row * p.row_words;
  w.bin_count = reinterpret_cast<uint32_t*>(w.bin_weight + kBins);
  w.listed = w.bin_count + kBins;
  w.chunk_weight = w.bin_weight + kBins + kBins / 2u + 1u;
  w.chunk_top = w.chunk_weight + p.chunks;
  w.chunk_bins = w.chunk_top + p.chunks;
  w.list = w.chunk_bins + (size_t)p.chunks * kBins;
  return w;
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t x) {
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const uint64_t y = (uint64_t)__shfl_xor((long long)x, step, 64);
    x = y > x ? y : x;
  }
  return x;
}

// Largest over the workgroup of kWaves waves.
template <uint32_t kWaves>
__device__ __forceinline__ uint64_t block_max(uint64_t x, uint64_t* s) {
  x = wave_max_u64(x);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) {
    s[threadIdx.x >> 6] = x;
  }
  __syncthreads();
  x = s[0];
  for (uint32_t i = 1; i < kWaves; ++i) {
    x = s[i] > x ? s[i] : x;
  }
  return x;
}

// Exclusive prefix sums of (weight, count) pairs over the workgroup, and the totals.
template <uint32_t kWaves>
__device__ __forceinline__ void block_scan(uint64_t& x, uint32_t& n, uint64_t& all, uint32_t& all_n,
                                           uint64_t* sums, uint32_t* counts) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint64_t own = x;
  const uint32_t own_n = n;
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const uint64_t y = (uint64_t)__shfl_up((long long)x, step, 64);
    const uint32_t m = (uint32_t)__shfl_up((int)n, step, 64);
    x += lane >= (uint32_t)step ? y : 0u;
    n += lane >= (uint32_t)step ? m : 0u;
  }
  __syncthreads();
  if (lane == 63u) {
    sums[wave] = x;
    counts[wave] = n;
  }
  __syncthreads();
  all = 0;
  all_n = 0;
  uint64_t before = 0;
  uint32_t before_n = 0;
#pragma unroll
  for (uint32_t i = 0; i < kWaves; ++i) {
    before += i < wave ? sums[i] : 0u;
    before_n += i < wave ? counts[i] : 0u;
    all += sums[i];
    all_n += counts[i];
  }
  x = x - own + before;
  n = n - own_n + before_n;
}

template <uint32_t kWaves>
__device__ __forceinline__ uint64_t block_sum(uint64_t x, uint64_t* s) {
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    x += (uint64_t)__shfl_xor((long long)x, step, 64);
  }
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) {
    s[threadIdx.x >> 6] = x;
  }
  __syncthreads();
  x = 0;
  for (uint32_t i = 0; i < kWaves; ++i) {
    x += s[i];
  }
  return x;
}

// Calls f(index, logit) for this thread's logits of [begin, end) of a row, four at a
// time where the row is 16-byte aligned.
template <class F>
__device__ __forceinline__ void each_logit(const float* logits, uint32_t begin, uint32_t end, F f) {
  if (((uintptr_t)logits & 15u) == 0) {
    const uint32_t whole = begin + ((end - begin) & ~3u);
#pragma unroll 4
    for (uint32_t i = begin + 4u * threadIdx.x; i < whole; i += 4u * kThreads) {
      const float4_t x = *reinterpret_cast<const float4_t*>(logits + i);
      f(i, x[0]);
      f(i + 1u, x[1]);
      f(i + 2u, x[2]);
      f(i + 3u, x[3]);
    }
    if (whole + threadIdx.x < end) {
      f(whole + threadIdx.x, logits[whole + threadIdx.x]);
    }
  } else {
#pragma unroll 4
    for (uint32_t i = begin + threadIdx.x; i < end; i += kThreads) {
      f(i, logits[i]);
    }
  }
}

__global__ __launch_bounds__(kThreads) void sample_top_kernel(SampleArgs a, Plan p) {
  __shared__ uint64_t s[kThreads / 64u];
  const uint32_t row = blockIdx.y, chunk = blockIdx.x;
  const float* logits = a.logits + (size_t)row * a.row_stride;
  const RowWork w = row_work(p, row);
  const uint32_t begin = chunk * p.chunk, end = min(a.size, begin + p.chunk);
  uint64_t top = (uint32_t)~a.size;  // of NaNs alone: key 0, index `size`
  each_logit(logits, begin, end, [&](uint32_t i, float x) {
    const uint32_t key = key_of(x);
    const uint64_t both = (uint64_t)key << 32 | (uint32_t)~i;
    top = key != 0u && both > top ? both : top;
  });
  top = block_max<kThreads / 64u>(top, s);
  if (threadIdx.x == 0) {
    w.chunk_top[chunk] = top;
  }
  if (chunk == 0) {
    for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
      w.bin_weight[i] = 0;
      w.bin_count[i] = 0;
    }
    if (threadIdx.x == 0) {
      *w.listed = 0;
    }
  }
}

// The row's largest key, from its chunks'.
template <uint32_t kWaves>
__device__ __forceinline__ uint64_t row_top(const RowWork& w, uint32_t chunks, uint64_t* s) {
  uint64_t top = 0;
  for (uint32_t i = threadIdx.x; i < chunks; i += kWaves * 64u) {
    top = w.chunk_top[i] > top ? w.chunk_top[i] : top;
  }
  return block_max<kWaves>(top, s);
}

__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleArgs a, Plan p) {
  constexpr uint32_t kWaves = kThreads / 64u;
  __shared__ uint64_t s[kWaves];
  __shared__ uint64_t weights[kBins];
  __shared__ uint32_t counts[kBins];
  const uint32_t row = blockIdx.y, chunk = blockIdx.x;
  const RowRule rule = row_rule(a, row);
  const RowWork w = row_work(p, row);
  const uint32_t top = (uint32_t)(row_top<kWaves>(w, p.chunks, s) >> 32);
  if (takes_top(rule, top)) {
    return;
  }
  for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
    weights[i] = 0;
    counts[i] = 0;
  }
  __syncthreads();
  const float scale = (float)(8.0 * 1.4426950408889634 * rule.inverse_temperature);
  const uint32_t begin = chunk * p.chunk, end = min(a.size, begin + p.chunk);
  each_logit(a.logits + (size_t)row * a.row_stride, begin, end, [&](uint32_t, float x) {
    const uint32_t key = key_of(x);
    if (key != 0u) {
      const uint32_t bin = bin_of(key, top, scale);
      const uint64_t v = fixed(weight_of(key, top, rule.inverse_temperature), p.shift);
      atomicAdd((unsigned long long*)&weights[bin], (unsigned long long)v);
      atomicAdd(&counts[bin], 1u);
    }
  });
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
    w.chunk_bins[(size_t)chunk * kBins + i] = weights[i];
    if (counts[i] != 0u) {
      atomicAdd((unsigned long long*)&w.bin_weight[i], (unsigned long long)weights[i]);
      atomicAdd(&w.bin_count[i], counts[i]);
    }
  }
}

// Which bins a row's threshold can lie in.
struct Bounds {
  uint32_t sure;       // bins below are kept whatever the threshold
  uint32_t last;       // bins sure .. last are listed; none if last < sure
  bool cut;            // top-k or top-p cuts inside the list
  uint64_t above;      // weight and number of the bins below `sure`
  uint32_t above_n;
  uint64_t total;      // weight of the row
};

struct BoundScratch {
  uint64_t sums[16];
  uint32_t counts[16];
  uint64_t before[kBins];    // weight of the bins before
  uint64_t k_before, k_weight;
  uint32_t before_n[kBins];
  uint32_t k_bin, p_first, p_last;
};

// kWaves * 64 threads, kBins / that many bins each (at least one).
template <uint32_t kWaves>
__device__ Bounds row_bounds(const RowRule& rule, const RowWork& w, BoundScratch& s) {
  constexpr uint32_t kPer = kBins > kWaves * 64u ? kBins / (kWaves * 64u) : 1u;
  const bool holds = threadIdx.x * kPer < kBins;
  uint64_t weight[kPer], x = 0, total;
  uint32_t count[kPer], n = 0, all_n;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    weight[i] = holds ? w.bin_weight[threadIdx.x * kPer + i] : 0u;
    count[i] = holds ? w.bin_count[threadIdx.x * kPer + i] : 0u;
    x += weight[i];
    n += count[i];
  }
  block_scan<kWaves>(x, n, total, all_n, s.sums, s.counts);
  if (threadIdx.x == 0) {
    s.k_bin = kBins;
    s.k_before = total;
    s.k_weight = 0;
    s.p_first = 0;
    s.p_last = 0;
  }
  __syncthreads();
  uint64_t at = x;
  uint32_t at_n = n;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    if (holds) {
      const uint32_t bin = threadIdx.x * kPer + i;
      s.before[bin] = at;
      s.before_n[bin] = at_n;
      if (rule.top_k != 0u && at_n < rule.top_k && at_n + count[i] >= rule.top_k) {
        s.k_bin = bin;  // one bin only
        s.k_before = at;
        s.k_weight = weight[i];
      }
      at += weight[i];
      at_n += count[i];
    }
  }
  __syncthreads();
  const uint32_t k_bin = s.k_bin;
  if (rule.top_p < 1.0) {
    // The last bin before which less than the target lies, for the least and the
    // largest weight that top-k may leave.
    const double least = rule.top_p * (double)s.k_before;
    const double most = rule.top_p * (double)(s.k_before + s.k_weight);
    at = x;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      const uint32_t bin = threadIdx.x * kPer + i;
      if (holds && count[i] != 0u && bin <= k_bin) {
        if ((double)at < least) {
          atomicMax(&s.p_first, bin);
        }
        if ((double)at < most) {
          atomicMax(&s.p_last, bin);
        }
      }
      at += weight[i];
    }
  }
  __syncthreads();
  Bounds b;
  b.total = total;
  b.cut = rule.top_k != 0u || rule.top_p < 1.0;
  b.sure = rule.top_p < 1.0 ? s.p_first : k_bin;
  b.last = rule.top_k != 0u ? k_bin : rule.top_p < 1.0 ? s.p_last : 0u;
  if (rule.min_p > 0.0) {
    // The border of min_p lies in its bin, or a neighbour of it by rounding.
    const uint32_t bin = (uint32_t)fmin(-8.0 * log2(rule.min_p), (double)(kBins - 1u));
    const uint32_t low = bin != 0u ? bin - 1u : 0u, high = min(bin + 1u, kBins - 1u);
    if (!b.cut || high < b.sure) {
      b.cut = false;  // top-k and top-p keep all that min-p does
      b.last = high;
    }
    b.sure = min(b.sure, low);
  } else if (!b.cut) {
    b.sure = kBins;
  }
  b.above = b.sure < kBins ? s.before[b.sure] : total;
  b.above_n = b.sure < kBins ? s.before_n[b.sure] : all_n;
  return b;
}

__global__ __launch_bounds__(kThreads) void sample_gather_kernel(SampleArgs a, Plan p) {
  constexpr uint32_t kWaves = kThreads / 64u;
  __shared__ uint64_t s[kWaves];
  __shared__ BoundScratch bs;
  const uint32_t row = blockIdx.y, chunk = blockIdx.x;
  const RowRule rule = row_rule(a, row);
  const RowWork w = row_work(p, row);
  const uint32_t top = (uint32_t)(row_top<kWaves>(w, p.chunks, s) >> 32);
  if (takes_top(rule, top)) {
    return;
  }
  const Bounds b = row_bounds<kWaves>(rule, w, bs);
  uint64_t sum = 0;
  for (uint32_t i = threadIdx.x; i < b.sure; i += kThreads) {
    sum += w.chunk_bins[(size_t)chunk * kBins + i];
  }
  sum = block_sum<kWaves>(sum, s);
  if (threadIdx.x == 0) {
    w.chunk_weight[chunk] = sum;
  }
  if (b.last < b.sure || b.sure == kBins) {
    return;  // no list
  }
  const float scale = (float)(8.0 * 1.4426950408889634 * rule.inverse_temperature);
  const uint32_t begin = chunk * p.chunk, end = min(a.size, begin + p.chunk);
  each_logit(a.logits + (size_t)row * a.row_stride, begin, end, [&](uint32_t i, float x) {
    const uint32_t key = key_of(x);
    const uint32_t bin = bin_of(key, top, scale);
    if (key != 0u && bin >= b.sure && bin <= b.last) {
      w.list[atomicAdd(w.listed, 1u)] = (uint64_t)key << 32 | i;
    }
  });
}

// The kept set within the list: keys above `key`, and those equal to it up to `index`.
struct Cut {
  uint32_t key, index;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const {
    return k > key || (k == key && i <= index);
  }
};

struct DrawScratch {
  uint64_t chunk_weight[kMaxChunks];
  union {
    struct {
      uint64_t bins[kDrawThreads];
      uint32_t counts[kDrawThreads];
    };
    BoundScratch bounds;
  };
  uint64_t sums[16];
  uint32_t wave_counts[16];
  uint64_t found_weight;
  uint32_t found, found_count, found_here;
};

// Radix selection in the list, ten bits of `field` at a time from its highest that
// differ.  Walking from the largest field down (each with its weight and count), the
// last value before which less than `target` (by weight, at least the first value) or
// fewer than `count` (by count) lie.  Returns the value; `before`, `before_n` become
// what lies before it and `here` the number of entries that have it.
template <class Field, class Weight>
__device__ __forceinline__ uint32_t select_value(uint32_t entries, bool by_weight, double target,
                                                 uint32_t count, Field field, Weight weight,
                                                 uint64_t& before, uint32_t& before_n,
                                                 uint32_t& here, DrawScratch& s) {
  constexpr uint32_t kWaves = kDrawThreads / 64u;
  // field(i, value) says whether entry i counts.
  uint32_t low = 0xffffffffu, high = 0, counted = 0;
  for (uint32_t i = threadIdx.x; i < entries; i += kDrawThreads) {
    uint32_t v;
    if (field(i, v)) {
      low = min(low, v);
      high = max(high, v);
      ++counted;
    }
  }
  here = (uint32_t)block_sum<kWaves>(counted, s.sums);
  high = (uint32_t)block_max<kWaves>(high, s.sums);
  low = ~(uint32_t)block_max<kWaves>((uint32_t)~low, s.sums);
  const uint32_t differ = low ^ high;
  int at = differ != 0u ? 32 - __builtin_clz(differ) : 0;
  // The bits above `at` are the same in all.
  uint32_t prefix = at < 32 ? high >> at << at : 0u;
  while (at > 0) {
    const int bits = min(at, 10), next = at - bits;
    __syncthreads();
    s.bins[threadIdx.x] = 0;
    s.counts[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < entries; i += kDrawThreads) {
      uint32_t v;
      if (field(i, v) && (at >= 32 || v >> at == prefix >> at)) {
        // The largest value first.
        const uint32_t digit = kDrawThreads - 1u - (v >> next & ((1u << bits) - 1u));
        atomicAdd(&s.counts[digit], 1u);
        if (by_weight) {
          atomicAdd((unsigned long long*)&s.bins[digit], (unsigned long long)weight(i));
        }
      }
    }
    __syncthreads();
    uint64_t x = s.bins[threadIdx.x], all;
    uint32_t n = s.counts[threadIdx.x], all_n;
    const uint32_t own = n;
    if (threadIdx.x == 0) {
      s.found = 0;
    }
    block_scan<kWaves>(x, n, all, all_n, s.sums, s.wave_counts);
    const bool reaches = own != 0u && (n == 0u || (by_weight ? (double)(before + x) < target
                                                             : before_n + n < count));
    if (reaches) {
      atomicMax(&s.found, threadIdx.x);
    }
    __syncthreads();
    if (s.found == threadIdx.x) {
      s.found_weight = before + x;
      s.found_count = before_n + n;
      s.found_here = own;
    }
    __syncthreads();
    prefix |= (kDrawThreads - 1u - s.found) << next;
    before = s.found_weight;
    before_n = s.found_count;
    here = s.found_here;
    at = next;
  }
  return prefix;
}

__global__ __launch_bounds__(kDrawThreads) void sample_draw_kernel(SampleArgs a, Plan p) {
  constexpr uint32_t kWaves = kDrawThreads / 64u;
  __shared__ DrawScratch s;
  const uint32_t row = blockIdx.x, size = a.size;
  const float* logits = a.logits + (size_t)row * a.row_stride;
  const RowRule rule = row_rule(a, row);
  const RowWork w = row_work(p, row);
  const uint64_t first = row_top<kWaves>(w, p.chunks, s.sums);
  const uint32_t top = (uint32_t)(first >> 32), top_index = ~(uint32_t)first;
  if (takes_top(rule, top)) {
    if (threadIdx.x == 0) {
      a.tokens[row] = (int32_t)top_index;
      if (a.probabilities != nullptr) {
        a.probabilities[row] = top > kMinusInfKey ? 1.0f : 0.0f;
      }
    }
    return;
  }
  const double inverse = rule.inverse_temperature;
  auto weight = [&](uint32_t key) { return fixed(weight_of(key, top, inverse), p.shift); };
  const Bounds b = row_bounds<kWaves>(rule, w, s.bounds);
  const uint32_t entries = b.last < b.sure || b.sure == kBins ? 0u : *w.listed;
  Cut cut{0u, 0xffffffffu};
  if (b.cut) {
    // The threshold's ties: all, or the first few by index.
    auto ties = [&](uint32_t key, uint32_t keep, uint32_t here) {
      cut.key = key;
      cut.index = 0xffffffffu;
      if (keep < here) {
        // Of the inverted indices the keep-th largest.
        uint64_t before = 0;
        uint32_t before_n = 0, equal;
        cut.index = ~select_value(
          entries, false, 0.0, keep,
          [&](uint32_t i, uint32_t& v) {
            const uint64_t e = w.list[i];
            v = ~(uint32_t)e;
            return (uint32_t)(e >> 32) == key;
          },
          [](uint32_t) { return (uint64_t)0; }, before, before_n, equal, s);
      }
    };
    uint64_t whole = b.total;
    if (rule.top_k != 0u) {
      uint64_t before = 0;
      uint32_t before_n = b.above_n, here;
      const uint32_t key = select_value(
        entries, false, 0.0, rule.top_k,
        [&](uint32_t i, uint32_t& v) {
          v = (uint32_t)(w.list[i] >> 32);
          return true;
        },
        [](uint32_t) { return (uint64_t)0; }, before, before_n, here, s);
      ties(key, rule.top_k - before_n, here);
      if (rule.top_p < 1.0) {
        uint64_t sum = 0;
        for (uint32_t i = threadIdx.x; i < entries; i += kDrawThreads) {
          const uint64_t e = w.list[i];
          sum += cut.keeps((uint32_t)(e >> 32), (uint32_t)e) ? weight((uint32_t)(e >> 32)) : 0u;
        }
        whole = b.above + block_sum<kWaves>(sum, s.sums);
      }
    }
    if (rule.top_p < 1.0) {
      const Cut within = cut;
      const double target = rule.top_p * (double)whole;
      uint64_t before = b.above;
      uint32_t before_n = b.above_n, here;
      const uint32_t key = select_value(
        entries, true, target, 0u,
        [&](uint32_t i, uint32_t& v) {
          const uint64_t e = w.list[i];
          v = (uint32_t)(e >> 32);
          return within.keeps(v, (uint32_t)e);
        },
        [&](uint32_t i) { return weight((uint32_t)(w.list[i] >> 32)); }, before, before_n, here,
        s);
      // The i-th tie is kept where before + i w < target.
      const uint64_t each = weight(key);
      uint32_t keep = here;
      if (each != 0u) {
        const double need = ceil((target - (double)before) / (double)each);
        keep = need < (double)here ? (need > 1.0 ? (uint32_t)need : 1u) : here;
      }
      if (key == within.key && keep >= here) {
        cut = within;  // its ties are cut already
      } else {
        ties(key, keep, here);
      }
    }
  }

  // The kept weight of an element of the list, and of any.
  auto kept_listed = [&](uint32_t key, uint32_t i) {
    const double x = weight_of(key, top, inverse);
    return cut.keeps(key, i) && x >= rule.min_p ? fixed(x, p.shift) : (uint64_t)0;
  };
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < p.chunks; i += kDrawThreads) {
    s.chunk_weight[i] = w.chunk_weight[i];
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < entries; i += kDrawThreads) {
    const uint64_t e = w.list[i];
    const uint64_t x = kept_listed((uint32_t)(e >> 32), (uint32_t)e);
    if (x != 0u) {
      atomicAdd((unsigned long long*)&s.chunk_weight[(uint32_t)e / p.chunk], (unsigned long long)x);
    }
  }
  __syncthreads();
  // The chunk: a run of chunks a thread.
  const uint32_t per = (p.chunks + kDrawThreads - 1u) / kDrawThreads;
  uint64_t x = 0, total;
  uint32_t n = 0, all_n;
  for (uint32_t i = threadIdx.x * per; i < min(p.chunks, (threadIdx.x + 1u) * per); ++i) {
    x += s.chunk_weight[i];
  }
  block_scan<kWaves>(x, n, total, all_n, s.sums, s.wave_counts);
  const uint64_t row_total = total;
  const double target = rule.uniform * (double)total;
  // Where no running sum passes the target (a uniform of 1), the last kept token.
  if (threadIdx.x == 0) {
    s.found = 0xffffffffu;
    s.found_here = 0;
  }
  __syncthreads();
  uint64_t at = x;
  for (uint32_t i = threadIdx.x * per; i < min(p.chunks, (threadIdx.x + 1u) * per); ++i) {
    const uint64_t here = s.chunk_weight[i];
    at += here;
    if (here != 0u) {
      if ((double)at > target) {
        atomicMin(&s.found, i);
      }
      atomicMax(&s.found_here, i);
    }
  }
  __syncthreads();
  const uint32_t chunk = s.found != 0xffffffffu ? s.found : s.found_here;
  if (threadIdx.x == chunk / per) {
    at = x;
    for (uint32_t i = threadIdx.x * per; i < chunk; ++i) {
      at += s.chunk_weight[i];
    }
    s.found_weight = at;
  }
  __syncthreads();
  uint64_t before = s.found_weight;
  const float scale = (float)(8.0 * 1.4426950408889634 * inverse);
  const uint32_t begin = chunk * p.chunk, end = min(size, begin + p.chunk);
  if (threadIdx.x == 0) {
    s.found = 0xffffffffu;
    s.found_here = 0;
  }
  // p.chunk is at most four logits a thread.
  uint64_t kept[4], sum = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t i = begin + 4u * threadIdx.x + j;
    kept[j] = 0;
    if (i < end) {
      const uint32_t key = key_of(logits[i]);
      const uint32_t bin = bin_of(key, top, scale);
      if (key != 0u && bin < b.sure) {
        kept[j] = weight(key);
      } else if (key != 0u && entries != 0u && bin <= b.last) {
        kept[j] = kept_listed(key, i);
      }
    }
    sum += kept[j];
  }
  block_scan<kWaves>(sum, n, total, all_n, s.sums, s.wave_counts);
  before += sum;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    before += kept[j];
    if (kept[j] != 0u) {
      const uint32_t i = begin + 4u * threadIdx.x + j;
      if ((double)before > target) {
        atomicMin(&s.found, i);
      }
      atomicMax(&s.found_here, i);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t token = s.found != 0xffffffffu ? s.found : s.found_here;
    a.tokens[row] = (int32_t)token;
    if (a.probabilities != nullptr) {
      const double x = weight_of(key_of(logits[token]), top, inverse);
      a.probabilities[row] = (float)(ldexp(x, p.shift) / (double)row_total);
    }
  }
}

Plan plan_of(const SampleArgs& a) {
  Plan p{};
  // 1024 logits a workgroup while that gives few of them (a single row is a matter of
  // latency), else 4096, the most that the draw scans.
  const uint64_t small = ((uint64_t)a.size + 1023u) / 1024u;
  p.chunk = small * a.rows <= 2048u && small <= kMaxChunks ? 1024u : 4096u;
  p.chunks = (a.size + p.chunk - 1u) / p.chunk;
  p.shift = 62;
  for (uint64_t n = a.size; n > 1u; n = (n + 1u) / 2u) {
    --p.shift;
  }
  p.row_words = words_per_row(p.chunks, a.size);
  return p;
}

// Rows at a time: those whose workspace takes no more than 1 GiB.
uint32_t rows_at_once(const SampleArgs& a, const Plan& p) {
  const uint64_t fit = (uint64_t{1} << 30) / (p.row_words * sizeof(uint64_t));
  return (uint32_t)std::min<uint64_t>(a.rows, std::max<uint64_t>(fit, 1u));
}

}  // namespace

size_t sample_workspace_bytes(const SampleArgs& a) {
  const Plan p = plan_of(a);
  return rows_at_once(a, p) * p.row_words * sizeof(uint64_t);
}

hipError_t launch_sample(const SampleArgs& a, void* workspace, hipStream_t stream) {
  Plan p = plan_of(a);
  p.work = static_cast<uint64_t*>(workspace);
  const uint32_t at_once = rows_at_once(a, p);
  for (uint32_t row = 0; row < a.rows; row += at_once) {
    SampleArgs g = a;
    g.rows = std::min(at_once, a.rows - row);
    g.logits += (size_t)row * a.row_stride;
    g.temperature += a.temperature != nullptr ? row : 0u;
    g.top_k += a.top_k != nullptr ? row : 0u;
    g.top_p += a.top_p != nullptr ? row : 0u;
    g.min_p += a.min_p != nullptr ? row : 0u;
    g.uniforms += row;
    g.tokens += row;
    g.probabilities += a.probabilities != nullptr ? row : 0u;
    const dim3 grid(p.chunks, g.rows);
    sample_top_kernel<<<grid, kThreads, 0, stream>>>(g, p);
    sample_bins_kernel<<<grid, kThreads, 0, stream>>>(g, p);
    sample_gather_kernel<<<grid, kThreads, 0, stream>>>(g, p);
    sample_draw_kernel<<<dim3(g.rows), kDrawThreads, 0, stream>>>(g, p);
  }
  return hipGetLastError();
}

}  // namespace kraken
