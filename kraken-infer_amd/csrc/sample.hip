// One token a row from logits, with temperature, top-k, top-p and min-p, by a given
// uniform number.
//
// Every filter keeps a prefix of the order of falling logits, so what is kept is a
// threshold: the logits above it and, of those equal to it, the first few by index.
// Nothing is sorted.  Logits are ordered by 32-bit keys.  A weight w = exp((l - max) / T)
// is formed in 64 bits and held as an integer of 2^-shift, with room for `size` of the
// largest: the sums are exact whatever their order, so that atomics give one result, and
// close enough to the real numbers (for 250000 tokens each weight is within 2^-45 of the
// largest and 7e-12 of itself) that a cut or a draw falls on their side of a border.
//
// Four launches, the first three with a workgroup for each chunk of a row:
//   top     the largest key of the chunk and its first index
//   bins    the row's histogram over 1/8 octaves of weight (how much, and how many where
//           top-k asks) and each chunk's own
//   gather  the histogram says which bins a threshold can lie in (one, or a few where
//           top-p depends on a top-k that is not resolved yet); their elements go to a
//           list, and what lies above them is summed by chunk from the chunk's bins
//   draw    one workgroup a row: the threshold in the list (each entry against each in a
//           short one, by radix selection in a long one), then the chunk in which the
//           draw falls, and the token by a scan of that chunk alone.
// So a row is read three times, from memory once (the rest from the caches), and each
// exponential is formed once but for those of the list and of the drawn chunk.
//
// 64 rows of 248320 take 72 to 76 us by their rules, 6 times the logits' way from memory;
// traced, which keeps dispatches apart, 12, 27, 18 and 22.  top runs at 5.2 TB/s.  Of bins,
// the sums of all workgroups in memory are 2 us, counts 3, the exponentials 5, and 18
// reading and adding in LDS.  gather repeats the scan of the row's histogram in each
// workgroup.  draw is a chain of some thirty barriers in one workgroup a row, and most of a
// small call's time (8 rows of 32000: 26 us, draw traced 17; one row of 248320: 28 and
// 14).  A launch costs 2 to 3 us, a release to the device within one
// more (31 us instead of 6), so that no launch ends with its last workgroup's join.
// Several chunks a workgroup, logits asked for ahead of the bounds, and short lists put
// in order by a network were no faster.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "context_internal.hpp"
#include "device_common.hpp"
#include "paged_q8_internal.hpp"

namespace kraken {
namespace {

constexpr uint32_t kThreads = 256;      // of the chunk kernels
constexpr uint32_t kDrawThreads = 512;  // of the draw
constexpr uint32_t kBins = 512;         // 1/8 octave each; the last takes all below 2^-63
constexpr uint32_t kMaxChunk = 4096;    // logits of a chunk
constexpr uint32_t kMaxChunks = 1024;   // of a row
// Histograms of a row that its chunks add to in turn, joined by who reads them: with one,
// 243 workgroups wait for each other (us, 1 row of 248320 / 64 of them: 30.4 / 81.7; two
// 27.9 / 80.1, four 27.0 / 77.9, eight 26.6 / 80.0).
constexpr uint32_t kCopies = 4;
constexpr uint32_t kHeld = 8192;        // entries of the list that the draw holds in LDS
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

// A row's weights: exp((l - max) / T) 2^shift as an integer, and the bins that they fall
// into.
struct Weights {
  float top;              // the largest logit
  double top_wide, factor;  // factor: log2(e) / T
  double one;             // 2^shift
  int shift;
};

__device__ __forceinline__ Weights weights_of(uint32_t top, const RowRule& rule, int shift) {
  const float logit = logit_of(top);
  const double factor = 1.4426950408889634074 * rule.inverse_temperature;
  return {logit, (double)logit, factor, ldexp(1.0, shift), shift};
}

// A logit's weight (not a NaN's), before rounding to a whole number: 2^y 2^shift with
// y = n + f, |f| <= 1/2, by the Taylor series of e^(f ln 2), whose first term left out is
// (ln 2 / 2)^10 / 10! = 7e-12.  Zero from y = -1000 down, and of -inf.
__device__ __forceinline__ double weight_real(float logit, const Weights& w) {
  const double y = ((double)logit - w.top_wide) * w.factor;
  const double n = rint(y);
  const double t = (y - n) * 0.69314718055994530942;
  double r = 1.0 / 362880.0;
  r = fma(r, t, 1.0 / 40320.0);
  r = fma(r, t, 1.0 / 5040.0);
  r = fma(r, t, 1.0 / 720.0);
  r = fma(r, t, 1.0 / 120.0);
  r = fma(r, t, 1.0 / 24.0);
  r = fma(r, t, 1.0 / 6.0);
  r = fma(r, t, 0.5);
  r = fma(r, t, 1.0);
  r = fma(r, t, 1.0);
  // The largest logit may be infinite, and so may the factor.
  return logit == w.top ? w.one : y > -1000.0 ? ldexp(r, (int)n + w.shift) : 0.0;
}

__device__ __forceinline__ uint64_t weight_fixed(float logit, const Weights& w) {
  // Up to 2^51, an addition of 2^52 leaves the rounded number in the low bits.
  return (uint64_t)__double_as_longlong(weight_real(logit, w) + 0x1p52) &
         ((uint64_t{1} << 52) - 1u);
}

// How many eighths of an octave a logit's weight lies below the largest, and its bin:
// falling logits have rising bins (each step of it is monotone).  NaN only of a NaN.  In 64
// bits, as the weight: two logits' difference, or 1 / T, may be beyond f32's largest.
__device__ __forceinline__ float eighths_of(float logit, const Weights& w) {
  const float z = (float)(((double)logit - w.top_wide) * w.factor * -8.0);
  return logit == w.top ? 0.0f : logit != logit ? z : z >= 0.0f ? z : (float)kBins;
}

__device__ __forceinline__ uint32_t bin_of(float logit, const Weights& w) {
  return (uint32_t)fminf(eighths_of(logit, w), (float)(kBins - 1u));
}

// Which bins a row's threshold can lie in, and the row's largest.
struct RowMeta {
  uint64_t above;      // weight and number of the bins below `sure`
  uint64_t total;      // weight of the row
  uint32_t above_n;
  uint32_t sure;       // bins below are kept whatever the threshold
  uint32_t last;       // bins sure .. last are listed; none if last < sure
  uint32_t cut;        // top-k or top-p cuts inside the list
  uint32_t top, top_index;
};

struct Entry {
  uint32_t index, key;
  uint64_t weight;
};

// A row's place in the workspace.
struct RowWork {
  RowMeta* meta;
  uint64_t* bin_weight;    // [kCopies][kBins]: chunk c adds to copy c % kCopies
  uint32_t* bin_count;     // [kCopies][kBins]
  uint64_t* chunk_weight;  // [chunks]: of what is kept whatever the threshold
  uint64_t* chunk_top;     // [chunks]: key << 32 | ~index
  uint32_t* chunk_listed;  // [chunks]: entries of the chunk's part of the list
  uint64_t* chunk_bins;    // [chunks][kBins]
  Entry* list;             // [chunks][chunk]
};

struct Plan {
  uint32_t chunk, chunks;  // logits per chunk, chunks per row
  int shift;
  uint64_t* work;
  size_t row_words;  // 8-byte words of the workspace per row
};

constexpr size_t kMetaWords = 8;

size_t words_per_row(const Plan& p) {
  return kMetaWords + kCopies * (kBins + kBins / 2u) + (size_t)p.chunks * (2u + kBins) +
         ((size_t)p.chunks / 2u + 1u) / 2u * 2u + 2u + 2u * (size_t)p.chunks * p.chunk;
}

__device__ __forceinline__ RowWork row_work(const Plan& p, uint32_t row) {
  static_assert(sizeof(RowMeta) <= kMetaWords * sizeof(uint64_t), "");
  RowWork w;
  uint64_t* at = p.work + (size_t)row * p.row_words;
  w.meta = reinterpret_cast<RowMeta*>(at);
  w.bin_weight = at + kMetaWords;
  w.bin_count = reinterpret_cast<uint32_t*>(w.bin_weight + kCopies * kBins);
  w.chunk_weight = w.bin_weight + kCopies * (kBins + kBins / 2u);
  w.chunk_top = w.chunk_weight + p.chunks;
  w.chunk_bins = w.chunk_top + p.chunks;
  // The list is 16-byte aligned: an even number of words before it.
  w.list = reinterpret_cast<Entry*>(w.chunk_bins + (size_t)p.chunks * kBins);
  w.chunk_listed = reinterpret_cast<uint32_t*>(w.list + (size_t)p.chunks * p.chunk);
  return w;
}

// Steps of a scan over a wave: lanes 1, 2, 4 and 8 before within a row of 16, then the
// last of the row before, and of the two rows before.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t lanes_before(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, kRows, 0xf, true);
}

template <int kCtrl, int kRows>
__device__ __forceinline__ uint64_t lanes_before(uint64_t x) {
  return (uint64_t)lanes_before<kCtrl, kRows>((uint32_t)(x >> 32)) << 32 |
         lanes_before<kCtrl, kRows>((uint32_t)x);
}

// Inclusive scan over the wave; 0 is the identity of `op`.
template <class T, class Op>
__device__ __forceinline__ T wave_scan(T x, Op op) {
  x = op(x, lanes_before<0x111, 0xf>(x));
  x = op(x, lanes_before<0x112, 0xf>(x));
  x = op(x, lanes_before<0x114, 0xf>(x));
  x = op(x, lanes_before<0x118, 0xf>(x));
  x = op(x, lanes_before<0x142, 0xa>(x));
  x = op(x, lanes_before<0x143, 0xc>(x));
  return x;
}

__device__ __forceinline__ uint64_t last_lane(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

struct Sum {
  template <class T>
  __device__ __forceinline__ T operator()(T x, T y) const {
    return x + y;
  }
};
struct Largest {
  template <class T>
  __device__ __forceinline__ T operator()(T x, T y) const {
    return x > y ? x : y;
  }
};

// op over a workgroup of kWaves waves, the result in every thread.
template <uint32_t kWaves, class Op>
__device__ __forceinline__ uint64_t block_reduce(uint64_t x, Op op, uint64_t* s) {
  x = last_lane(wave_scan(x, op));
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) {
    s[threadIdx.x >> 6] = x;
  }
  __syncthreads();
  x = s[0];
#pragma unroll
  for (uint32_t i = 1; i < kWaves; ++i) {
    x = op(x, s[i]);
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
  x = wave_scan(x, Sum{});
  n = wave_scan(n, Sum{});
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
  top = block_reduce<kThreads / 64u>(top, Largest{}, s);
  if (threadIdx.x == 0) {
    w.chunk_top[chunk] = top;
  }
  for (uint32_t copy = chunk; copy < kCopies; copy += p.chunks) {
    for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
      w.bin_weight[copy * kBins + i] = 0;
      w.bin_count[copy * kBins + i] = 0;
    }
  }
}

// Whether the condition holds here and in no later lane of the wave.
__device__ __forceinline__ bool last_that(bool condition) {
  const uint64_t all = __ballot(condition);
  return condition && (threadIdx.x & 63u) == 63u - (uint32_t)__builtin_clzll(all);
}

struct BoundScratch {
  uint64_t before[kBins];  // weight of the bins before
  uint32_t before_n[kBins];
  uint64_t k_before, k_weight;
  uint32_t k_bin, p_first, p_last;
};

// The bins that the row's threshold can lie in, from its histogram.
__device__ RowMeta row_bounds(const RowRule& rule, const RowWork& w, uint64_t* sums,
                              uint32_t* counts, BoundScratch& s) {
  constexpr uint32_t kWaves = kThreads / 64u, kPer = kBins / kThreads;
  uint64_t weight[kPer], x = 0, total;
  uint32_t count[kPer], n = 0, all_n;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    const uint32_t bin = threadIdx.x * kPer + i;
    weight[i] = 0;
    count[i] = 0;
#pragma unroll
    for (uint32_t copy = 0; copy < kCopies; ++copy) {
      weight[i] += w.bin_weight[copy * kBins + bin];
      count[i] += w.bin_count[copy * kBins + bin];
    }
    x += weight[i];
    n += count[i];
  }
  block_scan<kWaves>(x, n, total, all_n, sums, counts);
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
  __syncthreads();
  const uint32_t k_bin = s.k_bin;
  if (rule.top_p < 1.0) {
    // The last bin before which less than the target lies, for the least and the
    // largest weight that top-k may leave.
    const double least = rule.top_p * (double)s.k_before;
    const double most = rule.top_p * (double)(s.k_before + s.k_weight);
    at = x;
    uint32_t first = 0, last = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      const uint32_t bin = threadIdx.x * kPer + i;
      if (weight[i] != 0u && bin <= k_bin) {
        first = (double)at < least ? bin : first;
        last = (double)at < most ? bin : last;
      }
      at += weight[i];
    }
    // One atomic a wave, of its last thread that found one.
    if (last_that(first != 0u)) {
      atomicMax(&s.p_first, first);
    }
    if (last_that(last != 0u)) {
      atomicMax(&s.p_last, last);
    }
  }
  __syncthreads();
  RowMeta b;
  b.total = total;
  b.cut = rule.top_k != 0u || rule.top_p < 1.0;
  b.sure = rule.top_p < 1.0 ? s.p_first : k_bin;
  b.last = rule.top_k != 0u ? min(k_bin, kBins - 1u) : rule.top_p < 1.0 ? s.p_last : 0u;
  if (rule.min_p > 0.0) {
    // The border of min_p lies in its bin, or a neighbour of it by rounding.
    const uint32_t bin = (uint32_t)fmin(-8.0 * log2(rule.min_p), (double)(kBins - 1u));
    const uint32_t low = bin != 0u ? bin - 1u : 0u, high = min(bin + 1u, kBins - 1u);
    if (!b.cut || high < b.sure) {
      b.cut = 0;  // top-k and top-p keep all that min-p does
      b.last = high;
    }
    b.sure = min(b.sure, low);
  }
  if (b.sure == kBins) {
    b.last = 0;  // no list: everything is kept
  }
  b.above = b.sure < kBins ? s.before[b.sure] : total;
  b.above_n = b.sure < kBins ? s.before_n[b.sure] : all_n;
  return b;
}

__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleArgs a, Plan p) {
  constexpr uint32_t kWaves = kThreads / 64u;
  __shared__ uint64_t s[kWaves];
  __shared__ uint64_t bin_weight[kBins];
  __shared__ uint32_t bin_count[kBins];
  const uint32_t row = blockIdx.y, chunk = blockIdx.x;
  const RowRule rule = row_rule(a, row);
  const RowWork w = row_work(p, row);
  uint64_t first = 0;
  for (uint32_t i = threadIdx.x; i < p.chunks; i += kThreads) {
    first = w.chunk_top[i] > first ? w.chunk_top[i] : first;
  }
  for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
    bin_weight[i] = 0;
    bin_count[i] = 0;
  }
  first = block_reduce<kWaves>(first, Largest{}, s);
  const uint32_t top = (uint32_t)(first >> 32);
  if (chunk == 0 && threadIdx.x == 0) {
    w.meta->top = top;
    w.meta->top_index = ~(uint32_t)first;
  }
  if (takes_top(rule, top)) {
    return;
  }
  const Weights weights = weights_of(top, rule, p.shift);
  const bool counted = rule.top_k != 0u;
  const uint32_t begin = chunk * p.chunk, end = min(a.size, begin + p.chunk);
  each_logit(a.logits + (size_t)row * a.row_stride, begin, end, [&](uint32_t, float x) {
    if (x == x) {
      const uint32_t bin = bin_of(x, weights);
      atomicAdd((unsigned long long*)&bin_weight[bin],
                (unsigned long long)weight_fixed(x, weights));
      if (counted) {
        atomicAdd(&bin_count[bin], 1u);
      }
    }
  });
  __syncthreads();
  const uint32_t copy = chunk % kCopies * kBins;
  for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
    const uint64_t weight = bin_weight[i];
    w.chunk_bins[(size_t)chunk * kBins + i] = weight;
    if (weight != 0u) {
      atomicAdd((unsigned long long*)&w.bin_weight[copy + i], (unsigned long long)weight);
    }
    if (bin_count[i] != 0u) {
      atomicAdd(&w.bin_count[copy + i], bin_count[i]);
    }
  }
}

__global__ __launch_bounds__(kThreads) void sample_gather_kernel(SampleArgs a, Plan p) {
  constexpr uint32_t kWaves = kThreads / 64u;
  __shared__ uint64_t s[kWaves];
  __shared__ uint32_t wave_counts[kWaves];
  __shared__ BoundScratch bounds;
  __shared__ uint32_t found[kMaxChunk], founds;
  const uint32_t row = blockIdx.y, chunk = blockIdx.x;
  const RowRule rule = row_rule(a, row);
  const RowWork w = row_work(p, row);
  const uint32_t top = w.meta->top;
  if (takes_top(rule, top)) {
    return;
  }
  const RowMeta b = row_bounds(rule, w, s, wave_counts, bounds);
  const uint32_t sure = b.sure, last = b.last;
  if (chunk == 0 && threadIdx.x == 0) {
    // All but the largest, which is there already.
    w.meta->above = b.above;
    w.meta->total = b.total;
    w.meta->above_n = b.above_n;
    w.meta->sure = sure;
    w.meta->last = last;
    w.meta->cut = b.cut;
  }
  uint64_t sum = 0;
  for (uint32_t i = threadIdx.x; i < sure; i += kThreads) {
    sum += w.chunk_bins[(size_t)chunk * kBins + i];
  }
  if (threadIdx.x == 0) {
    founds = 0;
  }
  sum = block_reduce<kWaves>(sum, Sum{}, s);
  if (threadIdx.x == 0) {
    w.chunk_weight[chunk] = sum;
  }
  const Weights weights = weights_of(top, rule, p.shift);
  if (last >= sure) {
    // Bins sure .. last, the last bin without an end.
    const float from = (float)sure;
    const float to = last < kBins - 1u ? (float)(last + 1u) : INFINITY;
    const uint32_t begin = chunk * p.chunk, end = min(a.size, begin + p.chunk);
    each_logit(a.logits + (size_t)row * a.row_stride, begin, end, [&](uint32_t i, float x) {
      const float z = eighths_of(x, weights);
      if (z >= from && (z < to || to == INFINITY)) {
        found[atomicAdd(&founds, 1u)] = i;
      }
    });
  }
  __syncthreads();
  // The order of a list's entries changes nothing that is made of them.
  const uint32_t n = founds;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint32_t index = found[i];
    const float x = a.logits[(size_t)row * a.row_stride + index];
    w.list[(size_t)chunk * p.chunk + i] = {index, key_of(x), weight_fixed(x, weights)};
  }
  if (threadIdx.x == 0) {
    w.chunk_listed[chunk] = n;
  }
}

// The kept set within the list: keys above `key`, and those equal to it up to `index`.
struct Cut {
  uint32_t key, index;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const {
    return k > key || (k == key && i <= index);
  }
};

// A list this short is looked at entry against entry (8 rows of 32000: 29.5 us; by radix
// selection, or up to 256 entries this way, 31.1 and 30.0 us).
constexpr uint32_t kDirect = 128;
// So few left of a longer one end its radix selection (64 rows of 152000 alike: 88.5 us, 95
// without; up to 256 95, whose comparisons take what the steps did).
constexpr uint32_t kFew = 64;
constexpr uint32_t kDigits = 1024;  // of a step of the radix selection

struct DrawScratch {
  Entry held[kHeld];
  uint64_t chunk_weight[kMaxChunks];
  uint64_t bins[kDigits];
  uint32_t counts[kDigits];
  uint64_t sums[kDrawThreads / 64u];
  uint32_t wave_counts[kDrawThreads / 64u];
  uint64_t found_weight;
  uint32_t found, found_count, found_here;
  uint32_t cut_key, cut_index;
  uint64_t few_weights[kFew];
  uint32_t few_values[kFew], few;
};

// The entries of the list: in LDS, or (a row whose threshold has more than kHeld logits
// in its bins) in memory, a chunk a wave.
struct Entries {
  const RowWork* work;
  const Plan* plan;
  DrawScratch* s;
  uint32_t count;
  uint32_t low, high;  // their smallest and largest key

  // f(key, index, weight) for each of this thread's entries.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    if (count <= kHeld) {
      for (uint32_t i = threadIdx.x; i < count; i += kDrawThreads) {
        const Entry e = s->held[i];
        f(e.key, e.index, e.weight);
      }
    } else {
      for (uint32_t c = threadIdx.x / 64u; c < plan->chunks; c += kDrawThreads / 64u) {
        const uint32_t n = work->chunk_listed[c];
#pragma unroll 4
        for (uint32_t i = threadIdx.x & 63u; i < n; i += 64u) {
          const Entry e = work->list[(size_t)c * plan->chunk + i];
          f(e.key, e.index, e.weight);
        }
      }
    }
  }
};

// Radix selection in the list, ten bits of a field at a time until few are left.  field(key, index, value)
// says whether an entry counts, and its value, low <= value <= high.  Walking from the
// largest value down, the last one before which less than `target` (by weight; at least
// the first value) or fewer than `count` lie.  Returns the value; `before`, `before_n`
// become what lies before it and `here` the number of entries that have it.
template <bool kByWeight, class Field>
__device__ __forceinline__ uint32_t select_value(const Entries& e, double target, uint32_t count,
                                                 uint32_t low, uint32_t high, Field field,
                                                 uint64_t& before, uint32_t& before_n,
                                                 uint32_t& here, DrawScratch& s) {
  constexpr uint32_t kWaves = kDrawThreads / 64u, kPer = kDigits / kDrawThreads;
  const uint32_t differ = low ^ high;
  // The bits above `at` are the same in all; one step at least, which counts them.
  int at = differ != 0u ? 32 - __builtin_clz(differ) : 1;
  uint32_t prefix = at < 32 ? high >> at << at : 0u;
  here = 0;
  while (at > 0) {
    const int bits = min(at, 10), next = at - bits;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      s.bins[threadIdx.x + i * kDrawThreads] = 0;
      s.counts[threadIdx.x + i * kDrawThreads] = 0;
    }
    if (threadIdx.x == 0) {
      s.found = 0;
    }
    __syncthreads();
    e.each([&](uint32_t key, uint32_t index, uint64_t weight) {
      uint32_t v;
      if (field(key, index, v) && (at >= 32 || v >> at == prefix >> at)) {
        // The largest value first.
        const uint32_t digit = kDigits - 1u - (v >> next & ((1u << bits) - 1u));
        atomicAdd(&s.counts[digit], 1u);
        if (kByWeight) {
          atomicAdd((unsigned long long*)&s.bins[digit], (unsigned long long)weight);
        }
      }
    });
    __syncthreads();
    uint64_t weights[kPer], x = 0, all;
    uint32_t counts[kPer], n = 0, all_n;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      weights[i] = s.bins[threadIdx.x * kPer + i];
      counts[i] = s.counts[threadIdx.x * kPer + i];
      x += weights[i];
      n += counts[i];
    }
    block_scan<kWaves>(x, n, all, all_n, s.sums, s.wave_counts);
    uint64_t at_x = x;
    uint32_t at_n = n, best = 0;
    bool any = false;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      if (counts[i] != 0u && (at_n == 0u || (kByWeight ? (double)(before + at_x) < target
                                                       : before_n + at_n < count))) {
        best = threadIdx.x * kPer + i;
        any = true;
      }
      at_x += weights[i];
      at_n += counts[i];
    }
    if (last_that(any)) {
      atomicMax(&s.found, best);
    }
    __syncthreads();
    const uint32_t digit = s.found;
    if (digit / kPer == threadIdx.x) {
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) {
        if (digit % kPer == i) {
          s.found_weight = before + x;
          s.found_count = before_n + n;
          s.found_here = counts[i];
        }
        x += weights[i];
        n += counts[i];
      }
    }
    __syncthreads();
    prefix |= (kDigits - 1u - digit) << next;
    before = s.found_weight;
    before_n = s.found_count;
    here = s.found_here;
    at = next;
    if (at > 0 && here <= kFew) {
      // The few that are left, each against each.
      if (threadIdx.x == 0) {
        s.few = 0;
        s.found = 0xffffffffu;
      }
      __syncthreads();
      e.each([&](uint32_t key, uint32_t index, uint64_t weight) {
        uint32_t v;
        if (field(key, index, v) && v >> at == prefix >> at) {
          const uint32_t i = atomicAdd(&s.few, 1u);
          s.few_values[i] = v;
          s.few_weights[i] = weight;
        }
      });
      __syncthreads();
      bool reached = false;
      uint32_t own = 0, larger = 0, equal = 0;
      uint64_t heavier = 0;
      if (threadIdx.x < here) {
        own = s.few_values[threadIdx.x];
        for (uint32_t i = 0; i < here; ++i) {
          const uint32_t v = s.few_values[i];
          larger += v > own ? 1u : 0u;
          equal += v == own ? 1u : 0u;
          heavier += v > own ? s.few_weights[i] : 0u;
        }
        reached = larger == 0u || (kByWeight ? (double)(before + heavier) < target
                                             : before_n + larger < count);
        if (reached) {
          atomicMin(&s.found, own);
        }
      }
      __syncthreads();
      prefix = s.found;
      if (reached && own == prefix) {
        s.found_weight = before + heavier;
        s.found_count = before_n + larger;
        s.found_here = equal;
      }
      __syncthreads();
      before = s.found_weight;
      before_n = s.found_count;
      here = s.found_here;
      break;
    }
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
  const RowMeta b = *w.meta;
  const uint32_t top = b.top;
  if (takes_top(rule, top)) {
    if (threadIdx.x == 0) {
      a.tokens[row] = (int32_t)b.top_index;
      if (a.probabilities != nullptr) {
        a.probabilities[row] = top > kMinusInfKey ? 1.0f : 0.0f;
      }
    }
    return;
  }
  const Weights weights = weights_of(top, rule, p.shift);

  // The list into LDS: the chunks' places in it, then each entry from its chunk.
  const uint32_t per = (p.chunks + kDrawThreads - 1u) / kDrawThreads;
  const uint32_t run = min(p.chunks, threadIdx.x * per), run_end = min(p.chunks, run + per);
  uint64_t none = 0, none_all;
  uint32_t n = 0, all_n;
  for (uint32_t i = run; i < run_end; ++i) {
    n += w.chunk_listed[i];
  }
  block_scan<kWaves>(none, n, none_all, all_n, s.sums, s.wave_counts);
  Entries e{&w, &p, &s, all_n, 0u, 0u};
  for (uint32_t i = run; i < run_end; ++i) {
    s.chunk_weight[i] = n;
    n += w.chunk_listed[i];
  }
  __syncthreads();
  uint32_t high = 0, low = 0xffffffffu;
  if (all_n <= kHeld) {
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < all_n; i += kDrawThreads) {
      // The last chunk whose place is not behind i.
      uint32_t c = 0;
      for (uint32_t step = 1u << (31 - __builtin_clz(p.chunks)); step != 0u; step /= 2u) {
        c += c + step < p.chunks && s.chunk_weight[c + step] <= i ? step : 0u;
      }
      const Entry x = w.list[(size_t)c * p.chunk + (i - (uint32_t)s.chunk_weight[c])];
      s.held[i] = x;
      high = max(high, x.key);
      low = min(low, x.key);
    }
  } else {
    e.each([&](uint32_t key, uint32_t, uint64_t) {
      high = max(high, key);
      low = min(low, key);
    });
  }
  Cut cut{0u, 0xffffffffu};
  if (b.cut != 0u && all_n != 0u && all_n <= kDirect) {
    // A short list: what lies before each entry, by looking at all others.
    constexpr uint32_t kShare = kDrawThreads / kDirect;
    __syncthreads();
    const uint32_t i = threadIdx.x / kShare;
    const bool real = i < all_n;
    const Entry own = s.held[real ? i : 0u];
    uint64_t before = 0;
    uint32_t place = 0;
    for (uint32_t j = threadIdx.x % kShare; j < all_n; j += kShare) {
      const Entry other = s.held[j];
      const bool first =
        other.key > own.key || (other.key == own.key && other.index < own.index);
      before += first ? other.weight : 0u;
      place += first ? 1u : 0u;
    }
#pragma unroll
    for (uint32_t step = 1; step < kShare; step *= 2u) {
      before += (uint64_t)__shfl_xor((long long)before, (int)step, 64);
      place += (uint32_t)__shfl_xor((int)place, (int)step, 64);
    }
    before += b.above;
    const uint64_t upto = before + own.weight;
    // The entries that top-k leaves, and the sum that top-p is of.
    const uint32_t left = rule.top_k != 0u ? min(rule.top_k - b.above_n, all_n) : all_n;
    if (real && place + 1u == left) {
      s.found_weight = upto;
    }
    __syncthreads();
    const uint64_t whole = rule.top_k != 0u ? s.found_weight : b.total;
    const double target = rule.top_p < 1.0 ? rule.top_p * (double)whole : (double)INFINITY;
    // An entry is kept where less than the target lies before it, and the first always;
    // the threshold is the last one kept.
    const bool kept = place == 0u || (double)before < target;
    if (real && place < left && kept && (place + 1u == left || !((double)upto < target))) {
      s.cut_key = own.key;
      s.cut_index = own.index;
    }
    __syncthreads();
    cut = {s.cut_key, s.cut_index};
  } else if (b.cut != 0u && all_n != 0u) {
    e.high = (uint32_t)block_reduce<kWaves>(high, Largest{}, s.sums);
    e.low = ~(uint32_t)block_reduce<kWaves>((uint32_t)~low, Largest{}, s.sums);
    // The threshold's ties: all, or the first few by index.
    auto ties = [&](uint32_t key, uint32_t keep, uint32_t here) {
      cut.key = key;
      cut.index = 0xffffffffu;
      if (keep < here) {
        // Of the indices counted down from the last, the keep-th largest.
        uint64_t before = 0;
        uint32_t before_n = 0, equal;
        cut.index = size - 1u - select_value<false>(
          e, 0.0, keep, 0u, size - 1u,
          [&](uint32_t k, uint32_t index, uint32_t& v) {
            v = size - 1u - index;
            return k == key;
          },
          before, before_n, equal, s);
      }
    };
    uint64_t whole = b.total;
    if (rule.top_k != 0u) {
      uint64_t before = 0;
      uint32_t before_n = b.above_n, here;
      const uint32_t key = select_value<false>(
        e, 0.0, rule.top_k, e.low, e.high,
        [](uint32_t k, uint32_t, uint32_t& v) {
          v = k;
          return true;
        },
        before, before_n, here, s);
      ties(key, rule.top_k - before_n, here);
      if (rule.top_p < 1.0) {
        uint64_t sum = 0;
        e.each([&](uint32_t k, uint32_t index, uint64_t x) {
          sum += cut.keeps(k, index) ? x : 0u;
        });
        whole = b.above + block_reduce<kWaves>(sum, Sum{}, s.sums);
      }
    }
    if (rule.top_p < 1.0) {
      const Cut within = cut;
      const double target = rule.top_p * (double)whole;
      uint64_t before = b.above;
      uint32_t before_n = b.above_n, here;
      const uint32_t key = select_value<true>(
        e, target, 0u, e.low, e.high,
        [&](uint32_t k, uint32_t index, uint32_t& v) {
          v = k;
          return within.keeps(k, index);
        },
        before, before_n, here, s);
      // The i-th tie is kept where before + i w < target.
      const uint64_t each = weight_fixed(logit_of(key), weights);
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

  // Each chunk's kept weight.
  auto above_min = [&](uint32_t key) {
    return rule.min_p == 0.0 ||
           weight_real(logit_of(key), weights) >= ldexp(rule.min_p, p.shift);
  };
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < p.chunks; i += kDrawThreads) {
    s.chunk_weight[i] = w.chunk_weight[i];
  }
  __syncthreads();
  // A thread takes neighbours in the list, which are of one chunk mostly, and adds what it
  // has of a chunk at once (an entry at a time, the 64 of a wave wait for each other).
  uint32_t own_chunk = 0;
  uint64_t own = 0;
  auto add = [&](uint32_t key, uint32_t i, uint64_t x) {
    if (x != 0u && cut.keeps(key, i) && above_min(key)) {
      const uint32_t c = i / p.chunk;
      if (c != own_chunk && own != 0u) {
        atomicAdd((unsigned long long*)&s.chunk_weight[own_chunk], (unsigned long long)own);
        own = 0;
      }
      own_chunk = c;
      own += x;
    }
  };
  if (all_n <= kHeld) {
    const uint32_t each = (all_n + kDrawThreads - 1u) / kDrawThreads;
    const uint32_t to = min(all_n, (threadIdx.x + 1u) * each);
    for (uint32_t i = threadIdx.x * each; i < to; ++i) {
      const Entry held = s.held[i];
      add(held.key, held.index, held.weight);
    }
  } else {
    e.each(add);
  }
  if (own != 0u) {
    atomicAdd((unsigned long long*)&s.chunk_weight[own_chunk], (unsigned long long)own);
  }
  // One running sum passes the target first; where none does (a uniform of 1), the last
  // kept token is drawn.
  if (threadIdx.x == 0) {
    s.found = 0xffffffffu;
    s.found_here = 0;
  }
  __syncthreads();
  uint64_t x = 0, total;
  n = 0;
  for (uint32_t i = run; i < run_end; ++i) {
    x += s.chunk_weight[i];
  }
  block_scan<kWaves>(x, n, total, all_n, s.sums, s.wave_counts);
  const double target = rule.uniform * (double)total;
  uint64_t at = x;
  for (uint32_t i = run; i < run_end; ++i) {
    const uint64_t here = s.chunk_weight[i];
    if ((double)at <= target && (double)(at + here) > target) {
      s.found = i;
    }
    if (here != 0u && at + here == total) {
      s.found_here = i;
    }
    at += here;
  }
  __syncthreads();
  const uint32_t chunk = s.found != 0xffffffffu ? s.found : s.found_here;
  if (run <= chunk && chunk < run_end) {
    for (uint32_t i = run; i < chunk; ++i) {
      x += s.chunk_weight[i];
    }
    s.found_weight = x;
  }
  __syncthreads();
  uint64_t before = s.found_weight;
  if (threadIdx.x == 0) {
    s.found = 0xffffffffu;
    s.found_here = 0;
  }
  // The chunk's logits, kPer a thread.
  constexpr uint32_t kPer = kMaxChunk / kDrawThreads;
  const uint32_t begin = chunk * p.chunk + kPer * threadIdx.x;
  const uint32_t end = min(size, (chunk + 1u) * p.chunk);
  uint64_t kept[kPer], sum = 0, rest;
#pragma unroll
  for (uint32_t j = 0; j < kPer; ++j) {
    kept[j] = 0;
    const uint32_t i = begin + j;
    if (i < end && logits[i] == logits[i]) {
      const uint32_t key = key_of(logits[i]), bin = bin_of(logits[i], weights);
      if (bin < b.sure || (bin <= b.last && cut.keeps(key, i) && above_min(key))) {
        kept[j] = weight_fixed(logits[i], weights);
      }
    }
    sum += kept[j];
  }
  n = 0;
  block_scan<kWaves>(sum, n, rest, all_n, s.sums, s.wave_counts);
  const uint64_t chunk_end = before + rest;
  before += sum;
#pragma unroll
  for (uint32_t j = 0; j < kPer; ++j) {
    if ((double)before <= target && (double)(before + kept[j]) > target) {
      s.found = begin + j;
    }
    if (kept[j] != 0u && before + kept[j] == chunk_end) {
      s.found_here = begin + j;
    }
    before += kept[j];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t token = s.found != 0xffffffffu ? s.found : s.found_here;
    a.tokens[row] = (int32_t)token;
    if (a.probabilities != nullptr) {
      a.probabilities[row] =
        (float)(weight_real(logits[token], weights) / (double)total);
    }
  }
}

Plan plan_of(const SampleArgs& a) {
  Plan p{};
  // 1024 logits a workgroup while that gives few of them (a single row is a matter of
  // latency), else 4096, the most that the draw scans at once.
  const uint64_t small = ((uint64_t)a.size + 1023u) / 1024u;
  p.chunk = small * a.rows <= 2048u && small <= kMaxChunks ? 1024u : 4096u;
  p.chunks = (a.size + p.chunk - 1u) / p.chunk;
  p.shift = 62;
  for (uint64_t n = a.size; n > 1u; n = (n + 1u) / 2u) {
    --p.shift;
  }
  p.shift = std::min(p.shift, 51);
  p.row_words = words_per_row(p);
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
