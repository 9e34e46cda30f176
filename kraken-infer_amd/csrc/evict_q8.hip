// Eviction from a paged 8-bit cache: which positions of each sequence and KV head stay,
// and their move into fresh pages.
//
// The k-th largest of n weights is found by digits of keys that order as the weights do: the
// digit at which the count from above reaches k, then the next digit of the keys that have
// it.  A row moves as its codes: by one ratio, its page's scale over the largest of the target
// page's sources (the target's scale), rounded once more where that is not 1.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "context_internal.hpp"
#include "device_common.hpp"
#include "paged_q8_internal.hpp"
#include "row_order.hpp"

namespace kraken {
namespace {

constexpr uint32_t kHeld = 32;  // keys that a thread holds
// Digits of a key, from the top: 11, 11 and 10 bits.  Softmax weights fill few values of the
// top eight bits, their exponents, so that counts by eight bits fall on few words.
constexpr uint32_t kDigitBits = 11, kBins = 1u << kDigitBits;

// Sum over the workgroup's waves before this one, and over all, of a value that each wave
// has one of.
template <uint32_t kWaves>
__device__ __forceinline__ uint32_t waves_before(uint32_t x, uint32_t& all, uint32_t* s) {
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) {
    s[threadIdx.x >> 6] = x;
  }
  __syncthreads();
  uint32_t before = 0;
  all = 0;
#pragma unroll
  for (uint32_t i = 0; i < kWaves; ++i) {
    before += i < threadIdx.x >> 6 ? s[i] : 0u;
    all += s[i];
  }
  return before;
}

// How many lanes before this one are in the mask.
__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Counts of each digit.  kCopies: of the first's, by lane, so that lanes of one digit do not
// wait for each other; keys that have the digits before are few.
template <uint32_t kThreads, uint32_t kCopies>
struct SelectScratch {
  uint32_t bins[(kCopies + 2u) * kBins];
  uint32_t waves[kThreads / 64u];
  uint32_t digit, above;
};

// The `most` positions of the largest of `weights` [0, count), in rising order, plus `first`.
// A wave takes a run of them, 64 at a time, a lane each: loads are of whole lines, and the
// positions in order of wave, time and lane.  kInRegisters: up to kHeld times, each read once.
template <uint32_t kThreads, uint32_t kCopies, bool kInRegisters>
__device__ __forceinline__ void select_between(const float* weights, uint32_t count, uint32_t most,
                                               uint32_t first, int32_t* kept,
                                               SelectScratch<kThreads, kCopies>& s) {
  constexpr uint32_t kWaves = kThreads / 64u, kPer = kBins / kThreads;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t times = (count + kThreads - 1u) / kThreads;  // of a wave
  const uint32_t begin = wave * times * 64u + lane;
  for (uint32_t i = tid; i < (kCopies + 2u) * kBins; i += kThreads) {
    s.bins[i] = 0;
  }
  uint32_t held[kInRegisters ? kHeld : 1];
  if constexpr (kInRegisters) {
    float x[kHeld];
#pragma unroll
    for (uint32_t j = 0; j < kHeld; ++j) {
      x[j] = j < times && begin + j * 64u < count ? weights[begin + j * 64u] : NAN;
    }
#pragma unroll
    for (uint32_t j = 0; j < kHeld; ++j) {
      held[j] = key_of(x[j]);
    }
  }
  // f(key, time) for this lane's; it has to ask whether the place is one.  (Of held keys, those
  // that are none are 0 and larger than nothing.)
  auto each = [&](auto f) {
    if constexpr (kInRegisters) {
#pragma unroll
      for (uint32_t j = 0; j < kHeld; ++j) {
        if (j < times) {  // uniform
          f(held[j], j);
        }
      }
    } else {
      // Eight loads at a time.  (Past the end: the last again, for f to leave out.)
      for (uint32_t j = 0; j < times; j += 8) {
        float x[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
          x[i] = weights[min(begin + (j + i) * 64u, count - 1u)];
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
          if (j + i < times) {  // uniform
            f(key_of(x[i]), j + i);
          }
        }
      }
    }
  };
  // The least key that is kept; `want` of those equal to it are.
  uint32_t least = 0, known = 0, want = most;  // known: bits of `least` that are settled
  auto settle = [&](auto copies, uint32_t* counts, uint32_t shift, uint32_t mask) {
    constexpr uint32_t kOf = decltype(copies)::value;
    uint32_t* bins = counts + lane % kOf * kBins;
    __syncthreads();
    each([&](uint32_t key, uint32_t j) {
      if (begin + j * 64u < count && (key & known) == least) {
        atomicAdd(&bins[key >> shift & mask], 1u);
      }
    });
    __syncthreads();
    // kPer bins a thread, from the largest digit down.
    uint32_t mine[kPer], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      mine[i] = 0;
#pragma unroll
      for (uint32_t copy = 0; copy < kOf; ++copy) {
        mine[i] += counts[copy * kBins + kBins - 1u - (kPer * tid + i)];
      }
      sum += mine[i];
    }
    const uint32_t upto = wave_scan(sum, Sum{});
    uint32_t all;
    uint32_t before = waves_before<kWaves>((uint32_t)__builtin_amdgcn_readlane((int)upto, 63), all,
                                           s.waves);
    before += upto - sum;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      if (before < want && want <= before + mine[i]) {
        s.digit = kBins - 1u - (kPer * tid + i);
        s.above = before;
      }
      before += mine[i];
    }
    __syncthreads();
    least |= s.digit << shift;
    known |= mask << shift;
    want -= s.above;
  };
  using One = std::integral_constant<uint32_t, 1>;
  settle(std::integral_constant<uint32_t, kCopies>{}, s.bins, 21u, kBins - 1u);
  settle(One{}, s.bins + kCopies * kBins, 10u, kBins - 1u);
  settle(One{}, s.bins + (kCopies + 1u) * kBins, 0u, 1023u);
  // How many larger and equal ones each wave has, then their places.
  uint32_t larger = 0, equal = 0;
  each([&](uint32_t key, uint32_t j) {
    const bool is = begin + j * 64u < count;
    larger += (kInRegisters || is) && key > least ? 1u : 0u;
    equal += is && key == least ? 1u : 0u;
  });
  larger = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(larger, Sum{}), 63);
  equal = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(equal, Sum{}), 63);
  uint32_t all;
  uint32_t ties = waves_before<kWaves>(equal, all, s.waves);
  uint32_t place = waves_before<kWaves>(larger, all, s.waves) + min(ties, want);
  if (equal == 0) {  // uniform, and so for nearly all waves where weights differ
    each([&](uint32_t key, uint32_t j) {
      const uint32_t i = begin + j * 64u;
      const bool keep = (kInRegisters || i < count) && key > least;
      const uint64_t kept_here = __ballot(keep);
      if (keep) {
        kept[place + lanes_below(kept_here)] = (int32_t)(first + i);
      }
      place += (uint32_t)__popcll(kept_here);
    });
    return;
  }
  each([&](uint32_t key, uint32_t j) {
    const uint32_t i = begin + j * 64u;
    const uint64_t same = __ballot(i < count && key == least);
    const bool keep =
      i < count && (key > least || (key == least && ties + lanes_below(same) < want));
    const uint64_t kept_here = __ballot(keep);
    if (keep) {
      kept[place + lanes_below(kept_here)] = (int32_t)(first + i);
    }
    ties += (uint32_t)__popcll(same);
    place += (uint32_t)__popcll(kept_here);
  });
}

// One workgroup a sequence and KV head; kAny: with more keys than it can hold, too.  Not
// bytes but the three counts, their barriers and the last pass over the keys are what it spends
// its time on: 512 keys of one pair take 8.7 us, 4096 10.1, 32768 20.3, 131072 93; 64 sequences
// of 32768, two heads each, 20.5.  (120 and 132 scalars are spilled, into lanes of vector
// registers.)
template <uint32_t kThreads, uint32_t kCopies, bool kAny>
__global__ __launch_bounds__(kThreads) void select_keys_kernel(SelectKeysArgs a) {
  __shared__ SelectScratch<kThreads, kCopies> s;
  const uint32_t pair = blockIdx.x, sequence = pair / a.kv_heads, tid = threadIdx.x;
  const uint32_t length = a.lengths[sequence], keep = a.keep[sequence];
  if (length > a.max_keys) {
    return;
  }
  const uint32_t k = min(keep, length);
  if (k > a.kept_stride) {
    return;
  }
  if (pair % a.kv_heads == 0 && tid == 0) {
    a.kept_lengths[sequence] = k;
  }
  // Positions [0, first) and [end, length) are kept, and `most` of those between.
  const uint32_t last = min(a.last, k), first = min(min(a.first, k - last), length - last);
  const uint32_t end = length - last, most = k - last - first;
  int32_t* kept = a.kept + (size_t)pair * a.kept_stride;
  for (uint32_t i = tid; i < first; i += kThreads) {
    kept[i] = (int32_t)i;
  }
  for (uint32_t i = tid; i < last; i += kThreads) {
    kept[k - last + i] = (int32_t)(end + i);
  }
  const float* weights = a.weights + (size_t)pair * a.weight_stride + first;
  if (most == 0) {
    return;
  }
  if (!kAny || end - first <= kHeld * kThreads) {
    select_between<kThreads, kCopies, true>(weights, end - first, most, first, kept + first, s);
  } else {
    select_between<kThreads, kCopies, false>(weights, end - first, most, first, kept + first, s);
  }
}

constexpr uint32_t kGatherThreads = 256;
constexpr uint32_t kGatherWaves = kGatherThreads / 64u;

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// A code times a ratio, rounded to even, in the low byte: an addition of 3 2^22 leaves the
// whole number there.  (At most 127 in size: no source's scale passes its new page's.)
__device__ __forceinline__ uint32_t rescaled(int code, float ratio) {
#pragma clang fp contract(off)
  const float x = (float)code * ratio;
  return __float_as_uint(x + 12582912.0f);
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u),
                               __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

__device__ __forceinline__ int code_at(uint32_t word, uint32_t byte) {
  return (int)(word << (24u - 8u * byte)) >> 24;
}

// One workgroup a target page, KV head, and of keys and values: the two have scales of their
// own.  A key's row is contiguous, 16 lanes of 16 bytes (head_dim 256) with one ratio.  Of
// values eight tokens lie side by side for each dimension, in the source as in the target: a
// wave builds a target run, a lane one dimension or two at a time from the eight sources' eight
// bytes each, of which it takes one.  The sources are the wave's, so that places, bytes and
// ratios are scalars.
//
// 4096 positions of each of 16 sequences of 8192 to 32768, two heads of 256: 62 us.  The keys
// are 34 MB to read and 34 to write, and 29 us by themselves; of the values 130 MB are read,
// the runs of eight that hold any, and 34 written.  Each load waits for the one that
// tells its place, four deep, and then for all of a page.  Asking for the rows before the
// page's scale is known took 67 us (its registers cost a wave in four), workgroups of 128 or
// 512 threads and stores or loads past the caches between 60 and 75.
template <int D>
__global__ __launch_bounds__(kGatherThreads) void gather_pages_kernel(GatherPagesArgs a,
                                                                      uint64_t items) {
  __shared__ uint2 places[128];  // of the source's row, or run of eight: its offset in bytes
  __shared__ uint32_t slots[128];  // in its page; kNone: there is none
  __shared__ float ratios[128];
  __shared__ float most[kGatherWaves];
  __shared__ uint32_t bad[kGatherWaves];
  constexpr uint32_t kNone = 0xffffffffu;
  const PagedQ8Args& c = a.cache;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, shift = c.page_shift;
  const uint32_t page_tokens = 1u << shift;
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    __syncthreads();
    const bool of_values = item % 2u != 0u;
    const uint64_t page_item = item / 2u;
    const uint32_t head = (uint32_t)(page_item % c.kv_heads);
    const uint64_t rest = page_item / c.kv_heads;
    const uint32_t p = (uint32_t)(rest % a.target_width);
    const uint32_t sequence = (uint32_t)(rest / a.target_width);
    const uint64_t pair = (uint64_t)sequence * c.kv_heads + head;
    const uint32_t n = a.kept_lengths[sequence];
    const uint64_t begin = (uint64_t)p << shift;
    if (begin >= n || n > a.kept_stride || n > (uint64_t)a.target_width << shift ||
        (a.weights != nullptr && n > a.weight_stride)) {
      continue;
    }
    const int32_t target = a.target_table[(size_t)sequence * a.target_width + p];
    const bool writes = target >= 0 && (uint32_t)target < c.pages;
    float scale = 0.0f;
    uint32_t slot = kNone;
    uint64_t place = 0;
    if (tid < page_tokens && begin + tid < n) {
      const int32_t position = a.kept[pair * a.kept_stride + begin + tid];
      if (a.weights != nullptr && !of_values) {
        const float* weights = a.weights + pair * a.weight_stride;
        a.weights_output[pair * a.weight_stride + begin + tid] =
          position >= 0 && (uint32_t)position < a.weight_stride ? weights[position] : 0.0f;
      }
      if (position >= 0 && (uint32_t)position >> shift < a.width) {
        const int32_t page = a.table[(size_t)sequence * a.width + ((uint32_t)position >> shift)];
        if (page >= 0 && (uint32_t)page < c.pages) {
          slot = (uint32_t)position & (page_tokens - 1u);
          place = (((uint64_t)page * c.kv_heads + head) << shift) * D +
                  (of_values ? slot / 8u * (8u * D) : slot * D);
          scale = (of_values ? c.value_scales : c.key_scales)[(size_t)page * c.kv_heads + head];
        }
      }
    }
    const bool not_finite = !finite(scale);
    const float largest = halves_max(across8_max(reduce8_max(not_finite ? 0.0f : scale)));
    const uint64_t spoiled = __ballot(not_finite);
    if (lane == 0) {
      most[wave] = largest;
      bad[wave] = spoiled != 0;
    }
    __syncthreads();
    if (!writes) {
      continue;
    }
    float page_scale = most[0];
    uint32_t any = bad[0];
#pragma unroll
    for (uint32_t w = 1; w < kGatherWaves; ++w) {
      page_scale = fmaxf(page_scale, most[w]);
      any |= bad[w];
    }
    if (tid < page_tokens) {
      places[tid] = make_uint2((uint32_t)place, (uint32_t)(place >> 32));
      slots[tid] = slot;
      // Of a page that becomes NaN, and of equal scales (zeros too), the codes stay.
      ratios[tid] = scale == page_scale || any != 0 ? 1.0f : scale / page_scale;
    }
    const size_t page_head = (size_t)target * c.kv_heads + head;
    if (tid == 0) {
      (of_values ? c.value_scales : c.key_scales)[page_head] = any != 0 ? NAN : page_scale;
    }
    __syncthreads();
    if (!of_values) {
      int8_t* to = c.keys + (page_head << shift) * D;
      constexpr uint32_t kLanes = D / 16;  // of a row
      constexpr uint32_t kRows = kGatherThreads / kLanes;
      const uint32_t chunk = tid % kLanes * 16u;
#pragma unroll 4
      for (uint32_t t = tid / kLanes; t < page_tokens; t += kRows) {
        const uint64_t from = (uint64_t)places[t].y << 32 | places[t].x;
        const float ratio = ratios[t];
        u32x4_t x = {0u, 0u, 0u, 0u};
        if (slots[t] != kNone) {
          x = *reinterpret_cast<const u32x4_t*>(c.keys + from + chunk);
        }
        if (ratio != 1.0f) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = low_bytes(rescaled(code_at(x[i], 0), ratio), rescaled(code_at(x[i], 1), ratio),
                             rescaled(code_at(x[i], 2), ratio), rescaled(code_at(x[i], 3), ratio));
          }
        }
        *reinterpret_cast<u32x4_t*>(to + t * D + chunk) = x;
      }
    } else {
      int8_t* to = c.values + (page_head << shift) * D;
      constexpr uint32_t kDims = D == 64 ? 1 : 2;      // of a lane at a time
      constexpr uint32_t kTimes = D / (64u * kDims);
      typedef uint32_t words_t __attribute__((ext_vector_type(2 * kDims)));
      for (uint32_t item = wave; item < page_tokens / 8u * kTimes; item += kGatherWaves) {
        const uint32_t run = item / kTimes, d = (item % kTimes * 64u + lane) * (8u * kDims);
        words_t x[8];
        uint32_t at[8];
        float ratio[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
          const uint32_t t = 8u * run + i;
          at[i] = (uint32_t)__builtin_amdgcn_readfirstlane((int)slots[t]);
          ratio[i] =
            __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(ratios[t])));
          const uint64_t from =
            (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)places[t].y) << 32 |
            (uint32_t)__builtin_amdgcn_readfirstlane((int)places[t].x);
          x[i] = words_t{};
          if (at[i] != kNone) {  // uniform
            x[i] = *reinterpret_cast<const words_t*>(c.values + from + d);
          }
        }
        words_t out;
#pragma unroll
        for (uint32_t w = 0; w < 2u * kDims; ++w) {  // tokens 4 (w % 2) on of dimension w / 2
          uint32_t y[4];
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t token = 4u * (w % 2u) + i;
            const uint32_t word =
              (at[token] & 4u) != 0u ? x[token][w / 2u * 2u + 1u] : x[token][w / 2u * 2u];
            y[i] = rescaled(code_at(word, at[token] & 3u), ratio[token]);
          }
          out[w] = low_bytes(y[0], y[1], y[2], y[3]);
        }
        *reinterpret_cast<words_t*>(to + (size_t)run * (8u * D) + d) = out;
      }
    }
  }
}

}  // namespace

hipError_t launch_select_keys(const SelectKeysArgs& a, hipStream_t stream) {
  const dim3 pairs(a.sequences * a.kv_heads);
  // By the keys that the threads can hold: barriers and scans of half the waves are sooner done
  // (one pair: 512 keys 8.7 us and 11.4, 4096 10.1 and 12.1, 16384 15.6 and 15.7).
  if (a.max_keys <= kHeld * 512u) {
    select_keys_kernel<512, 2, false><<<pairs, 512, 0, stream>>>(a);
  } else {
    select_keys_kernel<1024, 4, true><<<pairs, 1024, 0, stream>>>(a);
  }
  return hipGetLastError();
}

hipError_t launch_gather_pages(const GatherPagesArgs& a, hipStream_t stream) {
  const uint64_t items = 2u * (uint64_t)a.sequences * a.cache.kv_heads * a.target_width;
  const dim3 blocks((uint32_t)std::min<uint64_t>(items, uint64_t{1} << 20));
  if (a.cache.head_dim == 256u) {
    gather_pages_kernel<256><<<blocks, kGatherThreads, 0, stream>>>(a, items);
  } else if (a.cache.head_dim == 128u) {
    gather_pages_kernel<128><<<blocks, kGatherThreads, 0, stream>>>(a, items);
  } else {
    gather_pages_kernel<64><<<blocks, kGatherThreads, 0, stream>>>(a, items);
  }
  return hipGetLastError();
}

}  // namespace kraken
