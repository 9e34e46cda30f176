// Log probabilities of given tokens, their ranks, the entropy and the likeliest tokens of
// rows of logits.
//
// With M the largest logit of a row, y = (l - M) / T, and over all others
// S = sum e^y, A = sum y e^y:
//   log p = y - log(1 + S),  entropy = log(1 + S) - A / (1 + S).
// The largest logit's own 1 stays out of S, so that where it takes nearly everything S
// keeps its relative accuracy and with it log p and the entropy, both near zero (A is not
// positive: nothing cancels).  Partial sums of chunks join exactly like those of a
// softmax: S1 and S2 under M1 >= M2 to S1 + (1 + S2) e^(M2 - M1).
//
// Two launches: a workgroup for each chunk of a row, then one for each row that joins
// its chunks.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "context_internal.hpp"
#include "device_common.hpp"
#include "paged_q8_internal.hpp"
#include "row_order.hpp"

namespace kraken {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / 64u;
// y in log2 units from which on down a weight is zero in f32 (the product y 2^y too).
constexpr float kLowest = -256.0f;

// The softmax of a part of a row: the largest logit (-inf: none counts), the sum of the
// other weights, the sum of weight times y (log2 units), and how many logits stand before
// the given token.
struct Part {
  float top, others, moment;
  uint32_t before;
};

struct LogprobPlan {
  Part* parts;      // [rows][chunks]
  uint64_t* lists;  // [rows][chunks][top]: falling keys
  uint32_t chunk, chunks;
};

// (l - top) / T in log2 units, with `half_top` = top / 2 and twice = 2 log2(e) / T.  By
// halves, as the difference may pass f32's largest; NaN and -inf count as nothing.
__device__ __forceinline__ float exponent_of(float logit, float half_top, float twice) {
  return fmaxf(fmaf(logit, 0.5f, -half_top) * twice, kLowest);
}

__device__ __forceinline__ float temperature_of(const LogprobsArgs& a, uint32_t row) {
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  return t > 0.0f ? t : 1.0f;  // NaN: 1
}

// Position in the order of falling logits as one number, larger ones first.
__device__ __forceinline__ uint64_t place_of(uint32_t index, float logit) {
  return (uint64_t)key_of(logit) << 32 | (uint32_t)~index;
}

__device__ __forceinline__ Part join(const Part& x, const Part& y, float twice) {
  const Part& hi = x.top >= y.top ? x : y;
  const Part& lo = x.top >= y.top ? y : x;
  Part r = hi;
  r.before = x.before + y.before;
  if (lo.top > -INFINITY) {
    const float e = hi.top == lo.top ? 0.0f : exponent_of(lo.top, 0.5f * hi.top, twice);
    const float w = fast_exp2(e), all = 1.0f + lo.others;
    r.others = fmaf(all, w, hi.others);
    r.moment = fmaf(fmaf(e, all, lo.moment), w, hi.moment);
  }
  return r;
}

// The next `top` places below one another of the workgroup's, whose best below `bound`
// best(bound) gives, as list[0..top); 0 where none is left.
template <class Best>
__device__ __forceinline__ void list_top(uint64_t* list, uint32_t top, uint64_t* s, Best best) {
  uint64_t bound = ~uint64_t{0}, mine = best(bound);
  for (uint32_t i = 0; i < top; ++i) {
    const uint64_t found = block_reduce<kWaves>(mine, Largest{}, s);
    if (threadIdx.x == 0) {
      list[i] = found;
    }
    if (mine == found) {
      mine = best(found);
    }
  }
}

template <uint32_t kPer>
__global__ __launch_bounds__(kThreads) void logprob_chunk_kernel(LogprobsArgs a, LogprobPlan p) {
  __shared__ uint64_t s[kWaves];
  __shared__ float sums[kWaves][2];
  __shared__ uint32_t counts[kWaves][2];
  const uint32_t row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const float* logits = a.logits + (size_t)row * a.row_stride;
  const uint32_t begin = chunk * p.chunk, end = min(a.size, begin + p.chunk);
  const float twice = 2.0f * kLog2e / temperature_of(a, row);
  uint64_t given = 0;
  if (a.tokens != nullptr) {
    const uint32_t token = (uint32_t)a.tokens[row];
    given = token < a.size ? place_of(token, logits[token]) : 0u;
  }
  // NaN stands for what is not there.
  float x[kPer];
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    const uint32_t at = begin + i * kThreads + tid;
    x[i] = at < end ? logits[at] : NAN;
  }
  float top = -INFINITY;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    top = fmaxf(top, x[i]);
  }
  top = logit_of((uint32_t)block_reduce<kWaves>(key_of(top), Largest{}, s));
  float others = 0.0f, moment = 0.0f;
  uint32_t equal = 0, before = 0;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    const float y = exponent_of(x[i], 0.5f * top, twice), w = fast_exp2(y);
    const bool is_top = x[i] == top;
    others += is_top ? 0.0f : w;
    moment += is_top ? 0.0f : w * y;
    equal += is_top ? 1u : 0u;
    const uint32_t at = begin + i * kThreads + tid;
    before += at < end && place_of(at, x[i]) > given ? 1u : 0u;
  }
  others = wave_sum(others);
  moment = wave_sum(moment);
  equal = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(equal, Sum{}), 63);
  before = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(before, Sum{}), 63);
  if ((tid & 63u) == 0) {
    sums[tid >> 6][0] = others;
    sums[tid >> 6][1] = moment;
    counts[tid >> 6][0] = equal;
    counts[tid >> 6][1] = before;
  }
  __syncthreads();
  if (tid == 0) {
    Part r{top, 0.0f, 0.0f, 0u};
    equal = 0;
    for (uint32_t w = 0; w < kWaves; ++w) {
      r.others += sums[w][0];
      r.moment += sums[w][1];
      equal += counts[w][0];
      r.before += counts[w][1];
    }
    r.others += (float)(equal - 1u);
    p.parts[(size_t)row * p.chunks + chunk] =
      top > -INFINITY ? r : Part{-INFINITY, 0.0f, 0.0f, r.before};
  }
  if (a.top != 0u) {
    list_top(p.lists + ((size_t)row * p.chunks + chunk) * a.top, a.top, s, [&](uint64_t bound) {
      uint64_t best = 0;
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) {
        const uint64_t at = place_of(begin + i * kThreads + tid, x[i]);
        best = x[i] == x[i] && at < bound && at > best ? at : best;
      }
      return best;
    });
  }
}

__global__ __launch_bounds__(kThreads) void logprob_row_kernel(LogprobsArgs a, LogprobPlan p) {
  __shared__ uint64_t s[kWaves], list[kMaxTopLogprobs];
  __shared__ Part parts[kThreads];
  const uint32_t row = blockIdx.x, tid = threadIdx.x;
  const float t = temperature_of(a, row), twice = 2.0f * kLog2e / t;
  Part all{-INFINITY, 0.0f, 0.0f, 0u};
  for (uint32_t c = tid; c < p.chunks; c += kThreads) {
    all = join(all, p.parts[(size_t)row * p.chunks + c], twice);
  }
  parts[tid] = all;
  for (uint32_t n = kThreads / 2u; n != 0u; n /= 2u) {
    __syncthreads();
    if (tid < n) {
      parts[tid] = join(parts[tid], parts[tid + n], twice);
    }
  }
  __syncthreads();
  all = parts[0];
  const bool any = all.top > -INFINITY;
  const float log_sum = log1pf(all.others);
  auto logprob = [&](float logit) {
    if (!any || logit != logit || logit == -INFINITY) {
      return -INFINITY;
    }
    const float x = logit == all.top ? 0.0f : fmaf(logit, 0.5f, -0.5f * all.top) / t * 2.0f;
    return x - log_sum;
  };
  if (tid == 0) {
    if (a.tokens != nullptr) {
      const uint32_t token = (uint32_t)a.tokens[row];
      const bool real = token < a.size;
      if (a.logprobs != nullptr) {
        a.logprobs[row] =
          real ? logprob(a.logits[(size_t)row * a.row_stride + token]) : -INFINITY;
      }
      if (a.ranks != nullptr) {
        a.ranks[row] = (int32_t)(real ? all.before : a.size);
      }
    }
    if (a.entropies != nullptr) {
      // (S passes f32's largest for no row: it counts at most 2^22.)
      a.entropies[row] =
        any ? log_sum - all.moment * 0.69314718055994531f / (1.0f + all.others) : 0.0f;
    }
  }
  if (a.top != 0u) {
    const uint64_t* lists = p.lists + (size_t)row * p.chunks * a.top;
    list_top(list, a.top, s, [&](uint64_t bound) {
      uint64_t best = 0;
      for (uint32_t i = tid; i < p.chunks * a.top; i += kThreads) {
        const uint64_t at = lists[i];
        best = at < bound && at > best ? at : best;
      }
      return best;
    });
    __syncthreads();
    if (tid < a.top) {
      const uint64_t found = list[tid];
      const size_t at = (size_t)row * a.top + tid;
      if (a.top_tokens != nullptr) {
        a.top_tokens[at] = (int32_t)(found != 0u ? ~(uint32_t)found : a.size);
      }
      if (a.top_logprobs != nullptr) {
        a.top_logprobs[at] = found != 0u ? logprob(logit_of((uint32_t)(found >> 32))) : -INFINITY;
      }
    }
  }
}

LogprobPlan plan_of(const LogprobsArgs& a) {
  LogprobPlan p{};
  p.chunk = 16u * kThreads;
  p.chunks = (a.size + p.chunk - 1u) / p.chunk;
  return p;
}

}  // namespace

size_t token_logprobs_workspace_bytes(const LogprobsArgs& a) {
  const LogprobPlan p = plan_of(a);
  return (size_t)a.rows * p.chunks * (sizeof(Part) + a.top * sizeof(uint64_t));
}

hipError_t launch_token_logprobs(const LogprobsArgs& a, void* workspace, hipStream_t stream) {
  LogprobPlan p = plan_of(a);
  p.lists = static_cast<uint64_t*>(workspace);
  p.parts = reinterpret_cast<Part*>(p.lists + (size_t)a.rows * p.chunks * a.top);
  logprob_chunk_kernel<16><<<dim3(p.chunks, a.rows), kThreads, 0, stream>>>(a, p);
  logprob_row_kernel<<<dim3(a.rows), kThreads, 0, stream>>>(a, p);
  return hipGetLastError();
}

}  // namespace kraken
