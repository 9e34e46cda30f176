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
// its chunks.  512 rows of 248320 logits take 80 us, a read of their 509 MB at 6.4 TB/s (100 us
// with twice the operations on each logit); one row with 5 places 9.4 us, the two launches and
// what each waits for; 64 rows of 32000 with 20 places 13.1 us.
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
// Logits of a thread.  (512 rows of 248320: 8 84.6 us, 16 77.7, 32 75.3; 8 of them, with 20
// places: 16.0, 14.2, 15.2; one, with 5: 10.2, 10.5, 12.0.)
constexpr uint32_t kPer = 16;
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
  uint64_t* lists;  // [rows][top][chunks]: falling keys of each chunk
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

__device__ __forceinline__ float wave_max(float x) {
  return halves_max(across8_max(reduce8_max(x)));
}

template <int kCtrl>
__device__ __forceinline__ uint64_t quad_max(uint64_t x) {
  const uint64_t y =
    (uint64_t)(uint32_t)__builtin_amdgcn_mov_dpp((int)(x >> 32), kCtrl, 0xf, 0xf, true) << 32 |
    (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kCtrl, 0xf, 0xf, true);
  return x > y ? x : y;
}

constexpr uint32_t kGroups = kThreads / 4u;
constexpr uint32_t kCandidates = kMaxTopLogprobs * 4u * kPer;  // all that a chunk can have

struct TopScratch {
  uint64_t groups[kGroups], candidates[kCandidates], s[kWaves];
  uint32_t ranks[kWaves][kGroups];
  uint32_t count;
};

// The next `top` places below one another of the workgroup's, whose best below `bound`
// best(bound) gives, as list[0..top); 0 where none is left.
template <class Best>
__device__ __forceinline__ void list_by_rounds(uint64_t* list, uint32_t top, uint64_t* s,
                                               Best best) {
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

// Candidates for the `top` first of the workgroup's places (all distinct), as s.candidates,
// and their number.  `mine`: the first of the thread's, 0 for none; from(bound, take) hands
// the thread's of at least `bound` to take.
//
// The first places of 64 groups of threads are ranked: `top` of them, and so `top` places,
// reach the one of rank top - 1, so that no place below it counts, and those that reach it lie
// in `top` groups.  They are few where groups are alike (20 of 64 groups: 24 places).
template <class From>
__device__ __forceinline__ uint32_t collect(uint32_t top, uint64_t mine, TopScratch& s,
                                            From from) {
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint64_t first = quad_max<0x4e>(quad_max<0xb1>(mine));
  __syncthreads();
  if (tid % 4u == 0) {
    s.groups[tid / 4u] = first;
  }
  if (tid == 0) {
    s.count = 0;
  }
  __syncthreads();
  const uint64_t group = s.groups[lane];
  uint32_t rank = 0;
#pragma unroll
  for (uint32_t i = 0; i < kGroups / kWaves; ++i) {  // of every group, against a wave's share
    rank += s.groups[tid / 64u * (kGroups / kWaves) + i] > group ? 1u : 0u;
  }
  s.ranks[tid / 64u][lane] = rank;
  __syncthreads();
  rank = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    rank += s.ranks[w][lane];
  }
  const uint64_t last = __ballot(group != 0u && rank == top - 1u);
  uint64_t bound = 1;  // fewer groups have any
  if (last != 0u) {
    const int at = __builtin_ctzll(last);
    bound = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(group >> 32), at) << 32 |
            (uint32_t)__builtin_amdgcn_readlane((int)group, at);
  }
  if (mine >= bound) {
    from(bound, [&](uint64_t place) {
      const uint32_t slot = atomicAdd(&s.count, 1u);
      if (slot < kCandidates) {
        s.candidates[slot] = place;
      }
    });
  }
  __syncthreads();
  return s.count;
}

// The `top` first of the workgroup's places in order as list[0], list[stride] ..; 0 where none
// is left.  best(bound), for where there can be more candidates than LDS holds, is the thread's
// first below `bound`.
//
// More candidates than threads are bounded again, in whatever order they have come: half of
// the groups have no more than half of them.  (64 rows of 32000, 20 places: 13.1 us, and 32.2
// by 20 rounds of the largest that is left in a workgroup, which stays for a row's lists that
// do not fit.)
template <class From, class... Best>
__device__ __forceinline__ void list_top(uint64_t* list, size_t stride, uint32_t top,
                                         uint64_t mine, TopScratch& s, From from, Best... best) {
  const uint32_t tid = threadIdx.x;
  uint32_t count = collect(top, mine, s, from);
  while (count > kThreads && (sizeof...(best) == 0 || count <= kCandidates)) {
    uint64_t x[kCandidates / kThreads];
    mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < kCandidates / kThreads; ++i) {
      const uint32_t at = i * kThreads + tid;
      x[i] = at < count ? s.candidates[at] : 0u;
      mine = x[i] > mine ? x[i] : mine;
    }
    count = collect(top, mine, s, [&](uint64_t bound, auto take) {
#pragma unroll
      for (uint32_t i = 0; i < kCandidates / kThreads; ++i) {
        if (x[i] >= bound) {
          take(x[i]);
        }
      }
    });
  }
  if (count <= kThreads) {
    const uint64_t place = tid < count ? s.candidates[tid] : 0u;
    uint32_t rank = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < count; ++i) {
      rank += s.candidates[i] > place ? 1u : 0u;
    }
    if (tid < count && rank < top) {
      list[rank * stride] = place;
    }
    if (tid >= count && tid < top) {
      list[tid * stride] = 0;
    }
  } else {
    (list_by_rounds(list, top, s.s, best), ...);
  }
}

// A chunk's logits are in registers, kPer a thread.  What every logit costs bounds the kernel
// next to its bytes, so that it is a maximum, an exponential with five operations about it, and
// a comparison: what few need (ties with the largest, the order of the given token's equals,
// the candidates' places) stands aside under conditions of a wave or workgroup.
__global__ __launch_bounds__(kThreads) void logprob_chunk_kernel(LogprobsArgs a, LogprobPlan p) {
  __shared__ TopScratch s;
  __shared__ float tops[kWaves], sums[kWaves][2];
  __shared__ uint32_t counts[kWaves][2];
  const uint32_t row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const float* logits = a.logits + (size_t)row * a.row_stride;
  const uint32_t begin = chunk * p.chunk, end = min(a.size, begin + p.chunk);
  // NaN stands for what is not there.
  float x[kPer];
  if (begin + kPer * kThreads <= a.size) {
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      x[i] = __builtin_nontemporal_load(logits + begin + i * kThreads + tid);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      const uint32_t at = begin + i * kThreads + tid;
      x[i] = at < end ? logits[at] : NAN;
    }
  }
  const float twice = 2.0f * kLog2e / temperature_of(a, row);
  const uint32_t token = a.tokens != nullptr ? (uint32_t)a.tokens[row] : a.size;
  const float given = token < a.size ? logits[token] : 0.0f;
  float mine = -INFINITY;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    mine = fmaxf(mine, x[i]);
  }
  float top = wave_max(mine);
  if ((tid & 63u) == 0) {
    tops[wave] = top;
  }
  __syncthreads();
  top = tops[0];
#pragma unroll
  for (uint32_t w = 1; w < kWaves; ++w) {
    top = fmaxf(top, tops[w]);
  }
  const float half_top = 0.5f * top;
  float others = 0.0f, moment = 0.0f;
  uint32_t equal = 0, before = 0;
  if (__ballot(mine == top) == 0u) {
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      const float y = exponent_of(x[i], half_top, twice), w = fast_exp2(y);
      others += w;
      moment = fmaf(w, y, moment);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      const float y = exponent_of(x[i], half_top, twice), w = fast_exp2(y);
      const uint64_t is_top = __ballot(x[i] == top);
      equal += (uint32_t)__popcll(is_top);
      others += x[i] == top ? 0.0f : w;
      moment = fmaf(w, x[i] == top ? 0.0f : y, moment);
    }
  }
  if (token < a.size) {
    if (given == given && end <= token) {
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) {
        before += (uint32_t)__popcll(__ballot(x[i] >= given));
      }
    } else if (given == given && begin > token) {
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) {
        before += (uint32_t)__popcll(__ballot(x[i] > given));
      }
    } else {
      const uint64_t place = place_of(token, given);
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t at = begin + i * kThreads + tid;
        before += (uint32_t)__popcll(__ballot(at < end && place_of(at, x[i]) > place));
      }
    }
  }
  others = wave_sum(others);
  moment = wave_sum(moment);
  if ((tid & 63u) == 0) {
    sums[wave][0] = others;
    sums[wave][1] = moment;
    counts[wave][0] = equal;
    counts[wave][1] = before;
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
    uint64_t first = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      const uint32_t j = kPer - 1u - i;
      first = x[j] == mine ? place_of(begin + j * kThreads + tid, mine) : first;
    }
    list_top(
      p.lists + (size_t)row * p.chunks * a.top + chunk, p.chunks, a.top, first, s,
      [&](uint64_t bound, auto take) {
        const uint32_t key = (uint32_t)(bound >> 32);
        const float least = key != 0u ? logit_of(key) : -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) {
          if (x[i] >= least) {
            const uint64_t at = place_of(begin + i * kThreads + tid, x[i]);
            if (at >= bound) {
              take(at);
            }
          }
        }
      });
  }
}

// The first wave joins the chunks' parts; all list.
__global__ __launch_bounds__(kThreads) void logprob_row_kernel(LogprobsArgs a, LogprobPlan p) {
  __shared__ TopScratch s;
  __shared__ uint64_t list[kMaxTopLogprobs];
  __shared__ float joined[2];  // the largest logit, log(1 + S)
  const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid & 63u;
  const float t = temperature_of(a, row), twice = 2.0f * kLog2e / t;
  auto logprob = [&](float logit, float top, float log_sum) {
    if (!(top > -INFINITY) || logit != logit || logit == -INFINITY) {
      return -INFINITY;
    }
    // (Below an infinite logit -inf whatever the temperature, which may be infinite too.)
    const float half = logit == top ? 0.0f : fmaf(logit, 0.5f, -0.5f * top);
    return (half == -INFINITY ? half : half / t * 2.0f) - log_sum;
  };
  if (tid < 64u) {
    const uint32_t token = a.tokens != nullptr ? (uint32_t)a.tokens[row] : a.size;
    const float given = token < a.size ? a.logits[(size_t)row * a.row_stride + token] : 0.0f;
    const Part* parts = p.parts + (size_t)row * p.chunks;
    float top = -INFINITY;
    for (uint32_t c = lane; c < p.chunks; c += 64u) {
      top = fmaxf(top, parts[c].top);
    }
    top = wave_max(top);
    const bool any = top > -INFINITY;
    float others = 0.0f, moment = 0.0f;
    uint32_t equal = 0, before = 0;
    for (uint32_t c = lane; c < p.chunks; c += 64u) {
      const Part part = parts[c];
      before += part.before;
      if (part.top > -INFINITY) {
        const bool is_top = part.top == top;
        const float e = is_top ? 0.0f : exponent_of(part.top, 0.5f * top, twice);
        const float w = fast_exp2(e), all = 1.0f + part.others;
        equal += is_top ? 1u : 0u;
        others += is_top ? part.others : all * w;
        moment += fmaf(e, all, part.moment) * w;
      }
    }
    equal = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(equal, Sum{}), 63);
    before = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(before, Sum{}), 63);
    others = wave_sum(others) + (any ? (float)(equal - 1u) : 0.0f);
    moment = wave_sum(moment);
    const float log_sum = log1pf(others);
    if (lane == 0) {
      joined[0] = top;
      joined[1] = log_sum;
      const bool real = token < a.size;
      if (a.logprobs != nullptr) {
        a.logprobs[row] = real ? logprob(given, top, log_sum) : -INFINITY;
      }
      if (a.ranks != nullptr) {
        a.ranks[row] = (int32_t)(real ? before : a.size);
      }
      if (a.entropies != nullptr) {
        // (S passes f32's largest for no row: it counts at most 2^22.)
        a.entropies[row] =
          any ? log_sum - moment * 0.69314718055994531f / (1.0f + others) : 0.0f;
      }
    }
  }
  if (a.top != 0u) {
    const uint64_t* lists = p.lists + (size_t)row * p.chunks * a.top;
    const uint32_t places = p.chunks * a.top;
    auto best = [&](uint64_t bound) {
      uint64_t found = 0;
      for (uint32_t i = tid; i < places; i += kThreads) {
        const uint64_t at = lists[i];
        found = at < bound && at > found ? at : found;
      }
      return found;
    };
    list_top(
      list, 1, a.top, best(~uint64_t{0}), s,
      [&](uint64_t bound, auto take) {
        for (uint32_t i = tid; i < places; i += kThreads) {
          const uint64_t at = lists[i];
          if (at >= bound) {
            take(at);
          }
        }
      },
      best);
    __syncthreads();
    if (tid < a.top) {
      const uint64_t found = list[tid];
      const size_t at = (size_t)row * a.top + tid;
      if (a.top_tokens != nullptr) {
        a.top_tokens[at] = (int32_t)(found != 0u ? ~(uint32_t)found : a.size);
      }
      if (a.top_logprobs != nullptr) {
        a.top_logprobs[at] = found != 0u ? logprob(logit_of((uint32_t)(found >> 32)), joined[0],
                                                   joined[1])
                                         : -INFINITY;
      }
    }
  }
}

LogprobPlan plan_of(const LogprobsArgs& a) {
  LogprobPlan p{};
  p.chunk = kPer * kThreads;
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
  logprob_chunk_kernel<<<dim3(p.chunks, a.rows), kThreads, 0, stream>>>(a, p);
  logprob_row_kernel<<<dim3(a.rows), kThreads, 0, stream>>>(a, p);
  return hipGetLastError();
}

}  // namespace kraken
