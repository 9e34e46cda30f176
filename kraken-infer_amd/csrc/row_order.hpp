// What the kernels over rows of numbers share: keys that order as the numbers do, and
// reductions and scans over a wave and a workgroup.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace kraken {

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

}  // namespace kraken
