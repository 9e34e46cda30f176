// Parts shared by the attention kernels over 8-bit KV pages: codes as f16, query rows
// as f16 parts, the softmax's bookkeeping and where split results lie.
//
// The arithmetic.  A code is an integer of at most 8 bits, exact in f16, so the matrix
// cores take the codes themselves and the scales go elsewhere: a key page's scale into
// the score (one multiply that the softmax scale needs anyhow), a value page's scale
// sv = 2^b into the weight's exponent.  With a = score in log2 units, the running maximum
// M is kept of a + b, not of a, and the weight that multiplies the codes is 2^(a + b - M),
// at most 1 however far apart the scales of neighbouring pages lie; the softmax's sum
// takes its quotient with sv.  M follows the largest score only when that leads it by
// more than four octaves, which after the first keys it hardly does: the sums in
// registers (64 to 128 of them a lane) are seldom rescaled.  Weights, up to 2^4 then, are
// formed times 2^11 for f16: below its smallest normal value lies what is 2^-25 of the
// largest, and below its last place 2^-35.
// A query row is multiplied by the power of two that takes its largest value to
// [2^13, 2^14) and goes in as two f16 parts (hi, and what hi leaves), which holds 22
// bits of each value down to 2^-16 of the row's largest; the weights likewise.  f16
// queries are exact in the one part (what lies below 2^-38 of the row's largest aside).
// Their weights take one part too where it saves a product (tiles, blocks of 16 rows), in
// which each is off by at most 2^-12 of itself: the f16 output is then 2.23e-4 of itself off,
// by its own rounding alone 2.07e-4.  Two parts bring the latter and cost 1024 rows at 8192
// keys 118 us instead of 100, a batch of 17 sequences 65.6 instead of 61.3.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "device_common.hpp"
#include "paged_q8_internal.hpp"

namespace kraken {

// Below every score that counts; a running maximum starts here, so that a masked
// score's -inf gives a weight of 0 and not NaN.
constexpr float kLowestMax = -1e30f;
constexpr float kWeightShift = 11.0f;
constexpr float kMaxLead = 4.0f;

// Rows (new tokens x query heads per KV head) of a batch's largest sequence up to which the
// decode kernel takes all of it, in blocks of 16 that read the keys again (32 rows, 64
// sequences of up to 4096 keys: 99 us, by tiles 120; 48 rows 135 and 122).  In a batch with
// larger ones it takes the sequences of one block, the tiled kernel the others (32 rows
// there: 51 us instead of 46 for 24 sequences of up to 80 rows).
constexpr uint32_t kDecodeRows = 32;
constexpr uint32_t kDecodeBlock = 16;
// Rows of the tiled kernel's workgroups: 32 a wave.
constexpr uint32_t kTileRows = 128;

// How a call's keys are split, and where the partial results lie: f32 sums [D] and
// (M, l) of row r of (split, sequence, KV head) for the decode kernel, of (split, token,
// head) for the tiled one.
struct PagedSplit {
  uint32_t decode_most;   // rows of a sequence up to which the decode kernel takes it
  uint32_t decode_keys;   // keys per workgroup of the decode kernel
  uint32_t decode_rows;   // rows held per (split, sequence, KV head)
  uint32_t decode_splits;
  uint32_t tile_keys;     // keys per workgroup of the tiled kernel, the least if it chooses
  uint32_t tile_step;     // how far apart its choices are; 0: tile_keys it is
  uint32_t tile_slots;    // its workgroups that run at once
  uint32_t tile_splits;
  uint32_t tile_blocks;   // its workgroups, as many as a batch can need
  float* decode_o;
  float* decode_ml;
  float* tile_o;
  float* tile_ml;
  uint32_t* tile_chosen;  // the keys that it chose, for the join
};

// Four codes (one dword, two's complement) as f16.  0x64uu is 1024 + uu in f16, so a
// code offset to uu = code + 128 needs one byte permute for two values and one packed
// subtraction of 1152.
__device__ __forceinline__ half4_t codes_to_f16(uint32_t x) {
  x ^= 0x80808080u;
  const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);
  const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);
  const half2_t bias = {(half_t)-1152.0f, (half_t)-1152.0f};
  const half2_t a = __builtin_bit_cast(half2_t, lo) + bias;
  const half2_t b = __builtin_bit_cast(half2_t, hi) + bias;
  return half4_t{a[0], a[1], b[0], b[1]};
}

__device__ __forceinline__ half8_t codes_to_f16(uint32_t x, uint32_t y) {
  const half4_t a = codes_to_f16(x), b = codes_to_f16(y);
  return half8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// A value page's scale as what its weights are formed with.
struct ValueScale {
  float exponent;  // b
  float inverse;   // 2^-b, for the softmax's sum
};

// Not below the least that the prologue makes, so that the sum of quotients stays finite.
// (A NaN stays one.)
__device__ __forceinline__ ValueScale value_scale(float s) {
  const float held = s < kLeastScale ? kLeastScale : s;
  return {log2f(held), 1.0f / held};
}

// The exponent that takes a row's largest magnitude to [2^13, 2^14).
__device__ __forceinline__ int query_exponent(float largest) {
  return largest > 0.0f ? 14 - __builtin_amdgcn_frexp_expf(largest) : 0;
}

// Two f32 as f16: hi rounded towards zero, lo what it leaves.
__device__ __forceinline__ void split_pair(float x, float y, half2_t& hi, half2_t& lo) {
  hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(x, y));
  lo = __builtin_bit_cast(
    half2_t, __builtin_amdgcn_cvt_pkrtz(x - (float)hi[0], y - (float)hi[1]));
}

template <class T>
__device__ __forceinline__ void load4(const T* p, float v[4]) {
  if constexpr (std::is_same<T, float>::value) {
    const float4_t x = *reinterpret_cast<const float4_t*>(p);
    v[0] = x[0];
    v[1] = x[1];
    v[2] = x[2];
    v[3] = x[3];
  } else {
    const half4_t x = *reinterpret_cast<const half4_t*>(p);
    v[0] = x[0];
    v[1] = x[1];
    v[2] = x[2];
    v[3] = x[3];
  }
}

// The gate's factors of outputs at .. at + N - 1 (1 without a gate).  Asked for before the
// first output is stored, since the compiler has to keep a load behind a store that might
// be to the same place (256 rows without older keys: 44 us one value at a time).
template <class T, int N>
__device__ __forceinline__ void gate_factors(const PagedAttentionArgs& a, size_t at,
                                             float (&factor)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    factor[i] = 1.0f;
  }
  if constexpr (std::is_same<T, float>::value) {
    if (a.gate != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        factor[i] = a.gate[at + i];
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        factor[i] = 1.0f / (1.0f + expf(-factor[i]));
      }
    }
  }
}

// out = sum / l, gated.  A sum without any key (l = 0) is zero.
template <class T, int N>
__device__ __forceinline__ void store_outputs(const PagedAttentionArgs& a, size_t at,
                                              const float (&sum)[N], float inverse,
                                              const float (&factor)[N]) {
  typedef T packed_t __attribute__((ext_vector_type(N)));
  packed_t x;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = static_cast<T>(sum[i] * inverse * factor[i]);
  }
  *reinterpret_cast<packed_t*>(static_cast<T*>(a.output) + at) = x;
}

template <class T>
__device__ __forceinline__ void store_output(const PagedAttentionArgs& a, size_t at, float sum,
                                             float inverse) {
  float factor[1];
  gate_factors<T>(a, at, factor);
  static_cast<T*>(a.output)[at] = static_cast<T>(sum * inverse * factor[0]);
}

// 1 / l; l = 0: no key, NaN: NaN.
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

void launch_attention_paged_q8_tiles(const PagedAttentionArgs& a, const PagedSplit& split,
                                     hipStream_t stream);

}  // namespace kraken
