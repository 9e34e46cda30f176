// Causal attention of a ragged batch over 8-bit KV pages: the sequences that bring many
// rows (chunks of prompts).  The arithmetic is described in
// attention_paged_q8_common.hpp.
//
// A workgroup takes 128 rows (token x query head) of one KV head of one sequence, 32 a
// wave, and a run of its keys, a tile of kKeys at a time.  The next tile's codes are on
// their way into registers while a tile is multiplied; they become f16 as they go into
// LDS, once for the four waves.  Both products are transposed, S^T = K Q^T and
// O^T += V^T P^T (32x32x16), so that a query row is a lane: its maximum and sum are
// lane values that two lanes share.  The key rows of a product are read in an order that
// gives a lane the scores of whole runs of eight keys, which is the operand that P has to
// be, and the order in which the pages keep the values.  f32 queries and weights are two
// f16 parts: a second product with the same operand from LDS.
#include <hip/hip_runtime.h>

#include "attention_paged_q8_common.hpp"
#include "device_common.hpp"

namespace kraken {
namespace {

constexpr uint32_t kThreads = 256;

template <int D, class T, int kKeys, int kWavesPerSimd>
__global__ __launch_bounds__(kThreads, kWavesPerSimd) void attention_paged_tile_kernel(
  PagedAttentionArgs a, PagedSplit split) {
  constexpr bool kTwo = std::is_same<T, float>::value;
  constexpr int kStride = D + 8;                   // of a key row in LDS, in halves
  constexpr int kGranules = kKeys / 16;            // runs of 16 keys: of one page each
  constexpr int kChunks = kKeys * D / 16 / 256;    // 16-byte chunks of K, and of V, a thread
  constexpr int kSub = kKeys / 32;                 // 32-key products a tile
  constexpr int kBuffer = kKeys * kStride + kKeys * D;
  static_assert(kChunks >= 1, "a tile has a chunk for every thread");
  __shared__ __attribute__((aligned(16))) half_t lds[2 * kBuffer];

  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t n = lane & 31u, h = lane >> 5;
  const uint32_t part = blockIdx.x % split.tile_splits, tile = blockIdx.x / split.tile_splits;
  const uint32_t kv_head = blockIdx.y, sequence = blockIdx.z;
  const uint32_t shift = a.cache.page_shift, kv_heads = a.cache.kv_heads;
  const uint32_t group = a.heads / kv_heads;
  const PagedSequence s = paged_sequence(a.batch, sequence, shift);
  const uint32_t rows = s.count * group;
  const uint32_t first_row = tile * kTileRows;
  if (rows <= kDecodeRows || first_row >= rows) {
    return;
  }
  // The keys that the tile's last row sees, of this part.
  const uint32_t before = s.length - s.count;
  const uint32_t last_row = min(first_row + kTileRows, rows) - 1u;
  const uint32_t begin = part * split.tile_keys;
  const uint32_t end = min(before + last_row / group + 1u, begin + split.tile_keys);
  if (begin >= end) {
    return;
  }
  const uint32_t tiles = (end - begin + kKeys - 1u) / kKeys;
  const int32_t* table = a.batch.table + (size_t)sequence * a.batch.width;
  const uint32_t last_page = (s.length - 1u) >> shift;

  const uint32_t wave_row = first_row + wave * 32u;
  const uint32_t row = wave_row + n;
  const bool real = row < rows;
  const uint32_t token = real ? row / group : 0u;
  const uint32_t visible = real ? before + token + 1u : 0u;
  const size_t at = ((size_t)(s.start + token) * a.heads + kv_head * group +
                     (real ? row % group : 0u)) * D;
  // What every row of the wave sees, and what any does.
  const uint32_t open = before + wave_row / group + 1u;
  const uint32_t reach =
    wave_row < rows ? before + (min(wave_row + 32u, rows) - 1u) / group + 1u : 0u;

  // Lane l holds the page of granule l % kGranules of a tile.
  auto pages_of = [&](uint32_t t) {
    const uint32_t key = begin + t * kKeys + 16u * (lane % kGranules);
    return table[min(key >> shift, last_page)];
  };
  u32x4_t k[kChunks], v[kChunks];
  float key_scale = 0.0f, val_scale = 0.0f;
  bool inside = false;
  auto load = [&](uint32_t t, int32_t pages) {
    inside = pages >= 0 && (uint32_t)pages < a.cache.pages;
    const uint32_t held = inside ? (uint32_t)pages : 0u;
    const size_t scale_at = (size_t)held * kv_heads + kv_head;
    key_scale = a.cache.key_scales[scale_at];
    val_scale = a.cache.value_scales[scale_at];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const uint32_t c = tid + 256u * i;
      const uint32_t granule = (uint32_t)__builtin_amdgcn_readfirstlane((int)(c / D));
      const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)held, (int)granule);
      const uint32_t key = begin + t * kKeys + 16u * granule;
      const size_t from =
        ((((size_t)page * kv_heads + kv_head) << shift) + (key & ((1u << shift) - 1u))) * D;
      k[i] = *reinterpret_cast<const u32x4_t*>(a.cache.keys + from + (c % D) * 16u);
      v[i] = *reinterpret_cast<const u32x4_t*>(a.cache.values + from + (c % D) * 16u);
    }
  };

  int32_t pages = pages_of(0);
  // The query rows as operands: dimensions 16 c + 8 h .. + 7 of row n.
  half8_t q_hi[D / 16], q_lo[kTwo ? D / 16 : 1];
  float row_factor;
  {
    const T* p = static_cast<const T*>(a.query) + at + 8u * h;
    float largest = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      float x[8];
      load4(p + 16 * c, x);
      load4(p + 16 * c + 4, x + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        largest = fmaxf(largest, fabsf(x[i]));
      }
    }
    largest = xor32_max(real ? largest : 0.0f);
    const int e = query_exponent(largest);
    row_factor = ldexpf(kLog2e / (D == 64 ? 8.0f : D == 256 ? 16.0f : 11.313708498984761f), -e);
    // Read again (from the caches) rather than held: the operands take their registers.
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      float x[8];
      load4(p + 16 * c, x);
      load4(p + 16 * c + 4, x + 4);
      half8_t hi, lo;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        half2_t u, w;
        split_pair(real ? ldexpf(x[i], e) : 0.0f, real ? ldexpf(x[i + 1], e) : 0.0f, u, w);
        hi[i] = u[0];
        hi[i + 1] = u[1];
        lo[i] = w[0];
        lo[i + 1] = w[1];
      }
      q_hi[c] = hi;
      if constexpr (kTwo) {
        q_lo[c] = lo;
      }
    }
  }
  load(0, pages);
  pages = pages_of(min(1u, tiles - 1u));

  float16_t o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      o[i][j] = 0.0f;
    }
  }
  float top = kLowestMax, sum = 0.0f;
  // Row r of a product is key swap(r): bits 2 and 3 change places.
  const uint32_t key_row = (n & 19u) | (n & 4u) << 1 | (n & 8u) >> 1;

  for (uint32_t t = 0; t < tiles; ++t) {
    half_t* lds_k = lds + (t & 1u) * kBuffer;
    half_t* lds_v = lds_k + kKeys * kStride;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const uint32_t c = tid + 256u * i;
      half8_t* to = reinterpret_cast<half8_t*>(lds_k + c / (D / 16) * kStride + c % (D / 16) * 16);
      to[0] = codes_to_f16(k[i][0], k[i][1]);
      to[1] = codes_to_f16(k[i][2], k[i][3]);
      to = reinterpret_cast<half8_t*>(lds_v + c * 16u);
      to[0] = codes_to_f16(v[i][0], v[i][1]);
      to[1] = codes_to_f16(v[i][2], v[i][3]);
    }
    // The tile's scales; its granules' are lane values, read where they are needed.
    const ValueScale sv = value_scale(val_scale);
    const float tile_key_scale = inside ? key_scale : 0.0f;
    const float tile_exponent = inside ? sv.exponent : -INFINITY;
    const float tile_mantissa = inside ? sv.mantissa : 0.0f;
    const float tile_shift = sv.shift;
    // One barrier a tile: a wave that writes this buffer has passed the barrier that
    // every wave reached after it read the same buffer two tiles ago.
    __syncthreads();
    if (t + 1u < tiles) {
      load(t + 1u, pages);
      pages = pages_of(min(t + 2u, tiles - 1u));
    }
    const uint32_t first_key = begin + t * kKeys;
    if (first_key >= reach) {
      continue;  // no row of the wave sees the tile
    }
    float16_t score[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        score[u][j] = 0.0f;
      }
      const half_t* p = lds_k + (32u * u + key_row) * kStride + 8u * h;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const half8_t x = *reinterpret_cast<const half8_t*>(p + 16 * c);
        score[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q_hi[c], score[u], 0, 0, 0);
        if constexpr (kTwo) {
          score[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q_lo[c], score[u], 0, 0, 0);
        }
      }
    }
    auto of = [&](float x, int granule) {
      return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), granule));
    };
    float largest = kLowestMax;
    const bool masked = first_key + kKeys > open;  // uniform
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float factor = row_factor * of(tile_key_scale, 2 * u + b);
        const float offset = of(tile_exponent, 2 * u + b);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          score[u][8 * b + i] = fmaf(score[u][8 * b + i], factor, offset);
        }
        if (masked) {
          const uint32_t key = first_key + 32u * u + 16u * b + 8u * h;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            score[u][8 * b + i] = key + i < visible ? score[u][8 * b + i] : -INFINITY;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          largest = fmaxf(largest, score[u][8 * b + i]);
        }
      }
    }
    largest = xor32_max(largest);
    if (__any(largest > top)) {
      const float up = fmaxf(top, largest);
      const float keep = fast_exp2(top - up);
      top = up;
      sum *= keep;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        o[i] *= keep;
      }
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        // A page that the row does not see at all may have a NaN scale.
        const uint32_t key = first_key + 32u * u + 16u * b + 8u * h;
        float mantissa = of(tile_mantissa, 2 * u + b);
        if (masked) {
          mantissa = key < visible ? mantissa : 0.0f;
        }
        float w[8], all = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = fast_exp2(score[u][8 * b + i] - top);
          all += w[i];
        }
        sum = fmaf(all, of(tile_shift, 2 * u + b), sum);
        half8_t p_hi, p_lo;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          half2_t x, y;
          if constexpr (kTwo) {
            split_pair(w[i] * mantissa, w[i + 1] * mantissa, x, y);
          } else {
            x = half2_t{(half_t)(w[i] * mantissa), (half_t)(w[i + 1] * mantissa)};
            y = x;
          }
          p_hi[i] = x[0];
          p_hi[i + 1] = x[1];
          p_lo[i] = y[0];
          p_lo[i + 1] = y[1];
        }
        const half_t* p = lds_v + ((4u * u + 2u * b + h) * D + n) * 8u;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const half8_t x = *reinterpret_cast<const half8_t*>(p + 256 * i);
          o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p_hi, o[i], 0, 0, 0);
          if constexpr (kTwo) {
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p_lo, o[i], 0, 0, 0);
          }
        }
      }
    }
  }

  if (!real) {
    return;
  }
  sum = xor32_sum(sum);
  // The key count of the sequence decides for all of its rows, as in the join.
  const bool whole = s.length <= split.tile_keys;
  const float inverse = inverse_sum(sum);
  const size_t item = (size_t)part * a.batch.tokens * a.heads + at / D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // Registers 4 j .. + 3 are dimensions 32 i + 8 j + 4 h .. + 3.
      const uint32_t d = 32 * i + 8 * j + 4 * h;
      const float4_t x = {o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
      if (whole) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          store_output<T>(a, at + d + r, x[r], inverse);
        }
      } else {
        *reinterpret_cast<float4_t*>(split.tile_o + item * D + d) = x;
      }
    }
  }
  if (!whole && h == 0) {
    split.tile_ml[2 * item] = top;
    split.tile_ml[2 * item + 1] = sum;
  }
}

template <int D, class T>
void launch_tiles(const PagedAttentionArgs& a, const PagedSplit& split, hipStream_t stream) {
  const uint64_t rows = (uint64_t)a.batch.max_query * (a.heads / a.cache.kv_heads);
  const uint64_t tiles = (rows + kTileRows - 1u) / kTileRows;
  const dim3 grid((uint32_t)(tiles * split.tile_splits), a.cache.kv_heads, a.batch.sequences);
  constexpr int kKeys = D == 64 ? 64 : 32;
  constexpr int kWavesPerSimd = D == 256 && std::is_same<T, float>::value ? 1 : 2;
  attention_paged_tile_kernel<D, T, kKeys, kWavesPerSimd><<<grid, kThreads, 0, stream>>>(a, split);
}

template <class T>
void launch_type(const PagedAttentionArgs& a, const PagedSplit& split, hipStream_t stream) {
  if (a.cache.head_dim == 256u) {
    launch_tiles<256, T>(a, split, stream);
  } else if (a.cache.head_dim == 128u) {
    launch_tiles<128, T>(a, split, stream);
  } else {
    launch_tiles<64, T>(a, split, stream);
  }
}

}  // namespace

void launch_attention_paged_q8_tiles(const PagedAttentionArgs& a, const PagedSplit& split,
                                     hipStream_t stream) {
  if (a.f16) {
    launch_type<half_t>(a, split, stream);
  } else {
    launch_type<float>(a, split, stream);
  }
}

}  // namespace kraken
