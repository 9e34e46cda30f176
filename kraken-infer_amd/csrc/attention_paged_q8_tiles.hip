// Causal attention of a ragged batch over 8-bit KV pages: the sequences that bring many
// rows (chunks of prompts).  The arithmetic is described in
// attention_paged_q8_common.hpp.
//
// A workgroup takes 128 rows (token x query head) of one KV head of one sequence, 32 a
// wave, and a run of its keys, a tile of kKeys at a time.  The next tile's codes are on
// their way into registers while a tile is multiplied; they become f16 as they go into
// LDS, once for all waves.  Both products are transposed, S^T = K Q^T and
// O^T += V^T P^T (32x32x16), so that a query row is a lane: its maximum and sum are
// lane values that two lanes share.  The key rows of a product are read in an order that
// gives a lane the scores of whole runs of eight keys, which is the operand that P has to
// be, and the order in which the pages keep the values.  f32 queries and weights are two
// f16 parts: a second product with the same operand from LDS.
//
// 1024 rows of 8 heads of 256 at 7169 to 8192 keys: f16 100 us (640 TFLOP/s), f32 144 us
// (900 TFLOP/s of f16 products, two for each).  Of f16's time the vector units are busy for
// 40 % (the softmax, and codes to f16), the matrix cores for 29 %, and waves wait for 26 %
// (one wave a SIMD, so that nothing else runs while it does); the clock falls to 1.9 GHz.
// A workgroup spends 9 us on its query rows and its first tile, and 3 on its results,
// whatever its keys; query rows read whole and handed over in LDS were no faster.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <utility>

#include "attention_paged_q8_common.hpp"
#include "device_common.hpp"

namespace kraken {
namespace {

constexpr int kThreads = 256;

// f(0), f(1), .. f(N - 1) with compile-time indices.
template <class F, int... I>
__device__ __forceinline__ void static_for(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

template <int N, class F>
__device__ __forceinline__ void static_for(F f) {
  static_for(f, std::make_integer_sequence<int, N>{});
}

// The keys of a workgroup, for up to 64 sequences: of sixteen sizes the one whose rounds
// of `tile_slots` workgroups are soonest over, each round taking its keys and what a
// workgroup spends besides (about 128 keys' time).  Every wave comes to the same.
__device__ __forceinline__ uint32_t chosen_keys(const PagedAttentionArgs& a,
                                                const PagedSplit& split, uint32_t group) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t tiles = 0, length = 0;
  if (lane < a.batch.sequences) {
    const PagedSequence s = paged_sequence(a.batch, lane, a.cache.page_shift);
    const uint32_t rows = s.count * group;
    tiles = rows > split.decode_most ? (rows + kTileRows - 1u) / kTileRows : 0u;
    length = s.length;
  }
  uint32_t best = split.tile_keys;
  float least = INFINITY;
#pragma unroll
  for (uint32_t i = 0; i < 16; ++i) {
    const uint32_t keys = split.tile_keys + i * split.tile_step;
    const uint32_t parts = (uint32_t)((float)(length + keys - 1u) / (float)keys);
    const uint32_t all =
      (uint32_t)__builtin_amdgcn_readlane((int)wave_prefix(tiles * parts), 63) *
      a.cache.kv_heads;
    const float rounds = ceilf((float)all / (float)split.tile_slots);
    const float time = rounds * (float)(keys + 128u);
    best = time < least ? keys : best;
    least = fminf(time, least);
  }
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)best);
}

// One part of `part_keys` keys of one tile of rows.  `again`: the workgroup has done
// another before.
template <int D, class T, int kSub>
__device__ __forceinline__ void attention_paged_tile(const PagedAttentionArgs& a,
                                                     const PagedSplit& split,
                                                     const PagedItem& found, uint32_t kv_head,
                                                     uint32_t part_keys, bool again) {
  constexpr bool kTwo = std::is_same<T, float>::value;
  constexpr int kKeys = 32 * kSub;
  constexpr int kStride = D + 8;                      // of a key row in LDS, in halves
  constexpr int kGranules = kKeys / 16;               // runs of 16 keys: of one page each
  constexpr int kChunks = kKeys * D / 16 / kThreads;  // 16-byte chunks of K, and of V, a thread
  constexpr int kSteps = D / 16;                      // of a score product
  constexpr int kDims = D / 32;                       // tiles of the output
  constexpr int kTileK = kKeys * kStride, kTileV = kKeys * D;
  static_assert(kChunks >= 1, "a tile has a chunk for every thread");
  __shared__ __attribute__((aligned(16))) half_t lds[2 * (kTileK + kTileV)];

  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t n = lane & 31u, h = lane >> 5;
  const uint32_t shift = a.cache.page_shift, kv_heads = a.cache.kv_heads;
  const uint32_t group = a.heads / kv_heads;
  const PagedSequence s = found.sequence;
  const uint32_t sequence = found.index;
  const uint32_t parts = (s.length + part_keys - 1u) / part_keys;
  const uint32_t tile = found.item / parts, part = found.item % parts;
  const uint32_t rows = s.count * group;
  const uint32_t first_row = tile * kTileRows;
  // The keys that the tile's last row sees, of this part.
  const uint32_t before = s.length - s.count;
  const uint32_t last_row = min(first_row + kTileRows, rows) - 1u;
  const uint32_t begin = part * part_keys;
  const uint32_t end = min(before + last_row / group + 1u, begin + part_keys);
  if (begin >= end) {
    return;
  }
  const uint32_t tiles = (end - begin + kKeys - 1u) / kKeys;
  const int32_t* table = a.batch.table + (size_t)sequence * a.batch.width;

  const uint32_t wave_row = first_row + wave * 32u;
  const uint32_t row = wave_row + n;
  const bool real = row < rows;
  const uint32_t token = real ? row / group : 0u;
  const uint32_t visible = real ? before + token + 1u : 0u;
  const size_t at = ((size_t)(s.start + token) * a.heads + kv_head * group +
                     (real ? row % group : 0u)) * D;
  // What every row of the wave sees (0: a row without a query sees nothing).
  const uint32_t open = wave_row + 32u <= rows ? before + wave_row / group + 1u : 0u;

  // Lane l holds the page of granule l % kGranules of a tile; past the last tile, the
  // last one's again.
  auto pages_of = [&](uint32_t t) {
    const uint32_t key = begin + min(t, tiles - 1u) * kKeys + 16u * (lane % kGranules);
    return table[min(key >> shift, a.batch.width - 1u)];
  };
  auto held_page = [&](int32_t page) {
    return page >= 0 && (uint32_t)page < a.cache.pages ? (uint32_t)page : 0u;
  };
  u32x4_t k[kChunks], v[kChunks];
  // Where chunk i of tile t lies.
  auto place = [&](uint32_t t, int32_t pages, int i) {
    const uint32_t c = tid + kThreads * i;
    const uint32_t granule = (uint32_t)__builtin_amdgcn_readfirstlane((int)(c / D));
    const uint32_t page =
      (uint32_t)__builtin_amdgcn_readlane((int)held_page(pages), (int)granule);
    const uint32_t key = begin + min(t, tiles - 1u) * kKeys + 16u * granule;
    return ((((size_t)page * kv_heads + kv_head) << shift) + (key & ((1u << shift) - 1u))) * D;
  };
  auto load_k = [&](uint32_t t, int32_t pages, int i) {
    k[i] = *reinterpret_cast<const u32x4_t*>(a.cache.keys + place(t, pages, i) +
                                             (tid + kThreads * i) % D * 16u);
  };
  auto load_v = [&](uint32_t t, int32_t pages, int i) {
    v[i] = *reinterpret_cast<const u32x4_t*>(a.cache.values + place(t, pages, i) +
                                             (tid + kThreads * i) % D * 16u);
  };
  // A tile's scales, a granule a lane; outside the pool NaN stands for none.
  struct Scales {
    float key, value;
    bool inside;
  };
  auto scales_of = [&](int32_t page) {
    const size_t i = (size_t)held_page(page) * kv_heads + kv_head;
    return Scales{a.cache.key_scales[i], a.cache.value_scales[i],
                  page >= 0 && (uint32_t)page < a.cache.pages};
  };
  // Half of a chunk as f16 into LDS.
  auto convert = [&](const u32x4_t& x, half_t* to, int half) {
    *reinterpret_cast<half8_t*>(to + 8 * half) = codes_to_f16(x[2 * half], x[2 * half + 1]);
  };
  half_t* const lds_k = lds;
  half_t* const lds_v = lds + 2 * kTileK;
  auto store_k = [&](int parity, int i, int half) {
    const uint32_t c = tid + kThreads * i;
    convert(k[i], lds_k + parity * kTileK + c / kSteps * kStride + c % kSteps * 16, half);
  };
  auto store_v = [&](int parity, int i, int half) {
    convert(v[i], lds_v + parity * kTileV + (tid + kThreads * i) * 16u, half);
  };

  // By the parity of the tile: the pages of the tiles whose codes are loaded next, and
  // the scales of the tiles whose scores come next.
  int32_t pages[2] = {pages_of(0), pages_of(1)};
  const int32_t third = pages_of(2);
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    load_k(0, pages[0], i);
    load_v(0, pages[0], i);
  }
  Scales scales[2] = {scales_of(pages[0]), scales_of(pages[1])};
  // The query rows as operands: dimensions 16 c + 8 h .. + 7 of row n.
  half8_t q_hi[kSteps], q_lo[kTwo ? kSteps : 1];
  float row_factor;
  {
    const T* p = static_cast<const T*>(a.query) + at + 8u * h;
    float x[kSteps][8], largest = 0.0f;
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      load4(p + 16 * c, x[c]);
      load4(p + 16 * c + 4, x[c] + 4);
    }
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[c][i] = real ? x[c][i] : 0.0f;
        largest = fmaxf(largest, fabsf(x[c][i]));
      }
    }
    largest = xor32_max(largest);
    const int e = query_exponent(largest);
    row_factor = ldexpf(kLog2e / (D == 64 ? 8.0f : D == 256 ? 16.0f : 11.313708498984761f), -e);
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      half8_t hi, lo;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        half2_t u, w;
        split_pair(ldexpf(x[c][i], e), ldexpf(x[c][i + 1], e), u, w);
        hi[i] = u[0];
        hi[i + 1] = u[1];
        lo[i] = w[0];
        lo[i + 1] = w[1];
      }
      q_hi[c] = hi;
      if constexpr (kTwo) {
        q_lo[c] = lo;
      }
      if constexpr (D == 256) {
        // Into accumulator registers, where the products read them: the others are for
        // what the vector units work on.
        asm volatile("" : "+a"(q_hi[c]));
        if constexpr (kTwo) {
          asm volatile("" : "+a"(q_lo[c]));
        }
      }
    }
  }
  if (again) {
    __syncthreads();  // the tiles of the item before are read
  }
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    store_k(0, i, 0);
    store_k(0, i, 1);
    load_k(1, pages[1], i);
  }
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    store_v(0, i, 0);
    store_v(0, i, 1);
    load_v(1, pages[1], i);
  }

  float16_t o[kDims];
#pragma unroll
  for (int i = 0; i < kDims; ++i) {
    o[i] = float16_t{};
  }
  float top = kLowestMax, sum = 0.0f;
  // Row r of a product is key swap(r): bits 2 and 3 change places.
  const uint32_t key_row = (n & 19u) | (n & 4u) << 1 | (n & 8u) >> 1;

  // Fragment i of a tile's keys: step i / kSub, 32-key half i % kSub.
  constexpr int kKeyFrags = kSteps * kSub, kValueFrags = 2 * kSub * kDims, kRing = 4;
  auto key_frag = [&](int parity, int i) {
    return *reinterpret_cast<const half8_t*>(lds_k + parity * kTileK +
                                             (32u * (i % kSub) + key_row) * kStride + 8u * h +
                                             16 * (i / kSub));
  };
  // Fragment i of a tile's values: 16-key step i / kDims, dimensions 32 (i % kDims) on.
  auto value_frag = [&](int parity, int i) {
    return *reinterpret_cast<const half8_t*>(lds_v + parity * kTileV +
                                             ((2u * (i / kDims) + h) * D + n) * 8u +
                                             256 * (i % kDims));
  };
  auto score_product = [&](float16_t (&score)[kSub], const half8_t& x, int i) {
    score[i % kSub] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
      x, q_hi[i / kSub], i < kSub ? float16_t{} : score[i % kSub], 0, 0, 0);
    if constexpr (kTwo) {
      score[i % kSub] =
        __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q_lo[i / kSub], score[i % kSub], 0, 0, 0);
    }
  };

  __syncthreads();
  float16_t scores[2][kSub];
  // The scores of tile 0 while the keys of tile 1 arrive.
  {
    half8_t ring[kRing];
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      ring[i] = key_frag(0, i);
    }
    static_for<kKeyFrags>([&](auto slot) {
      constexpr int i = decltype(slot)::value;
      score_product(scores[0], ring[i % kRing], i);
      if constexpr (i + kRing < kKeyFrags) {
        ring[i % kRing] = key_frag(0, i + kRing);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  }

#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    store_k(1, i, 0);
    store_k(1, i, 1);
    load_k(2, third, i);
  }
  pages[0] = third;
  pages[1] = pages_of(3);

  auto of = [&](float x, int granule) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), granule));
  };
  // Step t.  The scores of tile t are there.  The matrix cores do the scores of tile
  // t + 1 while the vector units turn those of t into weights, then O += V^T P^T of tile
  // t while the codes that arrived (keys of t + 2, values of t + 1) become f16 in LDS and
  // those of the tiles after set out.  One barrier a step: what it publishes was written
  // in the step before, to buffers last read before the barrier before.
  // Registers and buffers go by the parity of t, so that nothing is copied from step to
  // step: a copy of what is still loading would wait for it.
  auto step = [&](auto even_odd, uint32_t t) __attribute__((always_inline)) {
    constexpr int kParity = decltype(even_odd)::value;
    float16_t(&score)[kSub] = scores[kParity];
    float16_t(&next)[kSub] = scores[1 - kParity];
    __syncthreads();
    const uint32_t first_key = begin + t * kKeys;
    const bool masked = first_key + kKeys > open;  // uniform
    const bool more = t + 1u < tiles;              // uniform
    half8_t ring[kRing];
    if (more) {
#pragma unroll
      for (int i = 0; i < kRing; ++i) {
        ring[i] = key_frag(1 - kParity, i);
      }
    }
    // The tile's scales by granule: of the scores, and of the weights.
    const Scales held = scales[kParity];
    const ValueScale sv = value_scale(held.value);
    const float lane_key = held.inside ? held.key : 0.0f;
    const float lane_exponent = held.inside ? sv.exponent : -INFINITY;
    const float lane_inverse = held.inside ? sv.inverse : 0.0f;
    float factor[2 * kSub], exponent[2 * kSub], inverse[2 * kSub];
#pragma unroll
    for (int b = 0; b < 2 * kSub; ++b) {
      // Not zero: a masked score's -inf has to stay one (a NaN stays NaN).
      const float f = row_factor * of(lane_key, b);
      factor[b] = f < 1e-37f ? 1e-37f : f;
      exponent[b] = of(lane_exponent, b);
      inverse[b] = of(lane_inverse, b);
    }
    if (masked) {
#pragma unroll
      for (int b = 0; b < 2 * kSub; ++b) {
        const uint32_t key = first_key + 16u * b + 8u * h;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          score[b / 2][8 * (b % 2) + i] =
            key + i < visible ? score[b / 2][8 * (b % 2) + i] : -INFINITY;
        }
        // A page that the row does not see at all may have NaN scales.
        factor[b] = key < visible ? factor[b] : 1.0f;
        exponent[b] = key < visible ? exponent[b] : 0.0f;
        inverse[b] = key < visible ? inverse[b] : 0.0f;
      }
    }
    __builtin_amdgcn_sched_barrier(0);

    float base[2 * kSub], all[2 * kSub], largest = kLowestMax, keep = 1.0f;
    bool lead = false;
    half8_t p_hi[2 * kSub], p_lo[kTwo ? 2 * kSub : 1];
    // The softmax in pieces, placed after the products of the scores: the largest of
    // each granule (a = score * factor + exponent), their join, and the weights by
    // pairs.  Each ends in an empty asm on its results, without which it would sink to
    // their first use.
    constexpr int kPieces = 2 * kSub + 1 + 8 * kSub;
    auto soft_piece = [&](auto piece) {
      constexpr int kPiece = decltype(piece)::value;
      if constexpr (kPiece < 2 * kSub) {
        constexpr int b = kPiece, r = 8 * (b % 2);
        const float16_t& x = score[b / 2];
        float run = fmaxf(fmaxf(x[r], x[r + 1]), x[r + 2]);
        run = fmaxf(fmaxf(run, x[r + 3]), x[r + 4]);
        run = fmaxf(fmaxf(run, x[r + 5]), x[r + 6]);
        largest = fmaxf(largest, fmaf(fmaxf(run, x[r + 7]), factor[b], exponent[b]));
        asm volatile("" : "+v"(largest));
      } else if constexpr (kPiece == 2 * kSub) {
        largest = xor32_max(largest);
        lead = largest > top + kMaxLead;
        const float up = lead ? largest : top;
        keep = fast_exp2(top - up);
        top = up;
        sum *= keep;
#pragma unroll
        for (int b = 0; b < 2 * kSub; ++b) {
          base[b] = exponent[b] - (top - kWeightShift);
        }
        asm volatile("" : "+v"(top), "+v"(keep), "+v"(sum));
      } else {
        constexpr int b = (kPiece - 2 * kSub - 1) / 4, j = (kPiece - 2 * kSub - 1) % 4;
        constexpr int r = 8 * (b % 2) + 2 * j;
        const float x = fast_exp2(fmaf(score[b / 2][r], factor[b], base[b]));
        const float y = fast_exp2(fmaf(score[b / 2][r + 1], factor[b], base[b]));
        // In f32: a page of small or zero scale counts whole in the sum though its
        // weights vanish in f16.
        all[b] = j == 0 ? x + y : all[b] + (x + y);
        half2_t hi, lo;
        if constexpr (kTwo) {
          split_pair(x, y, hi, lo);
          asm volatile("" : "+v"(hi), "+v"(lo), "+v"(all[b]));
          p_lo[b][2 * j] = lo[0];
          p_lo[b][2 * j + 1] = lo[1];
        } else {
          hi = half2_t{(half_t)x, (half_t)y};
          asm volatile("" : "+v"(hi), "+v"(all[b]));
        }
        if constexpr (j == 3) {
          sum = fmaf(all[b], inverse[b], sum);
          asm volatile("" : "+v"(sum));
        }
        p_hi[b][2 * j] = hi[0];
        p_hi[b][2 * j + 1] = hi[1];
      }
    };
    // Pieces [slot kPieces / slots, (slot + 1) kPieces / slots) after slot `slot`.
    if (more) {
      static_for<kKeyFrags>([&](auto slot) {
        constexpr int i = decltype(slot)::value;
        constexpr int kFrom = i * kPieces / kKeyFrags, kTo = (i + 1) * kPieces / kKeyFrags;
        score_product(next, ring[i % kRing], i);
        if constexpr (i + kRing < kKeyFrags) {
          ring[i % kRing] = key_frag(1 - kParity, i + kRing);
        }
        static_for<kTo - kFrom>([&](auto j) {
          soft_piece(std::integral_constant<int, kFrom + decltype(j)::value>{});
        });
        __builtin_amdgcn_sched_barrier(0);
      });
    } else {
      static_for<kPieces>(soft_piece);
    }

    // O += V^T P^T, and the codes' pieces: halves of K's and V's chunks in turn.
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      ring[i] = value_frag(kParity, i);
    }
    if (__any(lead)) {
#pragma unroll
      for (int i = 0; i < kDims; ++i) {
        o[i] *= keep;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    constexpr int kCodePieces = 4 * kChunks;
    // (Past the last tiles they fill buffers that nothing reads.)
    static_for<kValueFrags>([&](auto slot) {
      constexpr int i = decltype(slot)::value;
      constexpr int kFrom = i * kCodePieces / kValueFrags;
      constexpr int kTo = (i + 1) * kCodePieces / kValueFrags;
      o[i % kDims] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % kRing], p_hi[i / kDims],
                                                            o[i % kDims], 0, 0, 0);
      if constexpr (kTwo) {
        o[i % kDims] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % kRing], p_lo[i / kDims],
                                                              o[i % kDims], 0, 0, 0);
      }
      if constexpr (i + kRing < kValueFrags) {
        ring[i % kRing] = value_frag(kParity, i + kRing);
      }
      static_for<kTo - kFrom>([&](auto piece) {
        constexpr int j = kFrom + decltype(piece)::value, chunk = j / 4, half = j % 2;
        if constexpr (j % 4 < 2) {
          store_k(kParity, chunk, half);  // of tile t + 2
          if constexpr (half == 1) {
            load_k(t + 3u, pages[1 - kParity], chunk);
          }
        } else {
          store_v(1 - kParity, chunk, half);  // of tile t + 1
          if constexpr (half == 1) {
            load_v(t + 2u, pages[kParity], chunk);
          }
        }
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    scales[kParity] = scales_of(pages[kParity]);
    pages[kParity] = pages_of(t + 4u);
  };
  for (uint32_t t = 0;;) {
    step(std::integral_constant<int, 0>{}, t);
    if (++t == tiles) {
      break;
    }
    step(std::integral_constant<int, 1>{}, t);
    if (++t == tiles) {
      break;
    }
  }

  if (!real) {
    return;
  }
  sum = xor32_sum(sum);
  // The key count of the sequence decides for all of its rows, as in the join.
  const bool whole = s.length <= part_keys;
  const float inverse = inverse_sum(sum);
  const size_t item = (size_t)part * a.batch.tokens * a.heads + at / D;
  // Registers 4 j .. + 3 of product i are dimensions 32 i + 8 j + 4 h .. + 3.
  if (whole) {
    float factor[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      gate_factors<T>(a, at + 8 * i + 4 * h, factor[i]);
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const float x[4] = {o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1],
                          o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]};
      store_outputs<T>(a, at + 8 * i + 4 * h, x, inverse, factor[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const float4_t x = {o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1],
                          o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]};
      *reinterpret_cast<float4_t*>(split.tile_o + item * D + 8 * i + 4 * h) = x;
    }
  }
  if (!whole && h == 0) {
    split.tile_ml[2 * item] = top;
    split.tile_ml[2 * item + 1] = sum;
  }
}

// A workgroup (4 waves, 32 kSub keys a tile) takes every gridDim.x-th of the sequences'
// (tile, part) pairs, which stand one after another, so that no place without work stands
// between two with; the parts of a tile side by side, so that an XCD, which gets every
// eighth workgroup, reads few parts of a sequence's keys.
template <int D, class T, int kSub, int kWavesPerSimd>
__global__ __launch_bounds__(kThreads, kWavesPerSimd) void attention_paged_tile_kernel(
  PagedAttentionArgs a, PagedSplit split) {
  const uint32_t kv_heads = a.cache.kv_heads, group = a.heads / kv_heads;
  uint32_t part_keys = split.tile_keys;
  if (split.tile_step != 0u) {
    part_keys = chosen_keys(a, split, group);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      *split.tile_chosen = part_keys;
    }
  }
  for (uint32_t block = blockIdx.x;; block += gridDim.x) {
    const PagedItem found =
      paged_item(a.batch, block / kv_heads, a.cache.page_shift, [&](const PagedSequence& q) {
        const uint32_t r = q.count * group;
        return r > split.decode_most
                 ? (r + kTileRows - 1u) / kTileRows * ((q.length + part_keys - 1u) / part_keys)
                 : 0u;
      });
    if (found.sequence.count == 0) {
      return;
    }
    attention_paged_tile<D, T, kSub>(a, split, found, block % kv_heads, part_keys,
                                     block != blockIdx.x);
  }
}

template <int D, class T>
void launch_tiles(const PagedAttentionArgs& a, const PagedSplit& split, hipStream_t stream) {
  // One wave a SIMD for head_dim 256, whose operands take its 512 registers.  64 keys a
  // tile; 32 where two f32 parts of 256 dimensions, or two waves of 128, leave no
  // registers for more (a spilled one waits for every load under way: 17 sequences,
  // head_dim 128: 119 us with 64 keys, 104 with 32).
  constexpr int kWavesPerSimd = D == 256 ? 1 : 2;
  constexpr int kSub = D == 64 || (D == 256 && !std::is_same<T, float>::value) ? 2 : 1;
  // Two rounds of workgroups, which go on to further parts: of one for each part that a
  // batch could have most find none (17 sequences, 4096 workgroups for 512 parts: 77 us,
  // with 1024 61).  The loop costs 1 % where there is one part for each.
  const uint32_t blocks = std::min(split.tile_blocks, 2u * split.tile_slots);
  attention_paged_tile_kernel<D, T, kSub, kWavesPerSimd>
    <<<dim3(blocks), kThreads, 0, stream>>>(a, split);
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
