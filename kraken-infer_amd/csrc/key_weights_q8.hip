// The attention weight that cached keys receive from a batch's rows: for key j of a
// sequence and KV head the sum over rows of 2^(s - L), s the score in log2 units and L
// the log2 of the row's sum of 2^s.
//
// Two passes over the scores, the first for L, the second for the sums; in both the keys
// stay and the rows go by.  A wave holds 64 keys as operands of the matrix cores, made
// from their codes once (attention_paged_q8_common.hpp: codes exact in f16, f32 queries
// in two f16 parts), and takes the rows 32 at a time, S = K Q^T (32x32x16), so that a row
// is a lane and a key a register: the first pass's maxima and sums and the second's sums
// are taken in registers, those over rows across lanes only once, at the end.  The rows
// come from LDS, which a workgroup's four waves (256 keys) share; a launch before lays
// them out there-ready, by tiles of 32 consecutive rows of the batch (token x head of the
// KV head), whichever sequences have them.
//
// Launches: rows, first pass (maxima and sums by 256 keys), L of each row, second pass,
// and where it splits the rows over workgroups their sums' sum.
//
// 1024 f32 rows of a sequence of 8192 (two KV heads of 256, groups of four): 140 us (150 on a
// card of lower clocks), traced 65 for each pass (68 to 71), 19 the others.  A pass's products
// are 64 GFLOP in f16, 49 us at a large product's rate, and their time hides the exponentials
// and sums (two waves a SIMD; without those the pass takes as long).  With f16 queries 90 (94).
// 32 rows at the end of the same sequence: 27, five launches.  No vector register is spilled;
// 58 to 87 scalars of a pass are, into lanes of one (256 registers in all for f32 rows of 256).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attention_paged_q8_common.hpp"
#include "context_internal.hpp"
#include "device_common.hpp"
#include "key_weights_internal.hpp"

namespace kraken {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / 64u;
constexpr uint32_t kTile = 32;                       // rows of a product
constexpr uint32_t kWaveKeys = 64;
constexpr uint32_t kBlockKeys = kWaves * kWaveKeys;  // of a workgroup
constexpr int kRing = 2;  // fragments of rows on their way from LDS

// A call's rows [0, tokens * group) of each KV head in groups of tokens, and the
// workspace of one.
struct WeightPlan {
  uint32_t first_token, end_token;  // of this group of rows
  uint32_t group;                   // query heads of a KV head
  uint32_t rows, tiles;             // of the group of rows, by KV head
  uint32_t chunk_tiles;             // of a workgroup
  uint32_t chunks;                  // most of a sequence
  uint32_t blocks;                  // most 256-key blocks of a sequence
  uint32_t keys;                    // longest sequence
  uint32_t least_rows;              // sequences of fewer are another launch's
  half_t* queries;    // [kv_heads][tiles][parts][head_dim / 16][64][8]
  float* factors;     // [kv_heads][tiles * 32]: of a product to log2 units
  uint32_t* visible;  // [tiles * 32]: keys that the row sees; 0: counts nowhere
  float2* stats;      // [kv_heads][blocks][tiles * 32]: maximum and sum
  float* logs;        // [kv_heads][tiles * 32]
  float* sums;        // [chunks][sequences][kv_heads][keys]
};

// A sequence's rows (by KV head, counted from the group's first token's) that count:
// [begin, end), empty where it is left out or has none here; and whether no earlier group
// has any.
struct RowRange {
  uint32_t begin, end;
  bool first;
};

__device__ __forceinline__ RowRange row_range(const KeyWeightsArgs& a, const WeightPlan& p,
                                              const PagedSequence& s) {
  const uint32_t rows = counted_rows(a, s, p.group);
  if (rows == 0 || rows < p.least_rows) {
    return {0u, 0u, false};
  }
  const uint32_t begin = s.start + s.count - min(s.count, a.window);
  const uint32_t from = max(begin, p.first_token), to = min(s.start + s.count, p.end_token);
  return from < to ? RowRange{(from - p.first_token) * p.group, (to - p.first_token) * p.group,
                              begin >= p.first_token}
                   : RowRange{0u, 0u, false};
}

// Tiles of 32 rows that hold a range's.
__device__ __forceinline__ uint32_t first_tile(const RowRange& r) { return r.begin / kTile; }
__device__ __forceinline__ uint32_t end_tile(const RowRange& r) {
  return (r.end + kTile - 1u) / kTile;
}

// Workgroups of a sequence and KV head: its blocks of keys times its rows' chunks.
__device__ __forceinline__ uint32_t work_of(const KeyWeightsArgs& a, const WeightPlan& p,
                                            const PagedSequence& s) {
  const RowRange r = row_range(a, p, s);
  return r.begin == r.end ? 0u
                          : (s.length + kBlockKeys - 1u) / kBlockKeys *
                              ((end_tile(r) - first_tile(r) + p.chunk_tiles - 1u) / p.chunk_tiles);
}

// What a key has when a group's sums are added: behind an earlier group the weight so far,
// else its earlier weight, if it had one, decayed.
__device__ __forceinline__ float earlier_weight(const KeyWeightsArgs& a, const RowRange& r,
                                                const float* at, bool had) {
  return r.first ? decayed_weight(a, at, had) : *at;
}

// One workgroup a tile of 32 rows of a KV head: eight threads a row.
template <int D, class T>
__global__ __launch_bounds__(kThreads) void weight_rows_kernel(KeyWeightsArgs a, WeightPlan p) {
  constexpr bool kTwo = std::is_same<T, float>::value;
  constexpr int kParts = kTwo ? 2 : 1, kSteps = D / 16, kPer = D / 8;
  __shared__ float largest[8][kTile];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, n = tid % kTile, j = tid / kTile;
  const uint32_t tile = blockIdx.x / a.rows.cache.kv_heads;
  const uint32_t kv_head = blockIdx.x % a.rows.cache.kv_heads;
  const uint32_t row = tile * kTile + n, token = p.first_token + row / p.group;
  const uint32_t from = p.first_token + tile * kTile / p.group;
  const uint32_t to = p.first_token + (tile * kTile + kTile - 1u) / p.group;
  // The sequences with rows in this tile, looked for 64 at a time.
  uint32_t visible = 0;
  for (uint32_t at = 0; at < a.rows.batch.sequences; at += 64) {
    PagedSequence s{0u, 0u, 0u};
    if (at + lane < a.rows.batch.sequences) {
      s = paged_sequence(a.rows.batch, at + lane, a.rows.cache.page_shift);
      const uint32_t rows = counted_rows(a, s, p.group);
      if (rows == 0 || rows < p.least_rows) {
        s.count = 0;
      }
    }
    uint64_t has = __ballot(s.count != 0 && s.start <= to && s.start + s.count > from);
    for (; has != 0; has &= has - 1u) {
      const int i = __builtin_ctzll(has);
      const uint32_t start = (uint32_t)__builtin_amdgcn_readlane((int)s.start, i);
      const uint32_t count = (uint32_t)__builtin_amdgcn_readlane((int)s.count, i);
      const uint32_t length = (uint32_t)__builtin_amdgcn_readlane((int)s.length, i);
      const uint32_t skip = count - min(count, a.window);
      if (token - start < count && token - start >= skip) {
        visible = length - count + (token - start) + 1u;
      }
    }
  }
  visible = row < p.rows ? visible : 0u;
  float x[kPer], most = 0.0f;
  if (visible != 0) {
    const T* q = static_cast<const T*>(a.rows.query) +
                 ((size_t)token * a.rows.heads + kv_head * p.group + row % p.group) * D + j * kPer;
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      load4(q + i, x + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      x[i] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    most = fmaxf(most, fabsf(x[i]));
  }
  largest[j][n] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    most = fmaxf(most, largest[i][n]);
  }
  const int e = query_exponent(most);
  const size_t place = ((size_t)kv_head * p.tiles + tile) * kTile + n;
  if (j == 0) {
    // (NaN for a row with an infinity.)
    const float factor =
      ldexpf(kLog2e / (D == 64 ? 8.0f : D == 256 ? 16.0f : 11.313708498984761f), -e);
    p.factors[place] = most < INFINITY ? factor : NAN;
    if (kv_head == 0) {
      p.visible[tile * kTile + n] = visible;
    }
  }
  half_t* to_tile = p.queries + ((size_t)kv_head * p.tiles + tile) * kParts * kSteps * 512u;
#pragma unroll
  for (int i = 0; i < kPer; i += 8) {
    half8_t hi, lo;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      half2_t u, w;
      split_pair(ldexpf(x[i + k], e), ldexpf(x[i + k + 1], e), u, w);
      hi[k] = u[0];
      hi[k + 1] = u[1];
      lo[k] = w[0];
      lo[k + 1] = w[1];
    }
    // Dimensions 32 q + 16 h + 8 s .. + 7 are what lanes 32 h .. hold in step 2 q + s.
    const uint32_t d = j * kPer + i;
    const uint32_t step = d / 32u * 2u + d / 8u % 2u, h = d / 16u % 2u;
    half_t* at = to_tile + (step * 64u + h * 32u + n) * 8u;
    *reinterpret_cast<half8_t*>(at) = hi;
    if constexpr (kTwo) {
      *reinterpret_cast<half8_t*>(at + kSteps * 512) = lo;
    }
  }
}

// A pass over a block of 256 keys and a chunk of row tiles.
template <int D, class T, bool kSums>
__global__ __launch_bounds__(kThreads, 2) void weight_pass_kernel(KeyWeightsArgs a, WeightPlan p) {
  constexpr bool kTwo = std::is_same<T, float>::value;
  constexpr int kParts = kTwo ? 2 : 1, kSteps = D / 16, kSubs = kWaveKeys / 32;
  constexpr uint32_t kTileHalves = kParts * kSteps * 512u;
  constexpr uint32_t kCopies = kTileHalves / 512u / kWaves;  // of 1024 bytes a wave
  __shared__ __attribute__((aligned(16))) half_t lds[2][kTileHalves];
  __shared__ float2 joined[2][kWaves][kTile];

  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t n = lane & 31u, h = lane >> 5;
  const uint32_t shift = a.rows.cache.page_shift, kv_heads = a.rows.cache.kv_heads;
  const uint32_t kv_head = blockIdx.x % kv_heads;
  const uint32_t padded = p.tiles * kTile;
  for (uint32_t block = blockIdx.x;; block += gridDim.x) {
    const PagedItem found =
      paged_item(a.rows.batch, block / kv_heads, shift,
                 [&](const PagedSequence& q) { return work_of(a, p, q); });
    const PagedSequence s = found.sequence;
    if (s.count == 0) {
      return;
    }
    const RowRange range = row_range(a, p, s);
    const uint32_t blocks = (s.length + kBlockKeys - 1u) / kBlockKeys;
    const uint32_t key_block = found.item % blocks, chunk = found.item / blocks;
    const uint32_t begin_tile = first_tile(range) + chunk * p.chunk_tiles;
    const uint32_t stop_tile = min(begin_tile + p.chunk_tiles, end_tile(range));
    const uint32_t first_key = key_block * kBlockKeys + wave * kWaveKeys;
    const int32_t* table = a.rows.batch.table + (size_t)found.index * a.rows.batch.width;
    auto page_of = [&](uint32_t key) {
      return table[min(key >> shift, a.rows.batch.width - 1u)];
    };
    auto inside = [&](int32_t page) { return page >= 0 && (uint32_t)page < a.rows.cache.pages; };

    // A tile goes from memory to LDS by itself (registers on its way are what two waves a
    // SIMD do not have); the wave waits for its copies, the workgroup for all.
    auto copy = [&](uint32_t tile, uint32_t parity) {
      const i32x4_t from =
        rsrc_words(p.queries + ((size_t)kv_head * p.tiles + tile) * kTileHalves, kTileHalves * 2u);
#pragma unroll
      for (uint32_t i = 0; i < kCopies; ++i) {
        const uint32_t at = (wave * kCopies + i) * 512u;
        copy16_to_lds(from, at * 2u + lane * 16u, lds[parity] + at);
      }
    };
    auto arrived = [&]() {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    };
    __syncthreads();  // the item before has read its tiles
    copy(begin_tile, 0);

    // Row r of a product is key swap(r), bits 2 and 3 in each other's place, so that a
    // lane's registers are runs of eight keys: 8 b + i of half h is key 16 b + 8 h + i.
    const uint32_t key_row = (n & 19u) | (n & 4u) << 1 | (n & 8u) >> 1;
    half8_t k[kSubs][kSteps];
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) {
      const uint32_t key = first_key + 32u * sub + key_row;
      const int32_t page = page_of(key);
      const int8_t* at = a.rows.cache.keys +
                         ((((size_t)(inside(page) ? page : 0) * kv_heads + kv_head) << shift) +
                          (key & ((1u << shift) - 1u))) * D + 16u * h;
#pragma unroll
      for (int c = 0; c < kSteps / 2; ++c) {
        const u32x4_t x = *reinterpret_cast<const u32x4_t*>(at + 32 * c);
        k[sub][2 * c] = codes_to_f16(x[0], x[1]);
        k[sub][2 * c + 1] = codes_to_f16(x[2], x[3]);
      }
    }
    // Scales of the four runs of 16 keys, each of one page.
    float scale[2 * kSubs], offset[2 * kSubs];
    {
      const int32_t page = page_of(first_key + 16u * (lane & 3u));
      const float held =
        inside(page) ? finite_or_nan(a.rows.cache.key_scales[(size_t)page * kv_heads + kv_head])
                     : 0.0f;
      const float out = inside(page) ? 0.0f : -INFINITY;
#pragma unroll
      for (int b = 0; b < 2 * kSubs; ++b) {
        scale[b] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(held), b));
        offset[b] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(out), b));
      }
    }
    float16_t sums[kSubs];
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) {
      sums[sub] = float16_t{};
    }
    // The lane's row's values, a tile ahead.
    struct Values {
      uint32_t visible;
      float factor, log;
    };
    auto values_of = [&](uint32_t tile) {
      const uint32_t row = tile * kTile + n;
      return Values{p.visible[row], p.factors[(size_t)kv_head * padded + row],
                    kSums ? p.logs[(size_t)kv_head * padded + row] : 0.0f};
    };
    Values values = values_of(begin_tile);
    // The compiler, which does not count the copies, is told that the values have come with
    // them: a wait for a value behind the next copies would be one for these, too.
    auto settled = [&]() {
      arrived();
      asm volatile("" : "+v"(values.visible), "+v"(values.factor), "+v"(values.log));
    };
    settled();
    for (uint32_t tile = begin_tile; tile < stop_tile; ++tile) {
      const uint32_t parity = (tile - begin_tile) & 1u;
      const uint32_t following = min(tile + 1u, stop_tile - 1u);
      const uint32_t row = tile * kTile + n;
      const bool own = row >= range.begin && row < range.end;
      const uint32_t seen = own ? values.visible : 0u;
      const float factor = values.factor, log = values.log;
      values = values_of(following);
      if (tile + 1u < stop_tile) {
        copy(tile + 1u, parity ^ 1u);
      }
      float top = kLowestMax, sum = 0.0f;
      if constexpr (kSums) {
        // A row whose sum is NaN spoils all keys, those too that it does not see: its NaN stays
        // in the sums of the wave's first key, for the end.
        sums[0][0] = own && log != log ? log : sums[0][0];
      }
      const bool any = __any(seen > first_key);  // else no row sees the wave's keys
      float16_t score[kSubs];
      // Fragments of the rows kRing ahead of the products that take them.
      const half8_t* q = reinterpret_cast<const half8_t*>(lds[parity]) + lane;
      half8_t ring[kRing];
      if (any) {
#pragma unroll
        for (int i = 0; i < kRing; ++i) {
          ring[i] = q[i * 64];
        }
#pragma unroll
        for (int i = 0; i < kParts * kSteps; ++i) {
#pragma unroll
          for (int sub = 0; sub < kSubs; ++sub) {
            score[sub] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              k[sub][i % kSteps], ring[i % kRing], i == 0 ? float16_t{} : score[sub], 0, 0, 0);
          }
          if (i + kRing < kParts * kSteps) {
            ring[i % kRing] = q[(i + kRing) * 64];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        float scaled[2 * kSubs];
#pragma unroll
        for (int b = 0; b < 2 * kSubs; ++b) {
          scaled[b] = factor * scale[b];
        }
        // Keys that a row does not see add nothing, whatever their scores are: those from `left`
        // on, counted from the lane's first (against which all 32 compare with constants).
        const int left = (int)(seen - (first_key + 8u * h));
        auto soften = [&](auto masks) {
          constexpr bool kMasked = decltype(masks)::value;
          auto exponent = [&](int sub, int r, float base) {
            const int b = 2 * sub + r / 8;
            const float y = fmaf(score[sub][r], scaled[b], base);
            return !kMasked || 16 * b + r % 8 < left ? y : -INFINITY;
          };
          if constexpr (!kSums) {
            // (A scale is not negative: the largest score of a run of keys is that of its
            // largest product.)
#pragma unroll
            for (int b = 0; b < 2 * kSubs; ++b) {
              float largest = -INFINITY;
#pragma unroll
              for (int r = 8 * (b % 2); r < 8 * (b % 2) + 8; ++r) {
                const bool sees = !kMasked || 16 * b + r % 8 < left;
                largest = fmaxf(largest, sees ? score[b / 2][r] : -INFINITY);
              }
              const float y = fmaf(largest, scaled[b], offset[b]);
              top = largest > -INFINITY ? fmaxf(top, y) : top;
            }
            top = xor32_max(top);
          }
#pragma unroll
          for (int sub = 0; sub < kSubs; ++sub) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float base = offset[2 * sub + r / 8] - (kSums ? log : top);
              const float w = fast_exp2(exponent(sub, r, base));
              if constexpr (kSums) {
                sums[sub][r] += w;
              } else {
                sum += w;
              }
            }
          }
          if constexpr (!kSums) {
            sum = xor32_sum(sum);
          }
        };
        if (__any(seen < first_key + kWaveKeys)) {
          soften(std::true_type{});
        } else {
          soften(std::false_type{});
        }
      }
      if constexpr (!kSums) {
        if (h == 0) {
          joined[parity][wave][n] = make_float2(top, sum);
        }
      }
      settled();
      if constexpr (!kSums) {
        // (The other parity's are written meanwhile, these again behind another barrier.)
        if (wave == 0 && h == 0 && own) {
          float2 all = joined[parity][0][n];
#pragma unroll
          for (uint32_t w = 1; w < kWaves; ++w) {
            const float2 x = joined[parity][w][n];
            const float up = fmaxf(all.x, x.x);
            all.y = all.y * fast_exp2(all.x - up) + x.y * fast_exp2(x.x - up);
            all.x = up;
          }
          p.stats[((size_t)kv_head * p.blocks + key_block) * padded + row] = all;
        }
      }
    }
    if constexpr (kSums) {
      // Over the rows, which are the lanes of each half; lane n keeps register n.
      static_assert(16 * kSubs == 32, "a register for each lane of a half");
      const float first = reduce32_sum(sums[0][0]);
      float mine = first;
#pragma unroll
      for (int i = 1; i < 16 * kSubs; ++i) {
        const float all = reduce32_sum(sums[i / 16][i % 16]);
        mine = n == (uint32_t)i ? all : mine;
      }
      mine = first != first ? first : mine;
      const size_t pair = (size_t)found.index * kv_heads + kv_head;
      const uint32_t key = first_key + 16u * (n / 8u) + 8u * h + n % 8u;
      if (key < s.length) {
        if (p.chunks > 1u) {
          p.sums[((size_t)chunk * a.rows.batch.sequences * kv_heads + pair) * p.keys + key] = mine;
        } else {
          float* at = a.weights + pair * a.row_stride + key;
          *at = mine + earlier_weight(a, range, at, key < s.length - s.count);
        }
      }
    }
  }
}

// log2 of each row's sum over its keys: the join of its blocks' maxima and sums.  Rows
// without any key get infinity, which makes their weights zero.
__global__ __launch_bounds__(kThreads) void weight_logs_kernel(WeightPlan p,
                                                               uint32_t kv_heads) {
  const uint32_t row = blockIdx.x / kv_heads * kThreads + threadIdx.x;
  const uint32_t kv_head = blockIdx.x % kv_heads;
  const uint32_t padded = p.tiles * kTile;
  if (row >= padded) {
    return;
  }
  const uint32_t blocks = (p.visible[row] + kBlockKeys - 1u) / kBlockKeys;
  const float2* at = p.stats + (size_t)kv_head * p.blocks * padded + row;
  float top = kLowestMax, sum = 0.0f;
  for (uint32_t i = 0; i < blocks; i += 8) {
    float2 x[8];
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      x[j] = i + j < blocks ? at[(size_t)(i + j) * padded] : make_float2(kLowestMax, 0.0f);
    }
    float up = top;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      up = fmaxf(up, x[j].x);
    }
    sum *= fast_exp2(top - up);
    top = up;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      sum += x[j].y * fast_exp2(x[j].x - top);
    }
  }
  p.logs[(size_t)kv_head * padded + row] = sum == 0.0f ? INFINITY : top + log2f(sum);
}

// The sum over the rows' chunks, and what the key had.
__global__ __launch_bounds__(kThreads) void weight_sum_kernel(KeyWeightsArgs a, WeightPlan p) {
  const uint32_t kv_heads = a.rows.cache.kv_heads;
  const uint32_t sequence = blockIdx.x / kv_heads;
  const PagedSequence s = paged_sequence(a.rows.batch, sequence, a.rows.cache.page_shift);
  const RowRange r = row_range(a, p, s);
  if (r.begin == r.end) {
    return;
  }
  const uint32_t chunks = (end_tile(r) - first_tile(r) + p.chunk_tiles - 1u) / p.chunk_tiles;
  const size_t plane = (size_t)a.rows.batch.sequences * kv_heads * p.keys;
  const uint32_t before = s.length - s.count;
  for (uint32_t key = blockIdx.y * kThreads + threadIdx.x; key < s.length;
       key += gridDim.y * kThreads) {
    float* at = a.weights + (size_t)blockIdx.x * a.row_stride + key;
    float sum = 0.0f;
    for (uint32_t c = 0; c < chunks; ++c) {
      sum += p.sums[c * plane + (size_t)blockIdx.x * p.keys + key];
    }
    *at = sum + earlier_weight(a, r, at, key < before);
  }
}

constexpr size_t kStatsBytes = size_t{256} << 20;

size_t aligned(size_t bytes) { return (bytes + 255u) & ~size_t{255}; }

// The plan of the first group of rows, and how many tokens a group has; `workspace` null:
// only sizes count.  Returns its bytes.
size_t plan_of(const KeyWeightsArgs& a, int cu_count, void* workspace, WeightPlan& p,
               uint32_t& group_tokens) {
  const PagedQ8Args& c = a.rows.cache;
  p = WeightPlan{};
  p.group = a.rows.heads / c.kv_heads;
  p.keys = longest_length(a);
  p.least_rows = few_weights_bytes(a, cu_count) != 0u ? kFewRows + 1u : 0u;
  p.blocks = (p.keys + kBlockKeys - 1u) / kBlockKeys;
  // Rows in groups whose statistics take no more than 256 MiB (or one token's).
  const uint64_t token_bytes =
    (uint64_t)a.rows.heads * (p.blocks * sizeof(float2) + c.head_dim * 4u);
  group_tokens = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(kStatsBytes / token_bytes, 1u),
                                              a.rows.batch.tokens);
  p.rows = group_tokens * p.group;
  p.tiles = (p.rows + kTile - 1u) / kTile;
  // Row chunks, so that there is work for twice the CUs.
  const uint64_t pairs = (uint64_t)a.rows.batch.sequences * c.kv_heads;
  const uint32_t most_rows = std::min({a.window, a.rows.batch.max_query, group_tokens}) * p.group;
  const uint32_t most_tiles = std::min((most_rows + kTile - 1u) / kTile + 1u, p.tiles);
  const uint64_t want = (2u * (uint64_t)cu_count + pairs * p.blocks - 1u) / (pairs * p.blocks);
  p.chunk_tiles = (uint32_t)((most_tiles + want - 1u) / want);
  p.chunks = (most_tiles + p.chunk_tiles - 1u) / p.chunk_tiles;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    void* here = workspace == nullptr ? nullptr : static_cast<char*>(workspace) + at;
    at += aligned(bytes);
    return here;
  };
  const size_t padded = (size_t)p.tiles * kTile;
  p.queries = static_cast<half_t*>(
    take(c.kv_heads * padded * c.head_dim * sizeof(half_t) * (a.rows.f16 ? 1u : 2u)));
  p.factors = static_cast<float*>(take(c.kv_heads * padded * sizeof(float)));
  p.visible = static_cast<uint32_t*>(take(padded * sizeof(uint32_t)));
  p.stats = static_cast<float2*>(take(c.kv_heads * padded * p.blocks * sizeof(float2)));
  p.logs = static_cast<float*>(take(c.kv_heads * padded * sizeof(float)));
  p.sums = static_cast<float*>(take(p.chunks > 1u ? p.chunks * pairs * p.keys * sizeof(float) : 0u));
  return at;
}

template <int D, class T>
void launch_for(const KeyWeightsArgs& a, WeightPlan p, uint32_t group_tokens, int cu_count,
                hipStream_t stream) {
  const PagedQ8Args& c = a.rows.cache;
  const uint64_t pairs = (uint64_t)a.rows.batch.sequences * c.kv_heads;
  // As many workgroups as a batch can need, but of no use beyond a few rounds.
  const uint64_t work = pairs * p.blocks * p.chunks;
  // A multiple of the KV heads, so that a workgroup stays with one.
  const uint64_t rounds = (16u * (uint64_t)cu_count + c.kv_heads - 1u) / c.kv_heads * c.kv_heads;
  const uint32_t grid = (uint32_t)std::min(work, rounds);
  for (uint64_t token = 0; token < a.rows.batch.tokens; token += group_tokens) {
    p.first_token = (uint32_t)token;
    p.end_token = (uint32_t)std::min<uint64_t>(a.rows.batch.tokens, token + group_tokens);
    p.rows = (p.end_token - p.first_token) * p.group;
    weight_rows_kernel<D, T><<<dim3(p.tiles * c.kv_heads), kThreads, 0, stream>>>(a, p);
    weight_pass_kernel<D, T, false><<<dim3(grid), kThreads, 0, stream>>>(a, p);
    weight_logs_kernel<<<dim3((p.tiles * kTile + kThreads - 1u) / kThreads * c.kv_heads), kThreads,
                         0, stream>>>(p, c.kv_heads);
    weight_pass_kernel<D, T, true><<<dim3(grid), kThreads, 0, stream>>>(a, p);
    if (p.chunks > 1u) {
      const uint32_t across = std::min((p.keys + kThreads - 1u) / kThreads, 1024u);
      weight_sum_kernel<<<dim3((uint32_t)pairs, across), kThreads, 0, stream>>>(a, p);
    }
  }
}

template <class T>
void launch_type(const KeyWeightsArgs& a, const WeightPlan& p, uint32_t group_tokens, int cu_count,
                 hipStream_t stream) {
  if (a.rows.cache.head_dim == 256u) {
    launch_for<256, T>(a, p, group_tokens, cu_count, stream);
  } else if (a.rows.cache.head_dim == 128u) {
    launch_for<128, T>(a, p, group_tokens, cu_count, stream);
  } else {
    launch_for<64, T>(a, p, group_tokens, cu_count, stream);
  }
}

}  // namespace

namespace {

// Whether a sequence may have more rows than a call keeps scores of.
bool has_many(const KeyWeightsArgs& a, size_t few_bytes) {
  const uint64_t group = a.rows.heads / a.rows.cache.kv_heads;
  return few_bytes == 0u || std::min(a.window, a.rows.batch.max_query) * group > kFewRows;
}

}  // namespace

size_t key_weights_workspace_bytes(const KeyWeightsArgs& a, int cu_count) {
  WeightPlan p;
  uint32_t group_tokens;
  const size_t few = few_weights_bytes(a, cu_count);
  return std::max(few,
                  has_many(a, few) ? plan_of(a, cu_count, nullptr, p, group_tokens) : 0u);
}

hipError_t launch_key_weights(const KeyWeightsArgs& a, int cu_count, void* workspace,
                              hipStream_t stream) {
  // (One after the other on the stream, in the same workspace.)
  const size_t few = few_weights_bytes(a, cu_count);
  if (few != 0u) {
    launch_few_weights(a, cu_count, workspace, stream);
  }
  if (!has_many(a, few)) {
    return hipGetLastError();
  }
  WeightPlan p;
  uint32_t group_tokens;
  plan_of(a, cu_count, workspace, p, group_tokens);
  if (a.rows.f16) {
    launch_type<half_t>(a, p, group_tokens, cu_count, stream);
  } else {
    launch_type<float>(a, p, group_tokens, cu_count, stream);
  }
  return hipGetLastError();
}

}  // namespace kraken
