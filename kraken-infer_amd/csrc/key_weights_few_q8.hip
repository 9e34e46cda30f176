// The attention weight that cached keys receive: the sequences of few rows (the single
// tokens of a decode step).  Their keys pass through the matrix cores once, and the scores,
// 4 bytes for each row and key beside the key's own head_dim, are kept until the rows' sums
// are known.
//
// The first launch is the score half of the attention's decode kernel
// (attention_paged_q8.hip): a workgroup takes one KV head of one sequence and a run of its
// keys, its four waves 32-key steps in turn, S^T = K Q^T (16x16x32), the f32 query's two
// f16 parts in one product's columns up to 8 rows.  It leaves the scores in log2 units and
// each row's maximum and sum.  The second joins those and adds
// 2^(score - log2 of the row's sum) over the rows of each key.
//
// 64 sequences of up to 32768 keys, one token of four query heads for each of two KV heads of
// 256: 135 us for 537 MB of keys, 17 of weights read and written and 34 of scores each way, of
// which the second launch takes 15.  One sequence of 4096: 11.5, two launches of some 7 and 4 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "context_internal.hpp"
#include "device_common.hpp"
#include "key_weights_internal.hpp"

namespace kraken {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = 4;
constexpr uint32_t kSumKeys = 1024;  // of a workgroup of the second launch
constexpr size_t kMostBytes = size_t{1} << 30;

struct FewPlan {
  uint32_t group;      // query heads of a KV head
  uint32_t rows;       // most of a sequence
  uint32_t part_keys;  // of a workgroup of the first launch
  uint32_t parts;      // most of a sequence
  uint32_t steps;      // of 32 keys, most of a sequence
  float* scores;       // [sequences][kv_heads][steps][rows][32]
  float2* stats;       // [sequences][kv_heads][parts][rows]
};

__device__ __forceinline__ bool takes_few(uint32_t rows) { return rows != 0 && rows <= kFewRows; }

// (Whole numbers, the query as 31 bits in four columns of 8-bit products, spare the codes'
// way to f16, and took as long.  Without its stores the call of 64 sequences would take some
// 27 us less, whether they go out step by step or, by way of LDS, at a part's end.)
template <int D, class T, bool kStacked>
__global__ __launch_bounds__(kThreads, D == 256 && !kStacked ? 2 : 3) void few_scores_kernel(
  KeyWeightsArgs a, FewPlan p) {
  constexpr uint32_t kRows = kStacked ? 8 : 16;
  constexpr bool kTwo = !kStacked && std::is_same<T, float>::value;
  constexpr int kLoads = D / 64;        // of 16 keys: 1024 bytes each
  constexpr uint32_t kChunks = D / 16;  // of 16 bytes in a key row
  __shared__ float2 joined[kWaves][kRows];
  __shared__ __attribute__((aligned(16))) int8_t lds[kWaves][32 * D];

  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t n = lane & 15u, g = lane >> 4;
  const uint32_t shift = a.rows.cache.page_shift, kv_heads = a.rows.cache.kv_heads;
  const uint32_t kv_head = blockIdx.x % kv_heads;
  const PagedItem found =
    paged_item(a.rows.batch, blockIdx.x / kv_heads, shift, [&](const PagedSequence& q) {
      return takes_few(counted_rows(a, q, p.group))
               ? (q.length + p.part_keys - 1u) / p.part_keys
               : 0u;
    });
  const PagedSequence s = found.sequence;
  if (s.count == 0) {
    return;
  }
  const uint32_t rows = counted_rows(a, s, p.group), part = found.item;
  const uint32_t begin = part * p.part_keys, end = min(s.length, begin + p.part_keys);
  const uint32_t steps = (end - begin + 31u) / 32u;
  const size_t pair = (size_t)found.index * kv_heads + kv_head;
  auto first_key = [&](uint32_t step) { return begin + step * 32u; };
  // Lane 2 i + h has the page (-1: none) and the scale of granule h, 16 keys, of the wave's
  // step i: a part has up to 32 for each wave.  (Table loads between the keys' would be
  // waited for with all keys before them.)
  int32_t pages;
  float scales;
  {
    const uint32_t key = first_key(wave + kWaves * (lane >> 1)) + 16u * (lane & 1u);
    const int32_t page = a.rows.batch.table[(size_t)found.index * a.rows.batch.width +
                                            min(key >> shift, a.rows.batch.width - 1u)];
    pages = page >= 0 && (uint32_t)page < a.rows.cache.pages ? page : -1;
    scales = finite_or_nan(a.rows.cache.key_scales[(size_t)max(pages, 0) * kv_heads + kv_head]);
  }
  // A load of the wave is 1024 bytes of keys as they lie, 64 / kChunks rows; through LDS, a
  // region for each wave, they get to the lanes whose operands they are.  Chunk c of key row
  // r is held at place c ^ turn(r) of its row, so that the sixteen rows of an operand, runs
  // of four, lie in as many places.  Two steps' keys are on their way at a time.
  auto turn = [](uint32_t r) { return ((r >> 3 & 3u) * 4u + (r & 3u)) & (kChunks - 1u); };
  u32x4_t k[2][2 * kLoads];
  // (Past the wave's last step that one's again, which is in the caches.)
  const uint32_t last = (max(steps, wave + 1u) - 1u - wave) / kWaves;
  auto load_k = [&](auto parity, uint32_t of) {  // of the wave's step `of`
    constexpr int kBuffer = decltype(parity)::value;
    const uint32_t i = min(of, last);
    const uint32_t key = first_key(wave + kWaves * i);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int32_t page = __builtin_amdgcn_readlane(pages, (int)(2u * i + half & 63u));
      const uint32_t slot = (key + 16u * half) & ((1u << shift) - 1u);
      const int8_t* at = a.rows.cache.keys +
                         ((((size_t)max(page, 0) * kv_heads + kv_head) << shift) + slot) * D;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        k[kBuffer][half * kLoads + j] =
          __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(at + 1024u * j + lane * 16u));
      }
    }
  };
  // Scores at [step][row][32] of the part.  Lanes without a row, and steps past the last, lie
  // outside the resource.  (A store under a branch leaves the compiler not knowing how many
  // are under way, and a wait for keys then is one for keys behind them, too: so there is one
  // with each step's loads from the first on.)
  const __amdgpu_buffer_rsrc_t scores = make_buffer_rsrc(
    p.scores + (pair * p.steps + begin / 32u) * p.rows * 32u, steps * p.rows * 128u);
  constexpr uint32_t kNowhere = 0xffffffe0u;
  auto store4 = [&](const float* x, uint32_t at) {
    __builtin_amdgcn_raw_buffer_store_b128(
      u32x4_t{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
              __float_as_uint(x[3])}, scores, (int)at, 0, 0);
  };
  auto store_nothing = [&]() {
    const float x[4] = {};
    store4(x, kNowhere);
    if constexpr (!kStacked) {
      store4(x, kNowhere);
    }
  };
  using Even = std::integral_constant<int, 0>;
  using Odd = std::integral_constant<int, 1>;

  // Row n of a tile's product is key 8 (n / 4) + n % 4, of the second tile 4 on, so that a
  // lane's scores are those of run g of eight keys.
  const uint32_t key_row = 8u * (n >> 2) + (n & 3u), key_turn = turn(key_row);
  // This lane's query row and the keys that it sees of the part.
  const uint32_t row = n & (kRows - 1u);
  const bool real = row < rows;
  const uint32_t token = s.count - min(s.count, a.window) + (real ? row / p.group : 0u);
  const uint32_t visible = min(s.length - s.count + token + 1u, end);
  const T* query = static_cast<const T*>(a.rows.query) +
                   ((size_t)(s.start + token) * a.rows.heads + kv_head * p.group +
                    (real ? row % p.group : 0u)) * D + 16u * g;
  // Dimensions 64 c + 16 g .. + 15 of the row.
  half8_t q_hi[2 * kLoads], q_lo[kTwo ? 2 * kLoads : 1];
  float row_factor;
  {
    float x[kLoads][16], largest = 0.0f;
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        load4(query + 64 * c + 4 * i, &x[c][4 * i]);
      }
    }
    load_k(Even{}, 0u);
    store_nothing();
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[c][i] = real ? x[c][i] : 0.0f;
        largest = fmaxf(largest, fabsf(x[c][i]));
      }
    }
    largest = xor32_max(xor16_max(largest));
    const int e = query_exponent(largest);
    // 1 / sqrt(D) in log2 units, over the row's power of two; NaN for a row with an infinity.
    row_factor = ldexpf(kLog2e / (D == 64 ? 8.0f : D == 256 ? 16.0f : 11.313708498984761f), -e);
    row_factor = largest < INFINITY ? row_factor : NAN;
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        half8_t hi, lo;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          half2_t u, w;
          split_pair(ldexpf(x[c][8 * h + i], e), ldexpf(x[c][8 * h + i + 1], e), u, w);
          hi[i] = u[0];
          hi[i + 1] = u[1];
          lo[i] = w[0];
          lo[i + 1] = w[1];
        }
        // Stacked: the high parts of rows n, then the low ones of rows n - 8.
        q_hi[2 * c + h] = kStacked && n >= 8u ? lo : hi;
        if constexpr (kTwo) {
          q_lo[2 * c + h] = lo;
        }
      }
    }
  }
  load_k(Odd{}, 1u);
  store_nothing();

  float top = kLowestMax, sum = 0.0f;
  auto take = [&](auto parity, uint32_t i) {
    constexpr int kBuffer = decltype(parity)::value;
    const uint32_t step = wave + kWaves * i;
#pragma unroll
    for (int j = 0; j < 2 * kLoads; ++j) {
      const uint32_t r = (uint32_t)j * (64u / kChunks) + lane / kChunks;
      *reinterpret_cast<u32x4_t*>(&lds[wave][r * D + (lane % kChunks ^ turn(r)) * 16u]) =
        k[kBuffer][j];
    }
    // (A wave's own LDS instructions run in order; the compiler has to keep it.)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    auto chunk = [&](int tile, int c) {
      return *reinterpret_cast<const u32x4_t*>(
        &lds[wave][(key_row + 4u * tile) * D + ((4u * c + g) ^ key_turn) * 16u]);
    };
    float4_t score[2] = {float4_t{0.0f, 0.0f, 0.0f, 0.0f}, float4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const u32x4_t codes = chunk(tile, c);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const half8_t x = codes_to_f16(codes[2 * h], codes[2 * h + 1]);
          score[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q_hi[2 * c + h], score[tile],
                                                               0, 0, 0);
          if constexpr (kTwo) {
            score[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q_lo[2 * c + h],
                                                                 score[tile], 0, 0, 0);
          }
        }
      }
    }
    load_k(parity, i + 2u);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int from = (int)(2u * i & 63u);
    const bool second = g >= 2u;  // the run's granule
    const int32_t page0 = __builtin_amdgcn_readlane(pages, from);
    const int32_t page1 = __builtin_amdgcn_readlane(pages, from + 1);
    const int scale0 = __builtin_amdgcn_readlane(__float_as_int(scales), from);
    const int scale1 = __builtin_amdgcn_readlane(__float_as_int(scales), from + 1);
    const bool inside = (second ? page1 : page0) >= 0;
    const float factor = inside ? row_factor * __int_as_float(second ? scale1 : scale0) : 0.0f;
    const float offset = inside ? 0.0f : -INFINITY;
    const uint32_t key = first_key(step) + 8u * g, at = (step * p.rows + row) * 128u + 32u * g;
    float w[8], up = top;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = score[j / 4][j % 4];
      if constexpr (kStacked) {
        w[j] += dpp<kDppRowRor8>(w[j]);
      }
      w[j] = fmaf(w[j], factor, offset);
      w[j] = key + j < visible ? w[j] : -INFINITY;
      up = fmaxf(up, w[j]);
    }
    if constexpr (kStacked) {
      // (The upper lanes have the lower ones' scores, and store the second half of them.)
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = n < 8u ? w[j] : w[4 + j];
      }
      store4(x, real ? at + (n < 8u ? 0u : 16u) : kNowhere);
    } else {
      store4(w, real ? at : kNowhere);
      store4(w + 4, real ? at + 16u : kNowhere);
    }
    sum *= fast_exp2(top - up);
    top = up;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sum += fast_exp2(w[j] - top);
    }
  };
  for (uint32_t i = 0; wave + kWaves * i < steps; i += 2u) {
    take(Even{}, i);
    take(Odd{}, i + 1u);  // past the last step: no key counts
  }
  // The four runs of a step, then the waves.
  {
    const float up = xor32_max(xor16_max(top));
    sum = xor32_sum(xor16_sum(sum * fast_exp2(top - up)));
    top = up;
  }
  if (lane < kRows) {
    joined[wave][lane] = make_float2(top, sum);
  }
  __syncthreads();
  if (threadIdx.x < rows) {
    float2 all = joined[0][threadIdx.x];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) {
      const float2 x = joined[w][threadIdx.x];
      const float up = fmaxf(all.x, x.x);
      all.y = all.y * fast_exp2(all.x - up) + x.y * fast_exp2(x.x - up);
      all.x = up;
    }
    p.stats[(pair * p.parts + part) * p.rows + threadIdx.x] = all;
  }
}

// Four keys a thread.
__global__ __launch_bounds__(kThreads) void few_sums_kernel(KeyWeightsArgs a, FewPlan p) {
  static_assert(kSumKeys == 4u * kThreads, "");
  constexpr uint32_t kAhead = 4;  // rows whose scores are asked for before their logs are known
  __shared__ float logs[kFewRows];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t kv_heads = a.rows.cache.kv_heads, kv_head = blockIdx.x % kv_heads;
  const PagedItem found = paged_item(
    a.rows.batch, blockIdx.x / kv_heads, a.rows.cache.page_shift, [&](const PagedSequence& q) {
      return takes_few(counted_rows(a, q, p.group)) ? (q.length + kSumKeys - 1u) / kSumKeys : 0u;
    });
  const PagedSequence s = found.sequence;
  if (s.count == 0) {
    return;
  }
  const uint32_t rows = counted_rows(a, s, p.group);
  const size_t pair = (size_t)found.index * kv_heads + kv_head;
  const uint32_t parts = (s.length + p.part_keys - 1u) / p.part_keys;
  const uint32_t key = found.item * kSumKeys + 4u * threadIdx.x;
  // (Within the steps that were written: those of keys up to the length.)
  const uint32_t step = min(key / 32u, (s.length - 1u) / 32u);
  const float* scores = p.scores + (pair * p.steps + step) * p.rows * 32u + key % 32u;
  auto score = [&](uint32_t row) {
    return *reinterpret_cast<const float4_t*>(scores + min(row, rows - 1u) * 32u);
  };
  float4_t ahead[kAhead];
#pragma unroll
  for (uint32_t i = 0; i < kAhead; ++i) {
    ahead[i] = score(i);
  }
  float* at = a.weights + pair * a.row_stride + key;
  const uint32_t before = s.length - s.count;
  float earlier[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    earlier[i] = decayed_weight(a, at + i, key + i < before);
  }
  // log2 of each row's sum; infinity, which makes its weights zero, without any key.
  for (uint32_t row = wave; row < rows; row += kWaves) {
    float top = kLowestMax, sum = 0.0f;
    for (uint32_t i = lane; i < parts; i += 64u) {
      const float2 x = p.stats[(pair * p.parts + i) * p.rows + row];
      const float up = fmaxf(top, x.x);
      sum = sum * fast_exp2(top - up) + x.y * fast_exp2(x.x - up);
      top = up;
    }
    const float up = halves_max(across8_max(reduce8_max(top)));
    sum = wave_sum(sum * fast_exp2(top - up));
    if (lane == 0) {
      logs[row] = sum == 0.0f ? INFINITY : up + log2f(sum);
    }
  }
  __syncthreads();
  float sums[4] = {};
  auto add = [&](const float4_t& x, uint32_t row) {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      sums[i] += fast_exp2(x[i] - logs[row]);
    }
  };
#pragma unroll
  for (uint32_t i = 0; i < kAhead; ++i) {
    if (i < rows) {
      add(ahead[i], i);
    }
  }
  for (uint32_t row = kAhead; row < rows; ++row) {
    add(score(row), row);
  }
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    if (key + i < s.length) {
      at[i] = sums[i] + earlier[i];
    }
  }
}

FewPlan plan_of(const KeyWeightsArgs& a, int cu_count, size_t& bytes, void* workspace) {
  FewPlan p{};
  p.group = a.rows.heads / a.rows.cache.kv_heads;
  const uint64_t rows = (uint64_t)std::min(a.window, a.rows.batch.max_query) * p.group;
  p.rows = (uint32_t)std::min<uint64_t>(rows, kFewRows);
  const uint64_t pairs = (uint64_t)a.rows.batch.sequences * a.rows.cache.kv_heads;
  const uint32_t keys = longest_length(a);
  p.steps = (keys + 31u) / 32u;
  // Parts for eleven workgroups a CU (64 sequences of up to 32768 keys, two KV heads: 135 us,
  // with six 140), but of 768 keys where those make six (up to 8192 keys: 40.4 us, 51.6 with
  // 384), since a wave's way to its first keys is long; 512 at least where those give each CU
  // one (one sequence of 65536: 16.4 us, 19.3 with 256, 26.8 with 128), else 256 (four of 8192:
  // 15.0, 18.8 with 128, 16.7 with 512).
  const uint64_t all = pairs * keys, cus = (uint64_t)cu_count;
  uint64_t per = std::max(all / (11u * cus), std::min<uint64_t>(all / (6u * cus), 768u));
  per = std::max<uint64_t>(per, all >= 512u * cus ? 512u : 256u);
  per = std::min<uint64_t>((per + 127u) / 128u * 128u, 4096u);
  p.part_keys = (uint32_t)per;
  p.parts = (keys + p.part_keys - 1u) / p.part_keys;
  const double scores = (double)pairs * p.steps * p.rows * 128.0;
  const double stats = (double)pairs * p.parts * p.rows * sizeof(float2);
  // Where some sequences have more rows, these launches come on top of theirs, which a single
  // sequence and few keys are not worth: calls with both, and with all rows as many, of 24
  // sequences (two KV heads of 256) of up to 1000 keys 44.5 and 32.3 us, 4000 (52 MB of keys)
  // 60.1 and 46.9, 16000 (201 MB) 112 and 102; eight KV heads of 128: 37.2 and 25.7, 62.1 and
  // 61.8 (103 MB), 143 and 171; four sequences of 16000 (66 MB) 43.3 and 46.7.
  const double keys_bytes = (double)pairs * keys * a.rows.cache.head_dim;
  const bool beside = rows > kFewRows && (a.rows.batch.sequences == 1u || keys_bytes < 64e6);
  if (p.group > kFewRows || scores + stats > (double)kMostBytes || beside) {
    bytes = 0;
    return p;
  }
  p.scores = static_cast<float*>(workspace);
  p.stats = reinterpret_cast<float2*>(p.scores + pairs * p.steps * p.rows * 32u);
  bytes = (size_t)(scores + stats);
  return p;
}

template <int D, class T>
void launch_for(const KeyWeightsArgs& a, const FewPlan& p, hipStream_t stream) {
  const uint32_t pairs = a.rows.batch.sequences * a.rows.cache.kv_heads;
  const dim3 grid(pairs * p.parts);
  if (p.rows <= 8u) {
    few_scores_kernel<D, T, true><<<grid, kThreads, 0, stream>>>(a, p);
  } else {
    few_scores_kernel<D, T, false><<<grid, kThreads, 0, stream>>>(a, p);
  }
  const uint32_t blocks = (p.steps * 32u + kSumKeys - 1u) / kSumKeys;
  few_sums_kernel<<<dim3(pairs * blocks), kThreads, 0, stream>>>(a, p);
}

template <class T>
void launch_type(const KeyWeightsArgs& a, const FewPlan& p, hipStream_t stream) {
  if (a.rows.cache.head_dim == 256u) {
    launch_for<256, T>(a, p, stream);
  } else if (a.rows.cache.head_dim == 128u) {
    launch_for<128, T>(a, p, stream);
  } else {
    launch_for<64, T>(a, p, stream);
  }
}

}  // namespace

size_t few_weights_bytes(const KeyWeightsArgs& a, int cu_count) {
  size_t bytes;
  plan_of(a, cu_count, bytes, nullptr);
  return bytes;
}

void launch_few_weights(const KeyWeightsArgs& a, int cu_count, void* workspace,
                        hipStream_t stream) {
  size_t bytes;
  const FewPlan p = plan_of(a, cu_count, bytes, workspace);
  if (a.rows.f16) {
    launch_type<half_t>(a, p, stream);
  } else {
    launch_type<float>(a, p, stream);
  }
}

}  // namespace kraken
