// Causal attention of a ragged batch over 8-bit KV pages: the sequences that bring few
// rows (the single tokens of a decode step, drafted tokens to verify), and the join of
// split results.  The arithmetic is described in attention_paged_q8_common.hpp.
//
// A workgroup takes one KV head of one sequence and a run of its keys; its four waves
// take 32-key steps in turn, each with its own running maximum, sum and output, and
// join them at the end.  Nothing passes through LDS before that: K and V go from the
// pages to registers in the operand layout of the matrix cores.
//  - S^T = K Q^T (16x16x32): a lane loads 16 bytes of its key row at a time, which
//    are two operands; the order of the dimensions within a product is free, and Q is
//    laid out the same way.  The key rows of a 32-key step are dealt to the two row
//    tiles so that a lane's eight scores are those of one run of eight keys.
//  - O^T += V^T P^T: that run is what a lane's operand of P must hold, so P needs no
//    exchange between lanes, and since the pages keep the eight tokens of a run side
//    by side, the operand of V is eight bytes as they lie.
//  - The f32 operands need two f16 parts.  Up to 8 rows fill only half of the 16
//    columns, so the high parts take columns 0..7 and the low parts 8..15 of the same
//    product (kStacked) and the halves are added; a block of 16 rows takes two products.
//
// 64 sequences of up to 32768 keys, 2 KV heads of 256 (1.07 GB): 194 us, 5.5 TB/s, of the
// 6.95 that a read of as much reaches; the parts are of one size, so the last ones end
// alone.  One of 4096 keys: 8.6 us and 3.9 for the join, launch and latency (lengths, table,
// codes, exchange, one after another); its 4.2 MB would take 1.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention_paged_q8_common.hpp"
#include "context_internal.hpp"
#include "device_common.hpp"

namespace kraken {
namespace {

constexpr uint32_t kWaves = 4;
constexpr uint32_t kJoinAcross = 1u << 20;  // workgroups of the join along x

// Of sequences with pages of their own and one block of rows each code is read once, which
// the hint is for (64 of up to 32768 keys: 194 us, 204 without it).  It costs where codes are
// read again: by further blocks (64 sequences of 8 tokens: 97 us, 87 without) and of a prefix
// in shared pages (three quarters of the 64 in common: 176 us, 117 without).  The host cannot
// tell them apart: tables and row counts are the device's.
__device__ __forceinline__ u32x4_t load_once(const int8_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
}

// Workgroup `block`'s work; false where there is none.  `again`: the workgroup has done other
// before.
template <int D, class T, bool kStacked, class Work>
__device__ __forceinline__ bool attention_paged_decode(const PagedAttentionArgs& a,
                                                       const PagedSplit& split, const Work& work,
                                                       uint32_t block, bool again) {
  constexpr bool kShared = std::is_same<Work, SharedWork>::value;
  constexpr uint32_t kRows = kStacked ? 8 : kDecodeBlock;
  constexpr bool kTwo = !kStacked && std::is_same<T, float>::value;
  constexpr int kLoads = D / 64;  // 16-byte loads of a key row per lane and row tile
  constexpr int kStride = D + 4;  // of an output row in LDS, in floats
  __shared__ float lds_o[kWaves * kRows * kStride];
  __shared__ float lds_m[kWaves][kRows], lds_l[kWaves][kRows];

  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t n = lane & 15u, g = lane >> 4;
  const uint32_t shift = a.cache.page_shift, kv_heads = a.cache.kv_heads;
  const uint32_t group = a.heads / kv_heads;
  const uint32_t kv_head = block % kv_heads;
  uint32_t item = block / kv_heads, sequence = 0;
  PagedSequence s;
  // Of a shared call's item: its first key, and what it is.
  uint32_t first = 0, shared_group = kNoGroup;
  uint32_t part_keys = split.decode_keys;
  if constexpr (kShared) {
    const SharedFound found = shared_item(work, 0, item);
    if (found.item.count == 0) {
      return false;
    }
    s = {found.item.start, found.item.count, found.item.length};
    sequence = found.item.sequence;
    first = found.item.first;
    shared_group = found.item.group;
    item = found.work;
    part_keys = work.keys[0];
  } else if (a.batch.sequences > 1u) {
    // The sequences' parts one after another: no workgroup without keys stands between
    // two with, and the XCDs, which take workgroups in turn, get as many each.
    const PagedItem found = paged_item(a.batch, item, shift, [&](const PagedSequence& q) {
      const uint32_t r = q.count * group;
      return r <= split.decode_rows ? (r + kRows - 1u) / kRows *
                                        ((q.length + split.decode_keys - 1u) / split.decode_keys)
                                    : 0u;
    });
    s = found.sequence;
    sequence = found.index;
    item = found.item;
  } else {
    s.count = a.batch.max_query;
  }
  // The row blocks of a part stand side by side.  (A single sequence's are those of
  // max_query, which it may fall short of.)
  const uint32_t blocks = max(1u, (s.count * group + kRows - 1u) / kRows);
  const uint32_t part = item / blocks, first_row = item % blocks * kRows;
  const uint32_t begin = first + part * part_keys;
  // The first pages' ids are asked for together with a single sequence's length (in the
  // bounds of the table whatever that is): K and V wait for two loads in a row, not three.
  const int32_t* table = a.batch.table + (size_t)sequence * a.batch.width;
  auto page_of = [&](uint32_t key) { return table[min(key >> shift, a.batch.width - 1u)]; };
  auto first_key = [&](uint32_t step) { return begin + step * 32u; };
  // Of the lane's key rows (run n / 4 of the step's four) and of its own run g.
  int32_t page_k = page_of(first_key(wave) + 8u * (n >> 2));
  int32_t page_v = page_of(first_key(wave) + 8u * g);
  if constexpr (!kShared) {
    if (a.batch.sequences == 1u) {
      s = paged_sequence(a.batch, 0, shift);
    }
    if (s.count == 0 || s.count * group > split.decode_rows || first_row >= s.count * group ||
        begin >= s.length) {
      return false;
    }
  }
  const uint32_t rows = min(kRows, s.count * group - first_row);
  const uint32_t end = min(s.length, begin + part_keys);
  const uint32_t steps = (end - begin + 31u) / 32u;

  // This lane's query row and the keys that it sees.
  const uint32_t row = kStacked ? n & 7u : n;
  const bool real = row < rows;
  const uint32_t token = real ? (first_row + row) / group : 0u;
  // Keys before the row's own position and it; of a group's, all.
  const uint32_t before = shared_group == kIsGroup ? s.length - 1u : s.length - s.count;
  const uint32_t visible = shared_group == kIsGroup ? s.length : before + token + 1u;
  const size_t at = ((size_t)(s.start + token) * a.heads + kv_head * group +
                     (real ? (first_row + row) % group : 0u)) * D;

  u32x4_t k[2][kLoads], v[2 * kLoads];
  float key_scale, val_scale;
  bool inside;
  auto load_k = [&](uint32_t step, int32_t page) {
    const uint32_t key = first_key(step) + 8u * (n >> 2) + (n & 3u);
    const uint32_t held = page >= 0 && (uint32_t)page < a.cache.pages ? (uint32_t)page : 0u;
    const int8_t* p = a.cache.keys +
                      ((((size_t)held * kv_heads + kv_head) << shift) +
                       (key & ((1u << shift) - 1u))) * D + 16u * g;
#pragma unroll
    for (int i = 0; i < 2 * kLoads; ++i) {
      k[i / kLoads][i % kLoads] = load_once(p + i / kLoads * 4 * D + 64 * (i % kLoads));
    }
  };
  auto load_v = [&](uint32_t step, int32_t page) {
    const uint32_t key = first_key(step) + 8u * g;
    inside = page >= 0 && (uint32_t)page < a.cache.pages;
    const size_t page_head = (size_t)(inside ? (uint32_t)page : 0u) * kv_heads + kv_head;
    const int8_t* p = a.cache.values +
                      ((page_head << shift) + (key & ((1u << shift) - 1u))) * D + 16u * n;
#pragma unroll
    for (int c = 0; c < 2 * kLoads; ++c) {
      v[c] = load_once(p + 256 * c);
    }
    key_scale = a.cache.key_scales[page_head];
    val_scale = a.cache.value_scales[page_head];
  };

  // The query: D / 4 values a lane, those of its dimensions 64 c + 16 g .. + 15.
  half8_t q_hi[2 * kLoads], q_lo[kTwo ? 2 * kLoads : 1];
  float row_factor;
  {
    float x[kLoads][16], largest = 0.0f;
    const T* p = static_cast<const T*>(a.query) + at + 16u * g;
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        load4(p + 64 * c + 4 * i, &x[c][4 * i]);
      }
    }
    if (wave < steps) {
      load_k(wave, page_k);
      load_v(wave, page_v);
    }
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
    // 1 / sqrt(D) in log2 units, over the row's power of two.
    row_factor = ldexpf(kLog2e / (D == 64 ? 8.0f : D == 256 ? 16.0f : 11.313708498984761f), -e);
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
        if constexpr (kStacked) {
          q_hi[2 * c + h] = n < 8u ? hi : lo;
        } else {
          q_hi[2 * c + h] = hi;
          if constexpr (kTwo) {
            q_lo[2 * c + h] = lo;
          }
        }
      }
    }
  }

  float4_t o[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    o[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  float top = kLowestMax, sum = 0.0f;
  // Keys that every row sees need no mask.
  const uint32_t open = shared_group == kIsGroup ? s.length : before + first_row / group + 1u;

  for (uint32_t step = wave; step < steps; step += kWaves) {
    const uint32_t next = step + kWaves;
    if (next < steps) {
      page_k = page_of(first_key(next) + 8u * (n >> 2));
      page_v = page_of(first_key(next) + 8u * g);
    }
    float4_t score[2] = {float4_t{0.0f, 0.0f, 0.0f, 0.0f}, float4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
          const half8_t x = codes_to_f16(k[tile][c][2 * h], k[tile][c][2 * h + 1]);
          score[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q_hi[2 * c + h], score[tile],
                                                               0, 0, 0);
          if constexpr (kTwo) {
            score[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q_lo[2 * c + h],
                                                                 score[tile], 0, 0, 0);
          }
        }
      }
    }
    const ValueScale sv = value_scale(val_scale);
    const float factor = inside ? row_factor * key_scale : 0.0f;
    const float offset = inside ? sv.exponent : -INFINITY;
    float inverse = inside ? sv.inverse : 0.0f;
    const uint32_t key = first_key(step) + 8u * g;
    if (next < steps) {
      load_k(next, page_k);
    }
    float w[8], largest = kLowestMax;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = score[i / 4][i % 4];
      if constexpr (kStacked) {
        x += dpp<kDppRowRor8>(x);
      }
      w[i] = fmaf(x, factor, offset);
    }
    if (first_key(step) + 32u > open) {  // uniform
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = key + i < visible ? w[i] : -INFINITY;
      }
      // Of a page that the row does not see at all, the scale may be NaN.
      inverse = key < visible ? inverse : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      largest = fmaxf(largest, w[i]);
    }
    largest = xor32_max(xor16_max(largest));
    if (__any(largest > top + kMaxLead)) {
      const float up = fmaxf(top, largest);
      const float keep = fast_exp2(top - up);
      top = up;
      sum *= keep;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        o[i] *= keep;
      }
    }
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = fast_exp2(w[i] - (top - kWeightShift));
      all += w[i];
    }
    sum = fmaf(all, inverse, sum);
    half8_t p_hi, p_lo;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      half2_t u, l;
      if constexpr (!kStacked && !kTwo) {
        u = half2_t{(half_t)w[i], (half_t)w[i + 1]};
        l = u;
      } else {
        split_pair(w[i], w[i + 1], u, l);
      }
      p_hi[i] = u[0];
      p_hi[i + 1] = u[1];
      p_lo[i] = l[0];
      p_lo[i + 1] = l[1];
    }
    if constexpr (kStacked) {
      p_hi = n < 8u ? p_hi : p_lo;
    }
#pragma unroll
    for (int c = 0; c < 2 * kLoads; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const half8_t x = codes_to_f16(v[c][2 * h], v[c][2 * h + 1]);
        o[2 * c + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, p_hi, o[2 * c + h], 0, 0, 0);
        if constexpr (kTwo) {
          o[2 * c + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, p_lo, o[2 * c + h], 0, 0, 0);
        }
      }
    }
    if (next < steps) {
      load_v(next, page_v);
    }
  }

  // The waves' results to LDS, and their join.
  sum = xor32_sum(xor16_sum(sum));
  if constexpr (kStacked) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[i][j] += dpp<kDppRowRor8>(o[i][j]);
      }
    }
  }
  if (again) {
    __syncthreads();  // the results before are read
  }
  if (n < kRows) {
    if (g == 0) {
      lds_m[wave][n] = top;
      lds_l[wave][n] = sum;
    }
    float* p = lds_o + (wave * kRows + n) * kStride;
#pragma unroll
    for (int c = 0; c < 2 * kLoads; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // Row 4 g + j of product (c, h) is dimension 32 c + 2 (4 g + j) + h.
        *reinterpret_cast<float2*>(p + 32 * c + 8 * g + 2 * j) =
          make_float2(o[2 * c][j], o[2 * c + 1][j]);
      }
    }
  }
  __syncthreads();
  const bool whole = shared_group == kNoGroup && s.length <= part_keys;
  for (uint32_t e = threadIdx.x; e < rows * D; e += 256u) {
    const uint32_t r = e / D, d = e % D;
    float m = lds_m[0][r];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) {
      m = fmaxf(m, lds_m[w][r]);
    }
    float l = 0.0f, x = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      const float keep = fast_exp2(lds_m[w][r] - m);
      l = fmaf(keep, lds_l[w][r], l);
      x = fmaf(keep, lds_o[(w * kRows + r) * kStride + d], x);
    }
    const size_t out = ((size_t)(s.start + (first_row + r) / group) * a.heads +
                        kv_head * group + (first_row + r) % group);
    if (whole) {
      store_output<T>(a, out * D + d, x, inverse_sum(l));
    } else if constexpr (kShared) {
      const uint32_t kind = shared_group == kIsGroup ? 1u : 0u;
      const size_t i = (size_t)part * a.batch.tokens * a.heads + out;
      work.o[kind][i * D + d] = x;
      if (d == 0) {
        work.ml[kind][2 * i] = m;
        work.ml[kind][2 * i + 1] = l;
      }
    } else {
      const size_t i = (((size_t)part * a.batch.sequences + sequence) * kv_heads + kv_head) *
                         split.decode_rows + first_row + r;
      split.decode_o[i * D + d] = x;
      if (d == 0) {
        split.decode_ml[2 * i] = m;
        split.decode_ml[2 * i + 1] = l;
      }
    }
  }
  return true;
}

template <int D, class T, bool kStacked, class Work>
__global__ __launch_bounds__(256, 2) void attention_paged_decode_kernel(PagedAttentionArgs a,
                                                                        PagedSplit split,
                                                                        Work work) {
  if constexpr (std::is_same<Work, SharedWork>::value) {
    // Those of a shared call go on to further work: the host does not know how much there is.
    for (uint32_t block = blockIdx.x;
         attention_paged_decode<D, T, kStacked>(a, split, work, block, block != blockIdx.x);
         block += gridDim.x) {
    }
  } else {
    attention_paged_decode<D, T, kStacked>(a, split, work, blockIdx.x, false);
  }
}

// Joins split results: kParts waves per (row, head), which take its parts in turn, D / 64
// values a lane.  (One wave each: four of them a workgroup, along x and then y.)
template <int D, class T, int kParts>
__global__ __launch_bounds__(kParts > 4 ? 64 * kParts : 256) void attention_paged_join_kernel(
  PagedAttentionArgs a, PagedSplit split) {
  constexpr int kRegs = D / 64;
  __shared__ float lds[kParts > 1 ? kParts : 1][64 * kRegs];
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint64_t item =
    kParts > 1 ? blockIdx.x
               : ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4u + wave;
  if (item >= (uint64_t)a.batch.tokens * a.heads) {
    return;
  }
  const uint32_t token = (uint32_t)(item / a.heads), head = (uint32_t)(item % a.heads);
  const PagedRow found = paged_row(a.batch, token, a.cache.page_shift);
  const PagedSequence s = found.sequence;
  const uint32_t group = a.heads / a.cache.kv_heads;
  const bool decode = s.count * group <= split.decode_most;
  const uint32_t per = decode                  ? split.decode_keys
                       : split.tile_step != 0u ? *split.tile_chosen
                                               : split.tile_keys;
  if (s.count == 0 || s.length <= per) {
    return;  // of no sequence, or written by its workgroup
  }
  // Parts whose first key the row sees.
  const uint32_t visible = s.length - s.count + (token - s.start) + 1u;
  const uint32_t parts = (visible + per - 1u) / per;
  size_t first, stride;
  const float *o, *ml;
  if (decode) {
    first = ((size_t)found.index * a.cache.kv_heads + head / group) * split.decode_rows +
            (token - s.start) * group + head % group;
    stride = (size_t)a.batch.sequences * a.cache.kv_heads * split.decode_rows;
    o = split.decode_o;
    ml = split.decode_ml;
  } else {
    first = (size_t)token * a.heads + head;
    stride = (size_t)a.batch.tokens * a.heads;
    o = split.tile_o;
    ml = split.tile_ml;
  }
  // This wave's parts are part0, part0 + kParts, ..; four at a time, whose loads go out
  // together (past the last they repeat it, with weight 0).  Each wave keeps a maximum of
  // its own.
  const uint32_t part0 = kParts > 1 ? wave : 0u;
  float m = kLowestMax, l = 0.0f, x[kRegs] = {};
  for (uint32_t at = part0; at < parts; at += 4u * kParts) {
    float2 here[4];
    float sums[4][kRegs];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const size_t i = first + min(at + j * kParts, parts - 1u) * stride;
      here[j] = *reinterpret_cast<const float2*>(&ml[2 * i]);
#pragma unroll
      for (int r = 0; r < kRegs; ++r) {
        sums[j][r] = o[i * D + lane * kRegs + r];
      }
    }
    float up = m;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      up = fmaxf(up, here[j].x);
    }
    const float keep = fast_exp2(m - up);
    m = up;
    l *= keep;
#pragma unroll
    for (int r = 0; r < kRegs; ++r) {
      x[r] *= keep;
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const float w = at + j * kParts < parts ? fast_exp2(here[j].x - m) : 0.0f;
      l = fmaf(w, here[j].y, l);
#pragma unroll
      for (int r = 0; r < kRegs; ++r) {
        x[r] = at + j * kParts < parts ? fmaf(w, sums[j][r], x[r]) : x[r];
      }
    }
  }
  if constexpr (kParts > 1) {
    __shared__ float lds_m[kParts], lds_l[kParts];
    if (lane == 0) {
      lds_m[wave] = m;
      lds_l[wave] = l;
    }
#pragma unroll
    for (int r = 0; r < kRegs; ++r) {
      lds[wave][lane * kRegs + r] = x[r];
    }
    __syncthreads();
    // Thread i takes value i of the row.
    if (threadIdx.x >= (uint32_t)D) {
      return;
    }
    float top = lds_m[0], sum = 0.0f, value = 0.0f;
#pragma unroll
    for (int w = 1; w < kParts; ++w) {
      top = fmaxf(top, lds_m[w]);
    }
#pragma unroll
    for (int w = 0; w < kParts; ++w) {
      const float keep = fast_exp2(lds_m[w] - top);
      sum = fmaf(keep, lds_l[w], sum);
      value = fmaf(keep, lds[w][threadIdx.x], value);
    }
    store_output<T>(a, item * D + threadIdx.x, value, inverse_sum(sum));
  } else {
    float factor[kRegs];
    gate_factors<T>(a, item * D + lane * kRegs, factor);
    store_outputs<T>(a, item * D + lane * kRegs, x, inverse_sum(l), factor);
  }
}

PagedSplit split_of(const PagedAttentionArgs& a, int cu_count) {
  PagedSplit s{};
  const uint64_t group = a.heads / a.cache.kv_heads;
  const uint64_t rows = group * a.batch.max_query;
  // Keys per workgroup: 128 (a 32-key step for each wave) while all sequences at the
  // longest length make no more than eleven workgroups a CU, else as many as make so few,
  // up to 4096; enough for 128 parts of a sequence of up to 524288 keys, which one workgroup
  // joins (one sequence of 131072 keys: 34 us with 128 parts, 40 with 512, 56 with 1025),
  // beyond that 4096 all the same; more where the partial results would take over 256 MiB.
  // All of it goes by max_keys, so that a loose one makes parts too long (1 row, 4096 keys:
  // 12.8 us, with a bound of 262144 33).  (64 sequences of up to 32768 keys, 2 KV heads:
  // 512 keys 226 us, 1024 205, 1280 197, 1536 194, 2048 205.  One of 4096, 32 workgroups of
  // 128: 12.4 us.)
  const uint64_t lanes = (uint64_t)a.batch.sequences * a.cache.kv_heads;
  const uint64_t part_bytes =
    std::min<uint64_t>(rows, kDecodeRows) * (a.cache.head_dim + 2u) * sizeof(float);
  const uint64_t most = 11u * (uint64_t)cu_count;
  auto parts = [&](uint64_t k) { return lanes * ((a.batch.max_keys + k - 1u) / k); };
  uint64_t keys = (lanes * a.batch.max_keys + most - 1u) / most;
  keys = std::max<uint64_t>(keys, (a.batch.max_keys + 127u) / 128u);
  keys = std::min<uint64_t>((keys + 127u) / 128u * 128u, 4096u);
  while (parts(keys) > lanes && parts(keys) * part_bytes > (uint64_t{256} << 20)) {
    keys *= 2u;
  }
  // (A part of more keys than there are would only bring the sums of the two past 32 bits.)
  keys = std::min(keys, (a.batch.max_keys + 127u) / 128u * uint64_t{128});
  // A single sequence with many rows needs no second kernel beside the tiled one.
  s.decode_most = rows <= kDecodeRows       ? kDecodeRows
                  : a.batch.sequences > 1u ? kDecodeBlock
                                           : 0u;
  s.decode_keys = (uint32_t)keys;
  s.decode_rows = rows <= kDecodeRows ? (uint32_t)rows : kDecodeBlock;
  s.decode_splits = (uint32_t)((a.batch.max_keys + keys - 1u) / keys);
  // The tiled kernel's keys in parts of 128 at least, so that there is one for each
  // workgroup that the CUs hold at a time (one of head_dim 256, two of less), while the
  // results take no more than 256 MiB (one sequence, 37 rows at 6181 keys: 33.7 us in 100
  // parts, 31.7 in 196).  Sequences of several lengths are cut ill by the largest of them,
  // which is all that the host has: where a few parts more than fit made a second round, 17
  // sequences took 71 us in parts of 512 keys and 58 of 576.  So the kernel chooses among
  // sizes from an eighth of a round's on; of more than 64 sequences, which make rounds
  // enough, a quarter of a round's is taken.
  const uint64_t tiles = (rows + kTileRows - 1u) / kTileRows * a.cache.kv_heads;
  const uint64_t all_tiles =
    std::min<uint64_t>(tiles * a.batch.sequences,
                       ((uint64_t)a.batch.tokens * group + kTileRows - 1u) / kTileRows *
                           a.cache.kv_heads +
                         (uint64_t)a.batch.sequences * a.cache.kv_heads);
  const uint64_t row_bytes =
    (uint64_t)a.batch.tokens * a.heads * (a.cache.head_dim + 2u) * sizeof(float);
  const bool chooses = a.batch.sequences > 1u && a.batch.sequences <= 64u;
  s.tile_slots = (a.cache.head_dim == 256u ? 1u : 2u) * (uint32_t)cu_count;
  const uint64_t rounds = a.batch.sequences == 1u ? 1u : chooses ? 8u : 4u;
  uint64_t tile_keys = (a.batch.max_keys * all_tiles + rounds * s.tile_slots - 1u) /
                       (rounds * s.tile_slots);
  tile_keys = rows <= kDecodeRows ? a.batch.max_keys : std::max<uint64_t>(tile_keys, 128u);
  tile_keys = (tile_keys + 63u) / 64u * 64u;
  while (tile_keys < a.batch.max_keys &&
         (a.batch.max_keys + tile_keys - 1u) / tile_keys * row_bytes > (uint64_t{256} << 20)) {
    tile_keys *= 2u;
  }
  tile_keys = std::min(tile_keys, (a.batch.max_keys + 63u) / 64u * uint64_t{64});
  s.tile_keys = (uint32_t)tile_keys;
  // (The largest choice, 15 steps on, stays below 2^31.)
  s.tile_step = chooses && tile_keys < a.batch.max_keys
                  ? std::min((s.tile_keys / 4u + 63u) / 64u * 64u,
                             (0x7fffffffu - s.tile_keys) / 15u / 64u * 64u)
                  : 0u;
  s.tile_splits = (uint32_t)((a.batch.max_keys + s.tile_keys - 1u) / s.tile_keys);
  s.tile_blocks = (uint32_t)(all_tiles * s.tile_splits);
  return s;
}

size_t decode_parts(const PagedAttentionArgs& a, const PagedSplit& s) {
  return s.decode_splits <= 1u || s.decode_most == 0u ? 0u
                               : (size_t)s.decode_splits * a.batch.sequences * a.cache.kv_heads *
                                   s.decode_rows;
}

size_t tile_parts(const PagedAttentionArgs& a, const PagedSplit& s) {
  return s.tile_splits <= 1u ? 0u : (size_t)s.tile_splits * a.batch.tokens * a.heads;
}

template <int D, class T>
void launch_for(const PagedAttentionArgs& a, const PagedSplit& split, hipStream_t stream) {
  const uint32_t group = a.heads / a.cache.kv_heads;
  const uint64_t rows = (uint64_t)a.batch.max_query * group;
  if (group <= split.decode_most) {
    const uint32_t blocks = (split.decode_rows + kDecodeBlock - 1u) / kDecodeBlock;
    const dim3 grid(split.decode_splits * blocks * a.cache.kv_heads * a.batch.sequences);
    if (rows <= 8u) {
      attention_paged_decode_kernel<D, T, true><<<grid, 256, 0, stream>>>(a, split, PlainWork{});
    } else {
      attention_paged_decode_kernel<D, T, false><<<grid, 256, 0, stream>>>(a, split, PlainWork{});
    }
  }
  if (rows > kDecodeRows) {
    launch_attention_paged_q8_tiles(a, split, stream);
  }
  const uint64_t items = (uint64_t)a.batch.tokens * a.heads;
  const uint32_t parts = std::max(split.decode_most != 0u ? split.decode_splits : 1u,
                                  rows > kDecodeRows ? split.tile_splits : 1u);
  // Sixteen waves a row, or four, where there are many parts and few rows (one row of 33
  // parts: 7.3 us with one, 4 with four; a call with 129 parts of 8 rows 17.9 us with four,
  // 15.8 with sixteen), one where the rows alone fill the device (14544 rows, most of four
  // parts or fewer: 18.6 us with four, 9.0 with one).
  if (parts > 32u && items <= 1024u) {
    attention_paged_join_kernel<D, T, 16><<<dim3((uint32_t)items), 1024, 0, stream>>>(a, split);
  } else if (parts > 8u && items <= 4096u) {
    attention_paged_join_kernel<D, T, 4><<<dim3((uint32_t)items), 256, 0, stream>>>(a, split);
  } else if (parts > 1u) {
    // A dimension of the grid holds less than 2^32 threads, which 2^26 rows' waves are.
    const uint32_t blocks = (uint32_t)((items + 3u) / 4u);
    const uint32_t across = std::min(blocks, kJoinAcross);
    attention_paged_join_kernel<D, T, 1>
      <<<dim3(across, (blocks + across - 1u) / across), 256, 0, stream>>>(a, split);
  }
}

template <class T>
void launch_type(const PagedAttentionArgs& a, const PagedSplit& split, hipStream_t stream) {
  if (a.cache.head_dim == 256u) {
    launch_for<256, T>(a, split, stream);
  } else if (a.cache.head_dim == 128u) {
    launch_for<128, T>(a, split, stream);
  } else {
    launch_for<64, T>(a, split, stream);
  }
}

}  // namespace

namespace {

template <int D, class T>
void launch_shared_decode_for(const PagedAttentionArgs& a, const SharedWork& work,
                              uint32_t decode_rows, uint32_t workgroups, hipStream_t stream) {
  if (decode_rows == 8u) {
    attention_paged_decode_kernel<D, T, true>
      <<<dim3(workgroups), 256, 0, stream>>>(a, PagedSplit{}, work);
  } else {
    attention_paged_decode_kernel<D, T, false>
      <<<dim3(workgroups), 256, 0, stream>>>(a, PagedSplit{}, work);
  }
}

template <class T>
void launch_shared_decode_type(const PagedAttentionArgs& a, const SharedWork& work,
                               uint32_t decode_rows, uint32_t workgroups, hipStream_t stream) {
  if (a.cache.head_dim == 256u) {
    launch_shared_decode_for<256, T>(a, work, decode_rows, workgroups, stream);
  } else if (a.cache.head_dim == 128u) {
    launch_shared_decode_for<128, T>(a, work, decode_rows, workgroups, stream);
  } else {
    launch_shared_decode_for<64, T>(a, work, decode_rows, workgroups, stream);
  }
}

}  // namespace

void launch_shared_decode(const PagedAttentionArgs& a, const SharedWork& work,
                          uint32_t decode_rows, uint32_t workgroups, hipStream_t stream) {
  if (a.f16) {
    launch_shared_decode_type<half_t>(a, work, decode_rows, workgroups, stream);
  } else {
    launch_shared_decode_type<float>(a, work, decode_rows, workgroups, stream);
  }
}

size_t attention_paged_q8_workspace_bytes(const PagedAttentionArgs& a, int cu_count) {
  const PagedSplit s = split_of(a, cu_count);
  return (decode_parts(a, s) + tile_parts(a, s)) * (a.cache.head_dim + 2u) * sizeof(float) +
         sizeof(uint32_t);
}

hipError_t launch_attention_paged_q8(const PagedAttentionArgs& a, int cu_count, void* workspace,
                                     hipStream_t stream) {
  PagedSplit s = split_of(a, cu_count);
  s.decode_o = static_cast<float*>(workspace);
  s.tile_o = s.decode_o + decode_parts(a, s) * a.cache.head_dim;
  s.decode_ml = s.tile_o + tile_parts(a, s) * a.cache.head_dim;
  s.tile_ml = s.decode_ml + decode_parts(a, s) * 2u;
  s.tile_chosen = reinterpret_cast<uint32_t*>(s.tile_ml + tile_parts(a, s) * 2u);
  if (a.f16) {
    launch_type<half_t>(a, s, stream);
  } else {
    launch_type<float>(a, s, stream);
  }
  return hipGetLastError();
}

}  // namespace kraken
