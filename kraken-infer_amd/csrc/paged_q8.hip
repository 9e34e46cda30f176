// The attention prologue of a ragged batch into 8-bit KV pages, and pages read back
// as F16 rows.
//
// A page's codes stand for code * scale, one f32 scale for each page and KV head,
// keys and values apart.  With A the largest magnitude among a call's new rows of a
// page, the scale is A / 127 for a page begun by the call; for one that holds older
// rows it is the old scale times the least 2^j with A <= 127 s 2^j, and the older
// codes become rne(code 2^-j).  Doubling keeps the cost of many small growths
// bounded: each rounds the older codes by at most half a step of its scale, and half
// steps of s, 2s, 4s, .. add up to less than one step of the last.
//
// One workgroup owns the new rows of one (sequence, page, KV head, keys or values):
// it needs the largest magnitude of all of them before it can write the first code,
// so it holds them in registers (up to 8 rows a wave), and no second pass or launch is
// needed.  The codes go through LDS, from which they leave in the layout of the pages:
// rows for keys, runs of eight tokens a dimension for values.  The query heads are further
// workgroups of the same launch, a wave per token and run of heads.
//
// 1024 tokens of 8 query and 2 KV heads of 256 (39 MB read and written, 8 us at the rate of
// a copy) take 13.4 us, the query heads alone (34 MB; page numbers outside the pool) 10.8:
// the 68 workgroups of pages (17 pages, 2 heads, keys and values) run beside those.  Rows
// are loaded and stored a dword a lane.  4096 tokens 38.7 us, queries alone 30.  One token
// takes 6.2 us in a row of calls, 4.8 traced, of which a launch is 2 to 3.  Reading pages
// of 64 tokens back as F16: one 4.8 us, 17 5.2, 512 18.1 (5.6 TB/s), 2048 84 (4.8).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention_prologue_common.hpp"
#include "context_internal.hpp"
#include "device_common.hpp"
#include "paged_q8_internal.hpp"

namespace kraken {
namespace {

// The rotation of elements lane + 64 i below n_dims: turns per position (the angle
// over 2 pi, in double, so that a position of any size keeps its fraction), and the
// MRoPE row that the element's position comes from.
struct Rotation {
  double turns[4];
  uint32_t row[4];
};

__device__ __forceinline__ Rotation rotation_of(const PagedPrologueArgs& a, int lane) {
  Rotation r;
  const uint32_t half_dims = a.n_dims / 2u;
  const uint32_t sections = a.s0 + a.s1 + a.s2 + a.s3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t e = lane + 64u * i;
    if (e < a.n_dims) {
      const uint32_t pair = e < half_dims ? e : e - half_dims;
      const uint32_t sector = pair % sections;
      r.row[i] = sector < a.s0 ? 0u
                 : sector < a.s0 + a.s1 ? 1u
                 : sector < a.s0 + a.s1 + a.s2 ? 2u : 3u;
      r.turns[i] = exp2(-a.log2_theta * (double)(2u * pair) / (double)a.n_dims) *
                   0.15915494309189533577;
    }
  }
  return r;
}

// The angle is reduced to a part of a half turn in 64 bits and rounded to f32 there, which
// moves it by up to pi 2^-25, three of the sine's own roundings: a rotated query is 6.3e-8
// of itself off, with 64-bit sines 5.5e-8, and a few key codes in a million take the
// neighbour.  64-bit sines would be most of a short call's arithmetic.
__device__ __forceinline__ void sin_cos_of(const PagedPrologueArgs& a, const Rotation& rot,
                                           uint32_t token, uint32_t position, int lane,
                                           float sn[4], float cs[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t e = lane + 64u * i;
    if (e < a.n_dims) {
      const int32_t p = a.positions != nullptr
                          ? a.positions[min(token, a.batch.tokens - 1u) +
                                        (size_t)a.batch.tokens * rot.row[i]]
                          : (int32_t)position;
      const double t = (double)p * rot.turns[i];
      sincospif((float)(2.0 * (t - rint(t))), &sn[i], &cs[i]);
    }
  }
}

// norm_rope of the F16 prologue with the rotation in f32.
__device__ __forceinline__ void norm_rotate(const float v_in[4], const float w[4], uint32_t d_head,
                                            float eps, uint32_t n_dims, const float sn[4],
                                            const float cs[4], int lane, float r[4]) {
  float v[4], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum = fmaf(v_in[i], v_in[i], sum);
  }
  sum = wave_sum(sum);
  const float scale = 1.0f / sqrtf(sum / (float)d_head + eps);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = lane + 64u * i < d_head ? v_in[i] * scale * w[i] : 0.0f;
  }
  const uint32_t half_dims = n_dims / 2u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = v[i];
    const uint32_t e = lane + 64u * i;
    if (64u * i >= n_dims) {
      continue;  // uniform
    }
    const uint32_t p = e < half_dims ? e + half_dims : (e < n_dims ? e - half_dims : e);
    float partner = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (64u * j < n_dims) {
        const float x = __shfl(v[j], (int)(p & 63u), 64);
        partner = p >> 6 == (uint32_t)j ? x : partner;
      }
    }
    if (e < n_dims) {
      r[i] = e < half_dims ? v[i] * cs[i] - partner * sn[i] : v[i] * cs[i] + partner * sn[i];
    }
  }
}

// A wave: kHeads query heads of one token from `first` on.
template <int kHeads>
__device__ __forceinline__ void query_heads(const PagedPrologueArgs& a, uint32_t token,
                                            uint32_t first, int lane) {
  const uint32_t d_head = a.cache.head_dim;
  // Every load first; past the last head, its own again.
  float v[kHeads][4], g[kHeads][4], w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t d = lane + 64u * i;
    w[i] = d < d_head ? a.q_norm[d] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    const uint32_t head = min(first + k, a.heads - 1u);
    const float* src = a.q_gate + ((size_t)token * a.heads + head) * 2u * d_head;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t d = lane + 64u * i;
      v[k][i] = d < d_head ? src[d] : 0.0f;
      g[k][i] = d < d_head ? src[d_head + d] : 0.0f;
    }
  }
  const PagedSequence s = paged_row(a.batch, token, a.cache.page_shift).sequence;
  if (s.count == 0) {
    return;
  }
  const Rotation rot = rotation_of(a, lane);
  float sn[4], cs[4];
  sin_cos_of(a, rot, token, s.length - s.count + (token - s.start), lane, sn, cs);
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    float r[4];
    norm_rotate(v[k], w, d_head, a.eps, a.n_dims, sn, cs, lane, r);
    if (first + k < a.heads) {
      float* q_out = a.query_out + ((size_t)token * a.heads + first + k) * d_head;
      float* g_out = a.gate_out + ((size_t)token * a.heads + first + k) * d_head;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t d = lane + 64u * i;
        if (d < d_head) {
          q_out[d] = r[i];
          g_out[d] = g[k][i];
        }
      }
    }
  }
}

// The new scale of a page and the factor of its older codes.  `largest` holds the
// bits of the largest magnitude (above those of infinity: a NaN among the rows).
__device__ __forceinline__ void grow_scale(uint32_t largest_bits, float old_scale, bool begun,
                                           float& scale, float& factor) {
  factor = 1.0f;
  const float largest = __uint_as_float(largest_bits);
  const float nan = __uint_as_float(0x7fc00000u);
  if (largest_bits >= 0x7f800000u || !(begun || old_scale >= 0.0f)) {
    scale = nan;
    return;
  }
  if (begun || old_scale == 0.0f) {
    const float s = largest / 127.0f;
    scale = s < kLeastScale ? 0.0f : s;
    factor = 0.0f;  // older codes under a zero scale are zeros
    return;
  }
  // A <= 127 s 2^j exactly, in double; at most 277 steps from the smallest s.
  double limit = 127.0 * (double)old_scale;
  scale = old_scale;
  for (int j = 0; j < 300 && (double)largest > limit; ++j) {
    limit *= 2.0;
    scale *= 2.0f;
    factor *= 0.5f;
  }
}

// A page's new rows [first, last) (slots of the page), row `row` + slot - first of
// the batch; kRows rows a wave.
template <int kRows, int kWaves>
__device__ __forceinline__ void page_rows(const PagedPrologueArgs& a, bool is_value, uint32_t page,
                                          uint32_t kv_head, uint32_t first, uint32_t last,
                                          uint32_t row, uint32_t position, int8_t* codes,
                                          uint32_t* wave_largest) {
  constexpr uint32_t kThreads = 64 * kWaves;
  const int lane = threadIdx.x & 63;
  const uint32_t wave = threadIdx.x >> 6;
  const uint32_t d_head = a.cache.head_dim;
  const uint32_t rows = last - first;
  const uint32_t page_tokens = 1u << a.cache.page_shift;
  const size_t kv_dim = (size_t)a.cache.kv_heads * d_head;
  const float* src = (is_value ? a.value : a.key) + (size_t)row * kv_dim + (size_t)kv_head * d_head;
  const size_t page_head = (size_t)page * a.cache.kv_heads + kv_head;
  float* scale_at = (is_value ? a.cache.value_scales : a.cache.key_scales) + page_head;
  const float old_scale = *scale_at;
  int8_t* out = (is_value ? a.cache.values : a.cache.keys) + page_head * page_tokens * d_head;
  // The eight tokens of a dimension that this thread will write first, should some of them
  // be older ones; asked for here so that they arrive with the rows.
  uint64_t early = 0;
  if (is_value && first % 8u != 0 && threadIdx.x < d_head) {
    early = *reinterpret_cast<const uint64_t*>(
      out + ((size_t)(first / 8u) * d_head + threadIdx.x) * 8u);
  }

  float r[kRows][4];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const uint32_t at = wave + kWaves * k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t d = lane + 64u * i;
      r[k][i] = at < rows && d < d_head ? src[(size_t)at * kv_dim + d] : 0.0f;
    }
  }
  if (!is_value) {
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t d = lane + 64u * i;
      w[i] = d < d_head ? a.k_norm[d] : 0.0f;
    }
    const Rotation rot = rotation_of(a, lane);
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      // (Past the last row: of zeros.)
      const uint32_t at = wave + kWaves * k;
      float sn[4], cs[4], turned[4];
      sin_cos_of(a, rot, row + at, position + at, lane, sn, cs);
      norm_rotate(r[k], w, d_head, a.eps, a.n_dims, sn, cs, lane, turned);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r[k][i] = turned[i];
      }
    }
  }
  // The largest magnitude, by its bits: a NaN's lie above infinity's.
  uint32_t largest = 0;
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      largest = max(largest, __float_as_uint(r[k][i]) & 0x7fffffffu);
    }
  }
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    largest = max(largest, (uint32_t)__shfl_xor((int)largest, step, 64));
  }
  if (lane == 0) {
    wave_largest[wave] = largest;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    largest = max(largest, wave_largest[k]);
  }
  float scale, factor;
  grow_scale(largest, old_scale, first == 0, scale, factor);
  const float inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const uint32_t at = wave + kWaves * k;
    if (at < rows) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t d = lane + 64u * i;
        if (d < d_head) {
          // A NaN (its page's scale says so already) is held as zero.
          const float x = r[k][i] * inverse;
          const float q = fminf(fmaxf(rintf(x), -127.0f), 127.0f);
          codes[(size_t)at * d_head + d] = x == x ? (int8_t)(int)q : (int8_t)0;
        }
      }
    }
  }
  if (threadIdx.x == 0 && __float_as_uint(scale) != __float_as_uint(old_scale)) {
    *scale_at = scale;
  }
  __syncthreads();

  // Older codes change where the scale grew.
  const uint32_t older = factor == 1.0f ? 0u : first;
  auto shrink = [&](int8_t c) { return (int8_t)(int)rintf((float)c * factor); };
  if (!is_value) {
    // 16 bytes of a row at a time.
    const uint32_t per_row = d_head / 16u;
    const uint32_t from = older != 0 ? 0u : first;
    for (uint32_t i = threadIdx.x; i < (last - from) * per_row; i += kThreads) {
      const uint32_t slot = from + i / per_row, d = (i % per_row) * 16u;
      int4* at = reinterpret_cast<int4*>(out + (size_t)slot * d_head + d);
      if (slot >= first) {
        *at = *reinterpret_cast<const int4*>(codes + (size_t)(slot - first) * d_head + d);
      } else {
        int4 held = *at;
        int8_t* c = reinterpret_cast<int8_t*>(&held);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          c[k] = shrink(c[k]);
        }
        *at = held;
      }
    }
  } else {
    // Eight tokens of a dimension at a time: new ones from LDS, older ones shrunk
    // where the scale grew, those behind the last kept.
    const uint32_t from = (older != 0 ? 0u : first) / 8u, to = (last + 7u) / 8u;
    for (uint32_t i = threadIdx.x; i < (to - from) * d_head; i += kThreads) {
      const uint32_t octet = from + i / d_head, d = i % d_head;
      uint64_t* at = reinterpret_cast<uint64_t*>(out + ((size_t)octet * d_head + d) * 8u);
      const bool whole = octet * 8u >= first && octet * 8u + 8u <= last;
      uint64_t held = 0;
      if (!whole) {
        // (i is the dimension in the first run of them.)
        held = i < d_head && octet == first / 8u && first % 8u != 0 ? early : *at;
      }
      uint64_t made = 0;
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) {
        const uint32_t slot = octet * 8u + k;
        int8_t c = (int8_t)(held >> (8u * k));
        if (slot >= first && slot < last) {
          c = codes[(size_t)(slot - first) * d_head + d];
        } else if (slot < older) {
          c = shrink(c);
        }
        made |= (uint64_t)(uint8_t)c << (8u * k);
      }
      *at = made;
    }
  }
}

// Blocks [0, page_blocks): the new rows of a page for one KV head, keys or values.
// The rest: query heads, a wave per token and run of kHeads of them.  Both
// walk their items in steps of their blocks, whose number is bounded.
template <int kRows, int kWaves, int kHeads>
__global__ __launch_bounds__(64 * kWaves) void prologue_paged_q8_kernel(PagedPrologueArgs a,
                                                                        uint32_t spans,
                                                                        uint32_t page_blocks) {
  extern __shared__ __attribute__((aligned(16))) int8_t codes[];
  __shared__ uint32_t wave_largest[kWaves];
  if (blockIdx.x < page_blocks) {
    const uint32_t kinds = 2u * a.cache.kv_heads, shift = a.cache.page_shift;
    const uint64_t items = (uint64_t)a.batch.sequences * spans * kinds;
    for (uint64_t item = blockIdx.x; item < items; item += page_blocks) {
      const uint32_t kind = (uint32_t)(item % kinds);
      const uint64_t span = item / kinds;
      const uint32_t b = (uint32_t)(span / spans);
      const PagedSequence s = paged_sequence(a.batch, b, shift);
      const uint32_t begin = s.length - s.count;
      const uint64_t index = (begin >> shift) + span % spans;
      const uint64_t page_begin = index << shift;
      if (s.count == 0 || page_begin >= s.length) {
        continue;
      }
      const uint32_t first = max(begin, (uint32_t)page_begin);
      const uint32_t last = min(s.length, (uint32_t)page_begin + (1u << shift));
      const int32_t page = a.batch.table[(size_t)b * a.batch.width + index];
      if (page < 0 || (uint32_t)page >= a.cache.pages) {
        continue;
      }
      __syncthreads();  // the last item's codes have left LDS
      page_rows<kRows, kWaves>(a, kind & 1u, (uint32_t)page, kind >> 1,
                               first - (uint32_t)page_begin, last - (uint32_t)page_begin,
                               s.start + (first - begin), first, codes, wave_largest);
    }
    return;
  }
  const uint32_t groups = (a.heads + kHeads - 1u) / kHeads;
  const uint64_t items = (uint64_t)a.batch.tokens * groups;
  const uint64_t stride = (uint64_t)(gridDim.x - page_blocks) * kWaves;
  for (uint64_t item = (uint64_t)(blockIdx.x - page_blocks) * kWaves + (threadIdx.x >> 6);
       item < items; item += stride) {
    query_heads<kHeads>(a, (uint32_t)(item / groups), (uint32_t)(item % groups) * kHeads,
                        threadIdx.x & 63);
  }
}

__global__ __launch_bounds__(256) void dequantize_pages_q8_kernel(PagedQ8Args c,
                                                                  const int32_t* ids,
                                                                  half_t* key_rows,
                                                                  half_t* value_rows) {
  const uint32_t kv_head = blockIdx.x % c.kv_heads;
  const uint32_t i = blockIdx.x / c.kv_heads;
  const bool is_value = blockIdx.y != 0;
  const uint32_t page_tokens = 1u << c.page_shift, d_head = c.head_dim;
  const int32_t page = ids[i];
  const bool inside = page >= 0 && (uint32_t)page < c.pages;
  const size_t page_head = (size_t)(inside ? page : 0) * c.kv_heads + kv_head;
  const size_t row = (size_t)c.kv_heads * d_head;
  half_t* out = (is_value ? value_rows : key_rows) + (size_t)i * page_tokens * row +
                (size_t)kv_head * d_head;
  const float scale = (is_value ? c.value_scales : c.key_scales)[page_head];
  const int8_t* codes = (is_value ? c.values : c.keys) + page_head * page_tokens * d_head;
  const uint32_t groups = page_tokens * d_head / 8u;
  for (uint32_t k = threadIdx.x; k < groups; k += 256) {
    const uint64_t eight = inside ? reinterpret_cast<const uint64_t*>(codes)[k] : 0u;
    half8_t x;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = (float)(int8_t)(eight >> (8 * j)) * scale;
      x[j] = inside ? static_cast<half_t>(v) : static_cast<half_t>(0.0f);
    }
    if (is_value) {
      const uint32_t octet = k / d_head, d = k % d_head;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        out[(size_t)(octet * 8u + j) * row + d] = x[j];
      }
    } else {
      const uint32_t slot = k * 8u / d_head, d = k * 8u % d_head;
      *reinterpret_cast<half8_t*>(out + (size_t)slot * row + d) = x;
    }
  }
}

}  // namespace

namespace {

template <int kRows, int kWaves, int kHeads>
void launch_prologue(const PagedPrologueArgs& a, uint32_t rows, hipStream_t stream) {
  const uint32_t page_tokens = 1u << a.cache.page_shift;
  // Pages that max_query new tokens can reach into.
  const uint64_t spans = (a.batch.max_query + (uint64_t)page_tokens - 2u) / page_tokens + 1u;
  const uint64_t page_blocks =
    std::min<uint64_t>((uint64_t)a.batch.sequences * spans * a.cache.kv_heads * 2u, 1u << 20);
  const uint64_t groups = (a.heads + kHeads - 1u) / kHeads;
  const uint64_t blocks =
    page_blocks +
    std::min<uint64_t>((a.batch.tokens * groups + kWaves - 1u) / kWaves, 1u << 20);
  prologue_paged_q8_kernel<kRows, kWaves, kHeads>
    <<<dim3((uint32_t)blocks), 64 * kWaves, rows * a.cache.head_dim, stream>>>(
      a, (uint32_t)spans, (uint32_t)page_blocks);
}

}  // namespace

hipError_t launch_prologue_paged_q8(const PagedPrologueArgs& a, hipStream_t stream) {
  const uint32_t rows = std::min(1u << a.cache.page_shift, a.batch.max_query);
  // A decode step: a wave a row and a query head, four waves.  Chunks: as few waves on a
  // page's rows as eight rows each take, since a page's chain of loads, norms, the largest
  // magnitude and codes is as long for one row as for all, and many short workgroups share
  // a CU; four query heads a wave, which share the token's angles.  (us, with the pages
  // read back.  1 token 11.0 with 8 waves, 10.7 with 4; 64 tokens 14.6 and 12.2.  16
  // sequences, 2000 tokens, 8 heads of 128, pages of 16: 16 waves 178, 4 waves 56; 24
  // sequences, 1600 tokens, pages of 32: 70 and 39.  Pages of 64: 1024 tokens 20.1 with 16
  // waves, 20.4 with 8, 24 sequences 72 and 65; one query head a wave 22.9.)
  if (rows <= 4u) {
    launch_prologue<1, 4, 1>(a, rows, stream);
  } else if (rows <= 16u) {
    launch_prologue<4, 4, 4>(a, rows, stream);
  } else if (rows <= 32u) {
    launch_prologue<8, 4, 4>(a, rows, stream);
  } else if (rows <= 64u) {
    launch_prologue<8, 8, 4>(a, rows, stream);
  } else {
    launch_prologue<8, 16, 4>(a, rows, stream);
  }
  return hipGetLastError();
}

hipError_t launch_dequantize_pages_q8(const PagedQ8Args& c, const int32_t* ids, uint32_t count,
                                      void* key_rows, void* value_rows, hipStream_t stream) {
  dequantize_pages_q8_kernel<<<dim3(count * c.kv_heads, 2u), 256, 0, stream>>>(
    c, ids, static_cast<half_t*>(key_rows), static_cast<half_t*>(value_rows));
  return hipGetLastError();
}

}  // namespace kraken
