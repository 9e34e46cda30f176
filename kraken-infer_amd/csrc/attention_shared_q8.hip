// Causal attention of a ragged batch over 8-bit KV pages whose sequences share prefixes:
// each group's shared keys against all rows of its sequences, what is left of each
// sequence against its own rows, and the join of a row's two softmaxes.
//
// A prefix's part needs no mask (all its keys stand before all the group's new tokens),
// and its keys are read once for the group instead of once for each sequence.  Both kinds
// of item go through the kernels of the plain call: those of few rows through the decode
// kernel, which takes single keys' rows from memory to the matrix cores, the others
// through the tiled one, 128 rows a workgroup.  A launch before lists the items from the
// batch's arrays and cuts their keys, by their numbers and not by the host's bounds.
//
// 64 sequences of one token behind 32768 shared ones (two KV heads of 256, groups of four,
// up to 4096 keys of their own): 100 us, and 358 by the plain call.  Traced, the shared keys'
// tiles 51 us (17 GFLOP, twice for the f32 query's two parts: the matrix cores and the
// softmax in one wave a SIMD), the sequences' own keys 42 (134 MB), the join 10, the plan 6;
// one after another, as the tiles' registers leave no room beside them.  Three prompts of 8192
// with eight sequences of eight drafted tokens each (f16, eight heads of 128): 56 us, of which
// 29, 14, 11 and 6.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention_paged_q8_common.hpp"
#include "context_internal.hpp"
#include "device_common.hpp"
#include "row_order.hpp"

namespace kraken {
namespace {

constexpr uint32_t kPlanThreads = 256;
constexpr uint32_t kPlanWaves = kPlanThreads / 64u;
constexpr uint32_t kHeldItems = 1024;  // listed in LDS on the way to memory
constexpr uint32_t kChoices = 16;      // sizes of the tiled kernel's parts that are tried

// What the host gives the plan.
struct SharedLimits {
  uint32_t group;         // query heads of a KV head
  uint32_t decode_most;   // rows up to which an item goes to the decode kernel
  uint32_t decode_shift;  // log2 of the rows of a block of it
  uint32_t decode_many;   // workgroups beyond which they take more keys
  uint32_t decode_slots;  // workgroups that its work is cut into
  uint32_t tile_slots;    // workgroups of the tiled kernel that run at once
  uint32_t planes[2];     // parts that there is room for, of sequences and of groups
};

struct SharedLists {
  SharedItem* items;
  uint32_t* ends;
  uint32_t* keys;
};

// Rows' blocks of an item in the kernel that takes it (0: the decode kernel, 1: the tiled
// one); 0 blocks without rows.
struct ItemWork {
  uint32_t kind, blocks;
};

__device__ __forceinline__ ItemWork work_of(const SharedLimits& l, const SharedItem& i) {
  const uint32_t rows = i.count * l.group;
  const bool few = rows <= l.decode_most;
  const uint32_t shift = few ? l.decode_shift : 7u;
  static_assert(kTileRows == 1u << 7, "");
  return {few ? 0u : 1u, (rows + (1u << shift) - 1u) >> shift};
}

// One workgroup, which for 64 sequences takes 6 us: a chain of loads and scans.
__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(PagedAttentionArgs a,
                                                                   SharedPrefixArgs p,
                                                                   SharedLimits l,
                                                                   SharedLists lists) {
  __shared__ SharedItem held[kHeldItems];
  __shared__ uint32_t held_starts[kHeldItems + 1u];
  __shared__ float sums[kPlanWaves][2], times[kChoices];
  __shared__ uint32_t most[kPlanWaves][4], scans[kPlanWaves][2];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t sequences = a.batch.sequences, shift = a.cache.page_shift;
  const uint32_t count = p.groups + sequences;
  const bool small = count <= kHeldItems;
  SharedItem* const items = small ? held : lists.items;
  const uint32_t* const starts = small ? held_starts : a.batch.starts;

  // The arrays' loads go out together: of a wave's first group too.
  uint32_t group_begin = 0, group_end = 0, group_prefix = 0;
  if (wave < p.groups) {
    group_begin = p.starts[wave];
    group_end = p.starts[wave + 1u];
    group_prefix = p.lengths[wave];
  }
  for (uint32_t i = tid; i < count; i += kPlanThreads) {
    SharedItem item{0u, 0u, 0u, 0u, 0u, kIsGroup};
    if (i >= p.groups) {
      const PagedSequence q = paged_sequence(a.batch, i - p.groups, shift);
      item = {q.start, q.count, q.length, i - p.groups, 0u, kNoGroup};
      if (small) {
        held_starts[i - p.groups] = q.start;
        if (i + 1u == count) {
          held_starts[sequences] = a.batch.starts[sequences];
        }
      }
    }
    items[i] = item;
  }
  __syncthreads();

  // A wave a group.
  for (uint32_t g = wave; g < p.groups; g += kPlanWaves) {
    if (g != wave) {
      group_begin = p.starts[g];
      group_end = p.starts[g + 1u];
      group_prefix = p.lengths[g];
    }
    const uint32_t begin = group_begin, end = group_end;
    if (begin >= end || end > sequences || group_prefix > p.max_prefix) {
      continue;
    }
    const uint32_t row = starts[begin], stop = starts[end];
    if (row >= stop || stop > a.batch.tokens || stop - row > p.max_rows) {
      continue;
    }
    // Its sequences with rows: how many, the first, and the fewest tokens before the new
    // ones; whether all their rows lie in the group's.
    uint32_t least = group_prefix, first = end, live = 0;
    bool fits = true;
    for (uint32_t i = begin + lane; i < end; i += 64u) {
      const SharedItem q = items[p.groups + i];
      if (q.count != 0) {
        least = min(least, q.length - q.count);
        first = min(first, i);
        live += 1u;
        fits = fits && q.start >= row && q.start + q.count <= stop;
      }
    }
    // (The smallest of x is what the largest of ~x leaves.)
    least = ~(uint32_t)__builtin_amdgcn_readlane((int)wave_scan(~least, Largest{}), 63);
    first = ~(uint32_t)__builtin_amdgcn_readlane((int)wave_scan(~first, Largest{}), 63);
    live = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(live, Sum{}), 63);
    const uint32_t shared = least >> shift << shift;
    // (A single sequence would gain nothing.)
    if (!__all(fits) || live < 2u || shared == 0) {
      continue;
    }
    if (lane == 0) {
      items[g] = {row, stop - row, shared, first, 0u, kIsGroup};
    }
    for (uint32_t i = begin + lane; i < end; i += 64u) {
      SharedItem* q = &items[p.groups + i];
      if (q->count != 0) {
        // `first` and `group` in one store: of a sequence that two groups claim they are
        // those of one.
        __hip_atomic_store(reinterpret_cast<uint64_t*>(&q->first), (uint64_t)g << 32 | shared,
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
    }
  }
  __syncthreads();

  // Rows' blocks times keys for each kernel, and the longest of each kind of item in it.
  float all[2] = {0.0f, 0.0f};
  uint32_t longest[4] = {0, 0, 0, 0};
  for (uint32_t i = tid; i < count; i += kPlanThreads) {
    const SharedItem q = items[i];
    const ItemWork w = work_of(l, q);
    const uint32_t keys = w.blocks != 0 ? q.length - q.first : 0u;
    const uint32_t at = 2u * w.kind + (i < p.groups ? 1u : 0u);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      longest[k] = at == k ? max(longest[k], keys) : longest[k];
    }
    all[0] += w.kind == 0 ? (float)w.blocks * (float)keys : 0.0f;
    all[1] += w.kind == 1 ? (float)w.blocks * (float)keys : 0.0f;
  }
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    longest[k] = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(longest[k], Largest{}), 63);
  }
  all[0] = wave_sum(all[0]);
  all[1] = wave_sum(all[1]);
  if (lane == 0) {
    sums[wave][0] = all[0];
    sums[wave][1] = all[1];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      most[wave][k] = longest[k];
    }
  }
  __syncthreads();
  all[0] = all[1] = 0.0f;
#pragma unroll
  for (uint32_t w = 0; w < kPlanWaves; ++w) {
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
      all[k] += sums[w][k] * (float)a.cache.kv_heads;
      longest[2 * k] = max(longest[2 * k], most[w][2 * k]);
      longest[2 * k + 1] = max(longest[2 * k + 1], most[w][2 * k + 1]);
    }
  }
  // Keys of a part, so that an item's parts have room.
  uint32_t need[2];
#pragma unroll
  for (uint32_t k = 0; k < 2; ++k) {
    need[k] = max((longest[2 * k] + l.planes[0] - 1u) / l.planes[0],
                  (longest[2 * k + 1] + l.planes[1] - 1u) / l.planes[1]);
  }
  // The decode kernel's: as many workgroups as its slots, of 128 to 4096 keys; 256 at least
  // where they are more than 4 a CU all the same, as a workgroup's way to its first keys is
  // long (64 sequences of up to 4096 own keys: the call 110 us with 128, 100 with 256, 104
  // with 512; four of up to 256: 20.9 and 22.0).
  const float least = all[0] > 128.0f * (float)l.decode_many ? 256.0f : 128.0f;
  const float wanted = fminf(fmaxf(all[0] / (float)l.decode_slots, least), 4096.0f);
  const uint32_t decode_keys = (max((uint32_t)wanted, need[0]) + 127u) / 128u * 128u;
  // The tiled kernel's: of sixteen sizes the one whose rounds of `tile_slots` workgroups are
  // soonest over, each round taking its keys and what a workgroup spends besides (about 128
  // keys' time).  Tried are those that make one round, two .. eight if all parts were full,
  // and an eighth more.
  auto tile_keys = [&](uint32_t choice) {
    const float rounds = (float)(1u + choice / 2u) * (float)l.tile_slots;
    const float keys = all[1] / rounds * (choice % 2u != 0u ? 1.125f : 1.0f);
    return (max((uint32_t)fminf(fmaxf(keys, 128.0f), 1e9f), need[1]) + 63u) / 64u * 64u;
  };
  uint32_t best = 0;
  if (all[1] > 0.0f) {
    for (uint32_t c = wave; c < kChoices; c += kPlanWaves) {
      const float keys = (float)tile_keys(c);
      float total = 0.0f;
      for (uint32_t i = lane; i < count; i += 64u) {
        const SharedItem q = items[i];
        const ItemWork w = work_of(l, q);
        total += w.kind == 1 ? (float)w.blocks * ceilf((float)(q.length - q.first) / keys) : 0.0f;
      }
      total = wave_sum(total) * (float)a.cache.kv_heads;
      if (lane == 0) {
        times[c] = ceilf(total / (float)l.tile_slots) * (keys + 128.0f);
      }
    }
    __syncthreads();
    float least = times[0];
#pragma unroll
    for (uint32_t c = 1; c < kChoices; ++c) {
      best = times[c] < least ? c : best;
      least = fminf(times[c], least);
    }
  }
  const uint32_t part_keys[2] = {decode_keys, tile_keys(best)};
  if (tid == 0) {
    lists.keys[0] = part_keys[0];
    lists.keys[1] = part_keys[1];
  }
  // The workgroups up to each item.
  uint32_t before[2] = {0, 0};
  for (uint32_t base = 0; base < count; base += kPlanThreads) {
    const uint32_t i = base + tid;
    uint32_t upto[2] = {0, 0};
    if (i < count) {
      const SharedItem q = items[i];
      const ItemWork w = work_of(l, q);
      const uint32_t keys = part_keys[w.kind];
      const uint32_t mine = w.blocks * ((q.length - q.first + keys - 1u) / keys);
      upto[0] = w.kind == 0 ? mine : 0u;
      upto[1] = w.kind == 1 ? mine : 0u;
      if (small) {
        lists.items[i] = q;
      }
    }
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
      upto[k] = wave_scan(upto[k], Sum{});
    }
    __syncthreads();
    if (lane == 63u) {
      scans[wave][0] = upto[0];
      scans[wave][1] = upto[1];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
      upto[k] += before[k];
#pragma unroll
      for (uint32_t w = 0; w < kPlanWaves; ++w) {
        upto[k] += w < wave ? scans[w][k] : 0u;
        before[k] += scans[w][k];
      }
      if (i < count) {
        lists.ends[(size_t)k * count + i] = upto[k];
      }
    }
  }
}

// Joins the parts of a group and of a sequence: kParts waves per (row, head), which take
// them in turn, D / 64 values a lane; those of the group before the sequence's own.
template <int D, class T, int kParts>
__global__ __launch_bounds__(64 * kParts) void shared_join_kernel(PagedAttentionArgs a,
                                                                  SharedWork work, uint32_t groups,
                                                                  uint32_t decode_most) {
  constexpr int kRegs = D / 64;
  __shared__ float lds[kParts][64 * kRegs];
  __shared__ float lds_m[kParts], lds_l[kParts];
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t row = blockIdx.x, token = row / a.heads;
  const uint32_t group = a.heads / a.cache.kv_heads;
  const PagedRow found = paged_row(a.batch, token, a.cache.page_shift);
  if (found.sequence.count == 0) {
    return;
  }
  const SharedItem mine = work.items[groups + found.index];
  const uint32_t keys = work.keys[mine.count * group <= decode_most ? 0 : 1];
  if (mine.group == kNoGroup && mine.length <= keys) {
    return;  // written by its workgroup
  }
  const uint32_t visible = mine.length - mine.count + (token - mine.start) + 1u;
  const uint32_t own = (visible - mine.first + keys - 1u) / keys;
  uint32_t shared = 0;
  if (mine.group != kNoGroup) {
    const uint32_t rows = work.items[mine.group].count * group;
    const uint32_t per = work.keys[rows <= decode_most ? 0 : 1];
    shared = (mine.first + per - 1u) / per;
  }
  const uint32_t parts = shared + own;
  const size_t plane = (size_t)a.batch.tokens * a.heads;
  float m = kLowestMax, l = 0.0f, x[kRegs] = {};
  for (uint32_t at = wave; at < parts; at += 4u * kParts) {
    float2 here[4];
    float part[4][kRegs];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t q = min(at + j * kParts, parts - 1u);
      const uint32_t kind = q < shared ? 1u : 0u;
      const size_t i = (q < shared ? q : q - shared) * plane + row;
      here[j] = *reinterpret_cast<const float2*>(&work.ml[kind][2 * i]);
#pragma unroll
      for (int r = 0; r < kRegs; ++r) {
        part[j][r] = work.o[kind][i * D + lane * kRegs + r];
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
      l = at + j * kParts < parts ? fmaf(w, here[j].y, l) : l;
#pragma unroll
      for (int r = 0; r < kRegs; ++r) {
        x[r] = at + j * kParts < parts ? fmaf(w, part[j][r], x[r]) : x[r];
      }
    }
  }
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
  store_output<T>(a, (size_t)row * D + threadIdx.x, value, inverse_sum(sum));
}

// What a call is cut by, and its workspace.
struct SharedPlan {
  SharedLimits limits;
  uint32_t decode_workgroups, tile_workgroups;  // none: the kernel has no items
  SharedWork work;
  SharedLists lists;
  size_t bytes;
};

// Whether reading shared keys once can make up for the launches that it takes: the bytes
// that the plain call would read again, in every block of 16 rows of the decode kernel, as
// far as the host's bounds say.  Measured even, plain and shared: without the tiled kernel 26
// MB (4 sequences of 4 rows, 8192 tokens of 1 KiB: 21.4 us and 21.6; 32768: 42.6 and 26.8), with
// it about 100 MB (64 sequences, 2048 tokens: 48.8 and 45.6, 512 tokens 21 and 41; 8 of 32
// rows, 2048 tokens: 29 and 48, 8192: 73 and 58).
//
// Not where the sequences' rows fill tiles of their own, at the mean: nothing is then read
// again that counts, and rows pass through memory once more for the join.  Plain and shared,
// f32, eight heads of 256 on two KV heads: 64 sequences of 10 tokens behind 8192 261 us and 155,
// of 32 (128 rows) behind 4096 160 and 221; 8 of 512 behind 16384 1052 and 1163; a chunk of 512
// beside 63 single tokens (36 rows at the mean) behind 16384 328 and 212, of 2048 (132) behind
// 8192 433 and 459, of 512 beside 15 (132) behind 8192 144 and 131.  Sixteen heads of 128 on
// eight: 16 sequences of 128 tokens behind 4096 165 and 232, 24 of 20 (40 rows) behind 8192 214
// and 119; 32 chunks of 64 beside as many single tokens (65) behind 8192 359 and 385.
bool worth_sharing(const PagedAttentionArgs& a, const SharedPrefixArgs& p) {
  const uint64_t group = a.heads / a.cache.kv_heads;
  const uint64_t own = a.batch.max_query * group, all = std::max(own, p.max_rows * group);
  const uint64_t rows =
    std::min((uint64_t)a.batch.tokens, (uint64_t)a.batch.sequences * a.batch.max_query) * group;
  if (rows >= (uint64_t)kTileRows * a.batch.sequences) {
    return false;
  }
  const uint64_t blocks = own <= kDecodeBlock || own > kDecodeRows ? 1u : 2u;
  const double again = (double)(a.batch.sequences - p.groups) *
                       (double)std::min(p.max_prefix, a.batch.max_keys) *
                       (double)(2u * (uint64_t)a.cache.kv_heads * a.cache.head_dim * blocks);
  return again > (all > kDecodeRows ? 100e6 : 26e6);
}

SharedPlan plan_of(const PagedAttentionArgs& a, const SharedPrefixArgs& p, int cu_count,
                   void* workspace) {
  SharedPlan s{};
  SharedLimits& l = s.limits;
  l.group = a.heads / a.cache.kv_heads;
  // Rows of a sequence and of a group, as far as the host knows.
  const uint64_t own = (uint64_t)a.batch.max_query * l.group;
  const uint64_t all = std::max<uint64_t>(own, (uint64_t)p.max_rows * l.group);
  // Blocks of eight rows where all items, or those of single sequences, have no more; else of
  // sixteen, of which two are still faster than a tile of 128.
  const bool eight = all <= 8u || (own <= 8u && all > kDecodeRows);
  l.decode_shift = eight ? 3u : 4u;
  l.decode_most = eight ? 8u : own <= kDecodeRows ? kDecodeRows : kDecodeBlock;
  l.decode_slots = 11u * (uint32_t)cu_count;
  l.decode_many = 4u * (uint32_t)cu_count;
  l.tile_slots = (a.cache.head_dim == 256u ? 1u : 2u) * (uint32_t)cu_count;
  const uint64_t rows = (uint64_t)a.batch.tokens * a.heads;
  const uint64_t row_bytes = rows * (a.cache.head_dim + 2u) * sizeof(float);
  const uint32_t planes = (uint32_t)std::min<uint64_t>(
    std::max<uint64_t>((uint64_t{256} << 20) / row_bytes, 1u), 128u);
  l.planes[0] = std::min(planes, (a.batch.max_keys + 127u) / 128u);
  l.planes[1] = std::min(planes, (std::min(p.max_prefix, a.batch.max_keys) + 127u) / 128u);
  const uint64_t items = (uint64_t)a.batch.sequences + p.groups;
  const uint64_t pairs = items * a.cache.kv_heads;
  s.decode_workgroups = (uint32_t)std::min<uint64_t>(
    pairs * (l.decode_most >> l.decode_shift) * ((a.batch.max_keys + 127u) / 128u),
    l.decode_slots + std::min<uint64_t>(pairs, l.decode_slots));
  s.tile_workgroups = all > l.decode_most ? 2u * l.tile_slots : 0u;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    void* here = workspace == nullptr ? nullptr : static_cast<char*>(workspace) + at;
    at += (bytes + 255u) & ~size_t{255};
    return here;
  };
  for (int i = 0; i < 2; ++i) {
    s.work.o[i] =
      static_cast<float*>(take(l.planes[i] * rows * a.cache.head_dim * sizeof(float)));
    s.work.ml[i] = static_cast<float*>(take(l.planes[i] * rows * 2u * sizeof(float)));
  }
  s.lists.items = static_cast<SharedItem*>(take(items * sizeof(SharedItem)));
  s.lists.ends = static_cast<uint32_t*>(take(2u * items * sizeof(uint32_t)));
  s.lists.keys = static_cast<uint32_t*>(take(2u * sizeof(uint32_t)));
  s.work.items = s.lists.items;
  s.work.ends = s.lists.ends;
  s.work.keys = s.lists.keys;
  s.work.count = (uint32_t)items;
  s.bytes = at;
  return s;
}

template <int D, class T>
void launch_join(const PagedAttentionArgs& a, const SharedPrefixArgs& p, const SharedPlan& s,
                 hipStream_t stream) {
  const uint32_t rows = a.batch.tokens * a.heads;
  // (Up to some seventy parts of a row.  128 rows: the call 53.7 us with four waves, 49.2 with
  // sixteen; 512 rows 100 and 101; 192 tokens of sixteen heads, a few parts a row, 55.8 and 68.)
  if (rows <= 256u) {
    shared_join_kernel<D, T, 16>
      <<<dim3(rows), 1024, 0, stream>>>(a, s.work, p.groups, s.limits.decode_most);
  } else {
    shared_join_kernel<D, T, 4>
      <<<dim3(rows), 256, 0, stream>>>(a, s.work, p.groups, s.limits.decode_most);
  }
}

template <class T>
void launch_join_type(const PagedAttentionArgs& a, const SharedPrefixArgs& p, const SharedPlan& s,
                      hipStream_t stream) {
  if (a.cache.head_dim == 256u) {
    launch_join<256, T>(a, p, s, stream);
  } else if (a.cache.head_dim == 128u) {
    launch_join<128, T>(a, p, s, stream);
  } else {
    launch_join<64, T>(a, p, s, stream);
  }
}

}  // namespace

size_t attention_shared_q8_workspace_bytes(const PagedAttentionArgs& a, const SharedPrefixArgs& p,
                                           int cu_count) {
  return worth_sharing(a, p) ? plan_of(a, p, cu_count, nullptr).bytes
                             : attention_paged_q8_workspace_bytes(a, cu_count);
}

hipError_t launch_attention_shared_q8(const PagedAttentionArgs& a, const SharedPrefixArgs& p,
                                      int cu_count, void* workspace, hipStream_t stream) {
  if (!worth_sharing(a, p)) {
    return launch_attention_paged_q8(a, cu_count, workspace, stream);
  }
  const SharedPlan s = plan_of(a, p, cu_count, workspace);
  shared_plan_kernel<<<dim3(1), kPlanThreads, 0, stream>>>(a, p, s.limits, s.lists);
  launch_shared_decode(a, s.work, 1u << s.limits.decode_shift, s.decode_workgroups, stream);
  if (s.tile_workgroups != 0u) {
    launch_shared_tiles(a, s.work, s.tile_workgroups, stream);
  }
  if (a.f16) {
    launch_join_type<half_t>(a, p, s, stream);
  } else {
    launch_join_type<float>(a, p, s, stream);
  }
  return hipGetLastError();
}

}  // namespace kraken
