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
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention_paged_q8_common.hpp"
#include "context_internal.hpp"
#include "device_common.hpp"
#include "row_order.hpp"

namespace kraken {
namespace {

constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kPlanWaves = kPlanThreads / 64u;
constexpr uint32_t kHeldItems = 1024;  // listed in LDS on the way to memory

// What the host gives the plan.
struct SharedLimits {
  uint32_t group;         // query heads of a KV head
  uint32_t decode_most;   // rows up to which an item goes to the decode kernel
  uint32_t decode_rows;   // of a block of it
  uint32_t decode_slots;  // workgroups that its work is cut into
  uint32_t tile_slots;    // workgroups of the tiled kernel that run at once
  uint32_t planes[2];     // parts that there is room for, of sequences and of groups
};

struct SharedLists {
  SharedItem* items;
  uint32_t* ends;
  uint32_t* keys;
};

__device__ __forceinline__ uint32_t rows_of(const SharedLimits& l, const SharedItem& i) {
  return i.count * l.group;
}

// Workgroups (by KV head) of an item in `keys` keys each, of the kernel `kind`.
__device__ __forceinline__ uint32_t work_of(const SharedLimits& l, const SharedItem& i,
                                            uint32_t kind, uint32_t keys) {
  const uint32_t rows = rows_of(l, i);
  if (rows == 0 || (rows <= l.decode_most) != (kind == 0)) {
    return 0u;
  }
  const uint32_t across = kind == 0 ? l.decode_rows : kTileRows;
  return (rows + across - 1u) / across * ((i.length - i.first + keys - 1u) / keys);
}

// One workgroup.
__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(PagedAttentionArgs a,
                                                                   SharedPrefixArgs p,
                                                                   SharedLimits l,
                                                                   SharedLists lists) {
  __shared__ SharedItem held[kHeldItems];
  __shared__ uint64_t sums[kPlanWaves][2];
  __shared__ uint32_t most[kPlanWaves][4], scans[kPlanWaves], choice[kPlanWaves];
  __shared__ float times[kPlanWaves];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t sequences = a.batch.sequences, shift = a.cache.page_shift;
  const uint32_t kv_heads = a.cache.kv_heads, count = p.groups + sequences;
  SharedItem* const items = count <= kHeldItems ? held : lists.items;

  for (uint32_t i = tid; i < count; i += kPlanThreads) {
    SharedItem item{0u, 0u, 0u, 0u, 0u, kIsGroup};
    if (i >= p.groups) {
      const PagedSequence q = paged_sequence(a.batch, i - p.groups, shift);
      item = {q.start, q.count, q.length, i - p.groups, 0u, kNoGroup};
    }
    items[i] = item;
  }
  __syncthreads();

  // A wave a group.
  for (uint32_t g = wave; g < p.groups; g += kPlanWaves) {
    const uint32_t begin = p.starts[g], end = p.starts[g + 1], prefix = p.lengths[g];
    if (begin >= end || end > sequences || prefix > p.max_prefix) {
      continue;
    }
    const uint32_t row = a.batch.starts[begin], stop = a.batch.starts[end];
    if (row >= stop || stop > a.batch.tokens || stop - row > p.max_rows) {
      continue;
    }
    // Its sequences with rows: how many, the first, and the fewest tokens before the new
    // ones; whether all their rows lie in the group's.
    uint32_t least = prefix, first = end, live = 0;
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
    for (int step = 1; step < 64; step *= 2) {
      least = min(least, (uint32_t)__shfl_xor((int)least, step));
      first = min(first, (uint32_t)__shfl_xor((int)first, step));
      live += (uint32_t)__shfl_xor((int)live, step);
    }
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
  uint64_t all[2] = {0, 0};
  uint32_t longest[4] = {0, 0, 0, 0};
  for (uint32_t i = tid; i < count; i += kPlanThreads) {
    const SharedItem q = items[i];
    const uint32_t rows = rows_of(l, q), keys = q.length - q.first;
    const uint32_t kind = rows <= l.decode_most ? 0u : 1u;
    const uint32_t across = kind == 0 ? l.decode_rows : kTileRows;
    const uint32_t at = 2u * kind + (i < p.groups ? 1u : 0u);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      longest[k] = at == k && rows != 0 ? max(longest[k], keys) : longest[k];
    }
    const uint64_t work = (uint64_t)((rows + across - 1u) / across) * keys;
    all[0] += kind == 0 ? work : 0u;
    all[1] += kind == 1 ? work : 0u;
  }
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    longest[k] = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(longest[k], Largest{}), 63);
  }
  all[0] = last_lane(wave_scan(all[0], Sum{}));
  all[1] = last_lane(wave_scan(all[1], Sum{}));
  if (lane == 0) {
    sums[wave][0] = all[0];
    sums[wave][1] = all[1];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      most[wave][k] = longest[k];
    }
  }
  __syncthreads();
  all[0] = all[1] = 0;
  uint32_t need[2] = {0, 0};  // keys of a part, so that the parts have room
  for (uint32_t w = 0; w < kPlanWaves; ++w) {
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
      all[k] += sums[w][k];
      need[k] = max(need[k], (most[w][2 * k] + l.planes[0] - 1u) / l.planes[0]);
      need[k] = max(need[k], (most[w][2 * k + 1] + l.planes[1] - 1u) / l.planes[1]);
    }
  }
  // The decode kernel's: as many workgroups as its slots, of 128 to 4096 keys.
  uint64_t keys = (all[0] * kv_heads + l.decode_slots - 1u) / l.decode_slots;
  keys = min(max(keys, (uint64_t)128u), (uint64_t)4096u);
  const uint32_t decode_keys = (uint32_t)((max(keys, (uint64_t)need[0]) + 127u) / 128u * 128u);
  // The tiled kernel's: of sixteen sizes the one whose rounds of `tile_slots` workgroups are
  // soonest over, each round taking its keys and what a workgroup spends besides (about 128
  // keys' time).  Each wave tries one: those that make one round, two .. eight if all parts
  // were full, and an eighth more.
  {
    const uint64_t rounds = (uint64_t)l.tile_slots * (1u + wave / 2u);
    keys = (all[1] * kv_heads + rounds - 1u) / rounds;
    keys += wave % 2u != 0u ? keys / 8u : 0u;
    keys = max(min(max(keys, (uint64_t)128u), (uint64_t)0x3fffffc0u), (uint64_t)need[1]);
    const uint32_t mine = (uint32_t)((keys + 63u) / 64u * 64u);
    float total = 0.0f;
    for (uint32_t i = lane; i < count; i += 64u) {
      total += (float)work_of(l, items[i], 1u, mine);
    }
    total = wave_sum(total) * (float)kv_heads;
    if (lane == 0) {
      choice[wave] = mine;
      times[wave] = ceilf(total / (float)l.tile_slots) * ((float)mine + 128.0f);
    }
  }
  __syncthreads();
  uint32_t best = 0;
  for (uint32_t w = 1; w < kPlanWaves; ++w) {
    best = times[w] < times[best] ? w : best;
  }
  const uint32_t part_keys[2] = {decode_keys, choice[best]};
  if (tid < 2u) {
    lists.keys[tid] = part_keys[tid];
  }
  // The workgroups up to each item.
#pragma unroll
  for (uint32_t kind = 0; kind < 2; ++kind) {
    uint32_t before = 0;
    for (uint32_t base = 0; base < count; base += kPlanThreads) {
      const uint32_t i = base + tid;
      const uint32_t mine = i < count ? work_of(l, items[i], kind, part_keys[kind]) : 0u;
      uint32_t upto = wave_scan(mine, Sum{});
      __syncthreads();
      if (lane == 63u) {
        scans[wave] = upto;
      }
      __syncthreads();
      upto += before;
      for (uint32_t w = 0; w < kPlanWaves; ++w) {
        upto += w < wave ? scans[w] : 0u;
        before += scans[w];
      }
      if (i < count) {
        lists.ends[(size_t)kind * count + i] = upto;
      }
    }
  }
  if (items == held && tid < count) {
    lists.items[tid] = held[tid];
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
  l.decode_rows = all <= 8u || (own <= 8u && all > kDecodeRows) ? 8u : 16u;
  l.decode_most = l.decode_rows == 8u ? 8u
                  : all <= kDecodeRows || own <= kDecodeRows ? kDecodeRows : kDecodeBlock;
  l.decode_slots = 11u * (uint32_t)cu_count;
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
    pairs * (l.decode_most / l.decode_rows) * ((a.batch.max_keys + 127u) / 128u),
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
  if (rows <= 1024u) {
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
  return plan_of(a, p, cu_count, nullptr).bytes;
}

hipError_t launch_attention_shared_q8(const PagedAttentionArgs& a, const SharedPrefixArgs& p,
                                      int cu_count, void* workspace, hipStream_t stream) {
  const SharedPlan s = plan_of(a, p, cu_count, workspace);
  shared_plan_kernel<<<dim3(1), kPlanThreads, 0, stream>>>(a, p, s.limits, s.lists);
  launch_shared_decode(a, s.work, s.limits.decode_rows, s.decode_workgroups, stream);
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
