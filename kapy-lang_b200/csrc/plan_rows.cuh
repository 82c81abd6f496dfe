// Row plan: a stable counting sort of n indices into groups.
//
//   order[p]   = the entry at position p (entries of group 0 first, each group's in
//                ascending order of entry), -1 behind the last planned position
//   offsets[g] = first position of group g; offsets[groups] = number of planned entries
//   slots[i]   = position of entry i, -1 when its index names no group
//
// One launch without scratch memory: a cluster of CTAs splits the entries, every
// warp counts a contiguous piece of them in its own row of a shared-memory table (the
// lanes of a step that name one group find each other by a ballot per bit of the group
// number, so nothing is atomic and the order is that of the entries; match.any does the
// same in one instruction that takes some 240 clocks), the CTAs read one another's totals through distributed
// shared memory, and each warp walks its piece again to place it.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"
#include "ptx_sm100.cuh"

namespace kapyb {

constexpr int kPlanWarps = 32;
constexpr int kPlanBatch = 8;  // index loads in flight per lane
constexpr int kPlanMaxGroups = 1024;  // and one more for the rows of no adapter
constexpr int kPlanMaxCtas = 16;

struct PlanParams {
  const int32_t *index;
  int n, groups;
  int32_t *order, *offsets, *slots;
  int capacity;  // entries of order: n, more when groups are padded
  int align;     // groups start at multiples of this (a power of two); the gaps are -1
  int rest;      // 1: an index outside 0 .. groups - 2 names the last group
};

// Counters of one warp, an odd number of words so that a column of the table (one group,
// all warps) is free of bank conflicts.
__host__ __device__ inline int plan_pitch(int groups) { return groups | 1; }

inline size_t plan_smem_bytes(int groups) {
  // per-warp counters, this CTA's totals, first positions
  return (static_cast<size_t>(kPlanWarps) * plan_pitch(groups) + 2 * groups) * sizeof(int32_t);
}

__global__ void __launch_bounds__(kPlanWarps * 32) plan_rows_kernel(const PlanParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ int32_t plan_smem[];
  __shared__ int scan_part[kPlanWarps];
  ptx::griddep_launch();  // the product that reads the plan sets up meanwhile, as this does here
  const int G = p.groups;
  const int pitch = plan_pitch(G);
  int32_t *count = plan_smem;                       // [kPlanWarps][pitch]
  int32_t *total = plan_smem + kPlanWarps * pitch;  // [G]
  int32_t *first = total + G;                       // [G]
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int ctas = static_cast<int>(cluster.num_blocks()), me = static_cast<int>(cluster.block_rank());
  const int pieces = ctas * kPlanWarps;
  const long long step = ((static_cast<long long>(p.n) + pieces - 1) / pieces + 31) / 32 * 32;
  const long long lo = min(static_cast<long long>(p.n), (me * kPlanWarps + w) * step);
  const long long hi = min(static_cast<long long>(p.n), lo + step);

  for (int i = threadIdx.x; i < kPlanWarps * pitch; i += blockDim.x) count[i] = 0;
  ptx::griddep_wait();
  __syncthreads();
  int32_t *mine = count + w * pitch;
  // walks this warp's piece, kPlanBatch steps of 32 entries at a time so that their loads
  // overlap; step(i, g): entry i of group g (-1: none)
  auto walk = [&](auto &&step) {
    for (long long i0 = lo; i0 < hi; i0 += 32 * kPlanBatch) {
      int g[kPlanBatch];
#pragma unroll
      for (int u = 0; u < kPlanBatch; ++u) {
        const long long i = i0 + 32 * u + lane;
        g[u] = i < hi ? p.index[i] : -1;
      }
#pragma unroll
      for (int u = 0; u < kPlanBatch; ++u)
        if (i0 + 32 * u < hi) {
          const bool out = g[u] < 0 || g[u] >= G;
          step(i0 + 32 * u + lane, !out ? g[u] : p.rest && i0 + 32 * u + lane < hi ? G - 1 : -1);
        }
    }
  };
  const int bits = 32 - __clz(G);  // of 0 .. G, G standing for "no group"
  auto lanes_like = [&](int g) {
    const uint32_t code = g < 0 ? G : g;
    uint32_t same = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
      const bool one = (code >> b) & 1u;
      const uint32_t ones = __ballot_sync(0xffffffffu, one);
      same &= one ? ones : ~ones;
    }
    return same;
  };
  walk([&](long long, int g) {
    const uint32_t same = lanes_like(g);
    if (g >= 0 && lane == __ffs(same) - 1) mine[g] += __popc(same);
    __syncwarp();
  });
  __syncthreads();
  // a group's counters over the CTA's warps -> their exclusive sums: one warp per group,
  // lane k holding warp k's
  static_assert(kPlanWarps == 32, "one lane per warp");
  for (int g = w; g < G; g += kPlanWarps) {
    const int c = count[lane * pitch + g];
    int run = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += o;
    }
    count[lane * pitch + g] = run - c;
    if (lane == 31) total[g] = run;
  }
  cluster.sync();
  // first position of every group: exclusive scan over the groups of the cluster's
  // totals, plus what the CTAs in front of this one hold of the group.  A thread
  // owns a run of adjacent groups.
  const int per = (G + blockDim.x - 1) / blockDim.x;
  const int g0 = min(G, static_cast<int>(threadIdx.x) * per), g1 = min(G, g0 + per);
  int sum = 0;
  int held[2];  // entries of this thread's groups (at most two: see kPlanMaxGroups)
  static_assert(kPlanMaxGroups + 1 <= 2 * kPlanWarps * 32, "two groups a thread");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int g = g0 + h;
    if (g >= g1) break;
    int all = 0, before = 0;
    for (int c = 0; c < ctas; ++c) {
      const int t = cluster.map_shared_rank(total, c)[g];
      if (c < me) before += t;
      all += t;
    }
    first[g] = sum + before;
    if (me == 0) p.offsets[g] = sum;  // completed below
    held[h] = all;
    sum += (all + p.align - 1) & ~(p.align - 1);
  }
  int scan = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, scan, off);
    if (lane >= off) scan += o;
  }
  if (lane == 31) scan_part[w] = scan;
  __syncthreads();
  int base = scan - sum, planned = 0;
  for (int k = 0; k < kPlanWarps; ++k) {
    if (k < w) base += scan_part[k];
    planned += scan_part[k];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int g = g0 + h;
    if (g >= g1) break;
    first[g] += base;
    if (me == 0) {
      const int at = p.offsets[g] + base;
      p.offsets[g] = at;
      const int end = at + ((held[h] + p.align - 1) & ~(p.align - 1));
      for (int q = at + held[h]; q < end; ++q) p.order[q] = -1;
    }
  }
  if (me == 0 && threadIdx.x == 0) p.offsets[G] = planned;
  // the others' totals have been read: nobody leaves while they still may be
  cluster.sync();
  walk([&](long long i, int g) {
    const uint32_t same = lanes_like(g);
    int pos = -1;
    if (g >= 0) pos = first[g] + mine[g] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (g >= 0 && lane == __ffs(same) - 1) mine[g] += __popc(same);
    __syncwarp();
    if (i < hi) {
      if (pos >= 0) p.order[pos] = static_cast<int32_t>(i);
      if (p.slots) p.slots[i] = pos;
    }
  });
  for (long long q = planned + static_cast<long long>(me) * blockDim.x + threadIdx.x; q < p.capacity;
       q += static_cast<long long>(ctas) * blockDim.x)
    p.order[q] = -1;
}

}  // namespace kapyb
