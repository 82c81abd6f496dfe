// A shared projection with low-rank adapters beside it, for few rows (a decode step of up
// to 256 sequences):
//   out[t] = act(alpha x[t] . W + bias + low[t] . up[i(t)]),   low[t] = scale[i] x[t] . down[i]
//
// What such a call costs is reading W once, so the kernel is a weight stream: 128 columns
// of W fill the M side of the MMA, the at most 256 rows of x its N side, and a cluster of
// CTAs shares a column block by cutting K into pieces, so that every SM streams even when
// there are few column blocks.  The CTAs' partial sums meet in distributed shared memory,
// each CTA finishing its share of the rows, added in CTA order: no scratch in global
// memory, no atomics, the same bits on every run.
//
// The adapters' part has too few operations for a tensor core (every row may name another
// adapter) and too many bytes to come last: the warps that will drain the accumulator
// compute it, rows dealt out to warps, while the weights stream, and keep it in shared
// memory in f32.  low comes from a small kernel launched just before; this one is
// launched with programmatic serialization, starts on the weights at once and waits for
// low only where it is read.  (The kernel before the small one is complete when that one
// starts, so everything else the call reads may be read without waiting.)
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "grouped_sm100.cuh"
#include "ptx_sm100.cuh"

namespace kapyb {

__device__ __forceinline__ int round16(int v) { return (v + 15) & ~15; }

constexpr int kDecodeMaxRows = 256;
constexpr int kLowThreads = 512;
constexpr int kLowMaxSplit = 4;

struct LowParams {
  const uint16_t *x;
  long long x_s0;            // unit stride on K
  const uint16_t *down;
  long long d_s0, d_s1, d_group;
  int bf16, groups, rows, K, rank;
  const int32_t *index;
  const float *scale;
  float *low;                // [rows, rank]
  int split;                 // CTAs of a cluster that share a row's K
};

__device__ __forceinline__ float ld_shared_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <bool BF>
__device__ __forceinline__ float widen16(uint16_t h) {
  return cvt_16_to_f32(h, BF ? KAPYB_BF16 : KAPYB_F16);
}

// low[t]: a cluster of `split` blocks per row, each a run of K; the first one adds up.
// KMAJOR: down has its unit stride on K, a warp per column of it; otherwise unit stride on
// the rank, a thread per eight columns and K residue.  Sums in f32 in a fixed order.  Rows
// of down and x start on 16 bytes and rank is a multiple of 8 (!KMAJOR).
template <bool BF, bool KMAJOR>
__global__ void __launch_bounds__(kLowThreads) adapter_low_kernel(const LowParams p) {
  ptx::griddep_launch();
  constexpr int DT = BF ? KAPYB_BF16 : KAPYB_F16;
  __shared__ float part[kLowThreads / 32][128];
  __shared__ float mine[128];
  const long long t = blockIdx.x / p.split;
  const int rank = blockIdx.x % p.split;
  const int i = p.index[t];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (i < 0 || i >= p.groups) {  // the whole cluster
    if (rank == 0)
      for (int j = threadIdx.x; j < p.rank; j += kLowThreads) p.low[t * p.rank + j] = 0.0f;
    return;
  }
  const float scale = p.scale ? p.scale[i] : 1.0f;
  const uint16_t *x = p.x + t * p.x_s0;
  const uint16_t *down = p.down + i * p.d_group;
  // this block's run of K, in whole 16-byte pieces but for the last one's end
  const int pieces = (p.K + 7) / 8;
  const int first_k = static_cast<int>(static_cast<long long>(rank) * pieces / p.split) * 8;
  const int last_k = min(p.K, static_cast<int>(static_cast<long long>(rank + 1) * pieces / p.split) * 8);
  if constexpr (KMAJOR) {
    for (int j = w; j < p.rank; j += kLowThreads / 32) {
      const uint16_t *col = down + j * p.d_s1;
      float acc = 0.0f;
      const int whole = last_k / 8;
      constexpr int U = 4;
      for (int v = first_k / 8 + lane; v < whole; v += 32 * U) {
        uint4 a[U], b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          a[u] = b[u] = make_uint4(0u, 0u, 0u, 0u);
          if (v + 32 * u < whole) {
            a[u] = __ldg(reinterpret_cast<const uint4 *>(col) + v + 32 * u);
            b[u] = __ldg(reinterpret_cast<const uint4 *>(x) + v + 32 * u);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t as[4] = {a[u].x, a[u].y, a[u].z, a[u].w}, bs[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a0, a1, b0, b1;
            unpack2_16<DT>(as[e], a0, a1);
            unpack2_16<DT>(bs[e], b0, b1);
            acc = fmaf(a1, b1, fmaf(a0, b0, acc));
          }
        }
      }
      for (int k = max(first_k, whole * 8) + lane; k < last_k; k += 32)
        acc = fmaf(widen16<BF>(x[k]), widen16<BF>(col[k]), acc);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
      if (lane == 0) mine[j] = acc;
    }
  } else {
    const int chunks = p.rank / 8;
    int wide = 1;  // threads side by side on one K: chunks rounded up to a power of two
    while (wide < chunks) wide *= 2;
    const int chunk = threadIdx.x & (wide - 1), k0 = threadIdx.x / wide, step = kLowThreads / wide;
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    if (chunk < chunks) {
      constexpr int U = 8;
      for (int k = first_k + k0; k < last_k; k += step * U) {
        uint4 a[U];
        float xv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          a[u] = make_uint4(0u, 0u, 0u, 0u);
          xv[u] = 0.0f;
          if (k + step * u < last_k) {
            a[u] = __ldg(reinterpret_cast<const uint4 *>(down + (k + step * u) * p.d_s0) + chunk);
            xv[u] = widen16<BF>(__ldg(x + k + step * u));
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t as[4] = {a[u].x, a[u].y, a[u].z, a[u].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float lo, hi;
            unpack2_16<DT>(as[e], lo, hi);
            acc[2 * e] = fmaf(xv[u], lo, acc[2 * e]);
            acc[2 * e + 1] = fmaf(xv[u], hi, acc[2 * e + 1]);
          }
        }
      }
    }
    for (int off = wide; off < 32; off <<= 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], off);
    }
    if (lane < wide && chunk < chunks) {
#pragma unroll
      for (int e = 0; e < 8; ++e) part[w][chunk * 8 + e] = acc[e];
    }
    __syncthreads();
    // a warp holds every chunk as long as a K row's threads fit one (wide <= 16 always)
    for (int j = threadIdx.x; j < p.rank; j += kLowThreads) {
      float s = 0.0f;
      for (int k = 0; k < kLowThreads / 32; ++k) s += part[k][j];
      mine[j] = s;
    }
  }
  __syncthreads();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (rank == 0) {
    for (int j = threadIdx.x; j < p.rank; j += kLowThreads) {
      float s = 0.0f;
      for (int c = 0; c < p.split; ++c) s += ld_shared_cluster(ptx::mapa(ptx::smem_u32(&mine[j]), c));
      p.low[t * p.rank + j] = s * scale;
    }
  }
  ptx::cluster_arrive();  // nobody leaves while the first one may read
  ptx::cluster_wait();
}

struct DecodeParams {
  int rows, wide;        // rows of x; rounded up to 16
  int cols, num_kb;
  int stages, stage_bytes;
  int w_mn_major, bf16;
  uint32_t tmem_cols;
  const float *low;
  const int32_t *index;
  int groups, rank;
  const uint16_t *up;
  long long u_s0, u_s1, u_group;
  int up_form;           // 1: unit stride on the columns, 2: on the rank, both with aligned 16-byte pieces; 0: any
  void *out;
  long long out_s0, out_s1;
  int out_dtype;
  float alpha;
  const void *bias;
  int bias_dtype, bias_axis, activation, rounding;
  uint32_t *status;
  uint32_t wait_limit_us;
};

// low[t] . up[a] for columns n0 .. n0 + 127 into dst[128]; one warp.
template <bool BF>
__device__ __forceinline__ void adapter_delta(const DecodeParams &p, int t, int a, int n0, float *dst, int lane) {
  constexpr int DT = BF ? KAPYB_BF16 : KAPYB_F16;
  const bool on = a >= 0 && a < p.groups;
  const float *low = p.low + static_cast<long long>(t) * p.rank;
  const uint16_t *up = p.up + (on ? a * p.u_group : 0ll);
  if (!on) {
    reinterpret_cast<float4 *>(dst)[lane] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return;
  }
  if (p.up_form == 1) {
    // lane: eight columns, every other j; the two halves of the warp meet at the end
    const int c = (lane & 15) * 8, n = n0 + c;
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    constexpr int U = 8;
    for (int j = lane >> 4; j < p.rank; j += 2 * U) {
      uint4 q[U];
      float l[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        q[u] = make_uint4(0u, 0u, 0u, 0u);
        l[u] = 0.0f;
        if (j + 2 * u < p.rank && n < p.cols) {  // cols is a multiple of 8
          q[u] = __ldg(reinterpret_cast<const uint4 *>(up + (j + 2 * u) * p.u_s0 + n));
          l[u] = low[j + 2 * u];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t qs[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float lo, hi;
          unpack2_16<DT>(qs[e], lo, hi);
          acc[2 * e] = fmaf(l[u], lo, acc[2 * e]);
          acc[2 * e + 1] = fmaf(l[u], hi, acc[2 * e + 1]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 16);
    if (lane < 16) {
      reinterpret_cast<float4 *>(dst + c)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      reinterpret_cast<float4 *>(dst + c)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
  } else {
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.up_form == 2) {
      for (int j = 0; j < p.rank; j += 8) {  // rank is a multiple of 8
        uint4 q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int n = n0 + u * 32 + lane;
          q[u] = make_uint4(0u, 0u, 0u, 0u);
          if (n < p.cols) q[u] = __ldg(reinterpret_cast<const uint4 *>(up + n * p.u_s1 + j));
        }
        float l[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) l[e] = low[j + e];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t qs[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float lo, hi;
            unpack2_16<DT>(qs[e], lo, hi);
            acc[u] = fmaf(l[2 * e + 1], hi, fmaf(l[2 * e], lo, acc[u]));
          }
        }
      }
    } else {
      for (int j = 0; j < p.rank; ++j) {
        const float l = low[j];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int n = n0 + u * 32 + lane;
          if (n < p.cols) acc[u] = fmaf(l, widen16<BF>(up[j * p.u_s0 + n * p.u_s1]), acc[u]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) dst[u * 32 + lane] = acc[u];
  }
}

// One block of 128 columns per cluster, the cluster's CTAs sharing K.  tmW: W in boxes of
// 64 x 128 (K-major) or 64 x 64 (MN-major), 3-D with one group; tmX: x in boxes of
// 64 x wide.
template <bool BF>
__global__ void __launch_bounds__(192) adapter_decode_kernel(const __grid_constant__ CUtensorMap tmW,
                                                             const __grid_constant__ CUtensorMap tmX,
                                                             const DecodeParams p) {
  constexpr int kMaxStages = 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], done_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_words[2];
  volatile uint32_t *abort_flag = abort_words;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int split = static_cast<int>(gridDim.x) / ((p.cols + 127) / 128);  // CTAs of a cluster
  const int rank = static_cast<int>(blockIdx.x) % split;
  const int n0 = static_cast<int>(blockIdx.x) / split * 128;
  const int kb0 = static_cast<int>(static_cast<long long>(rank) * p.num_kb / split);
  const int kb1 = static_cast<int>(static_cast<long long>(rank + 1) * p.num_kb / split);
  // rows this CTA finishes
  const int r0 = rank * p.rows / split, r1 = (rank + 1) * p.rows / split;
  float *delta = reinterpret_cast<float *>(smem + p.stages * p.stage_bytes);  // [r1 - r0][128]
  float *partial = reinterpret_cast<float *>(smem);                           // [wide][128], over the ring

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(&done_bar), 1);
    abort_flag[0] = 0u;
    abort_flag[1] = p.wait_limit_us;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&tmW);
    ptx::prefetch_tensormap(&tmX);
  }
  if (warp == 1) {
    ptx::tmem_alloc<1>(ptx::smem_u32(&tmem_slot), p.tmem_cols);
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t x_off = 16384u;  // the rows of x behind the weights in a stage

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t once = ptx::make_l2_policy(1);  // the weights are read once
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!ptx::mbar_wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1u, abort_flag)) break;
        const uint32_t fb = ptx::smem_u32(&full_bar[stage]);
        const uint32_t dst = ptx::smem_u32(smem + stage * p.stage_bytes);
        ptx::mbar_arrive_expect_tx(fb, 16384u + static_cast<uint32_t>(p.wide) * 128u);
        if (p.w_mn_major) {
          ptx::tma_load_3d_hint(dst, &tmW, fb, n0, kb * 64, 0, once);
          ptx::tma_load_3d_hint(dst + 8192, &tmW, fb, n0 + 64, kb * 64, 0, once);
        } else {
          ptx::tma_load_3d_hint(dst, &tmW, fb, kb * 64, n0, 0, once);
        }
        tma_load_2d(dst + x_off, &tmX, fb, kb * 64, 0);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = ptx::make_idesc_f16(p.bf16, p.w_mn_major, 0, 128, p.wide);
    const uint32_t a_lo_c = ((p.w_mn_major ? 8192u : 16u) >> 4) << 16;
    const uint32_t a_step = (p.w_mn_major ? 2048u : 32u) >> 4;
    constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&full_bar[stage]), phase, abort_flag))) {
        ok = false;
        break;
      }
      ptx::tc_fence_after();
      if (ptx::elect_one()) {
        // descriptors take the offset inside the CTA's own memory; in a cluster the address
        // carries the CTA's rank above it
        const uint32_t at = ptx::smem_u32(smem + stage * p.stage_bytes) & 0x3ffffu;
        const uint32_t a_lo = a_lo_c | (at >> 4), b_lo = (1u << 16) | ((at + x_off) >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          ptx::umma_k<1, 0>(tmem, (static_cast<uint64_t>(hi) << 32) | (a_lo + k * a_step),
                            (static_cast<uint64_t>(hi) << 32) | (b_lo + k * 2u), idesc, (kb != kb0 || k != 0) ? 1u : 0u);
        ptx::umma_commit<1>(ptx::smem_u32(&empty_bar[stage]));
      }
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (ok && kb1 > kb0 && ptx::elect_one()) ptx::umma_commit<1>(ptx::smem_u32(&done_bar));
  } else {
    ptx::griddep_wait();  // low
    const int q = warp & 3;
    // row r of this CTA's belongs to warp r % 4; lane l looks up its l-th one's adapter
    for (int base = r0 + q; base < r1; base += 4 * 32) {
      const int look = base + 4 * lane < r1 ? p.index[base + 4 * lane] : -1;
#pragma unroll 2
      for (int i = 0; i < 32; ++i) {
        const int r = base + 4 * i;
        if (r >= r1) break;
        adapter_delta<BF>(p, r, __shfl_sync(0xffffffffu, look, i), n0, delta + (r - r0) * 128, lane);
      }
    }
    // (a K shorter than the cluster leaves some of its CTAs without a block)
    const bool some = kb1 > kb0;
    const bool ok = !some || __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&done_bar), 0u, abort_flag));
    ptx::tc_fence_after();
    if (!some) {
      for (int c = 0; c < p.rows; ++c) partial[c * 128 + q * 32 + lane] = 0.0f;
    } else if (ok) {
      // every MMA is done, so every stage has been read: the ring takes the partial sums
      const uint32_t src = tmem + (static_cast<uint32_t>(q * 32) << 16);
      for (int c = 0; c < p.rows; c += 16) {
        uint32_t v[16];
        ptx::tmem_ld_32x16(src + c, v);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) partial[(c + i) * 128 + q * 32 + lane] = __uint_as_float(v[i]);
      }
      ptx::tc_fence_before();
    }
  }
  __syncthreads();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (warp >= 2 && *abort_flag == 0u) {
    const int q = warp & 3;
    const int n = n0 + q * 32 + lane;
    if (n < p.cols) {
      const float bias_col = p.bias != nullptr && p.bias_axis == 1 ? load_as_f32(p.bias, p.bias_dtype, n) : 0.0f;
      constexpr int U = 8;  // rows whose remote loads overlap
      for (int r = r0; r < r1; r += U) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = 0.0f;
        for (int c = 0; c < split; ++c) {
          const uint32_t at = ptx::mapa(ptx::smem_u32(partial + r * 128 + q * 32 + lane), c);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (r + u < r1) v[u] += ld_shared_cluster(at + u * 512u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r + u >= r1) break;
          float o = v[u] * p.alpha + bias_col;
          if (p.bias != nullptr && p.bias_axis == 0) o += load_as_f32(p.bias, p.bias_dtype, r + u);
          o += delta[(r + u - r0) * 128 + q * 32 + lane];
          store_from_f32(p.out, p.out_dtype, (r + u) * p.out_s0 + n * p.out_s1, apply_activation(p.activation, o),
                         p.rounding);
        }
      }
    }
  }
  __syncthreads();
  if (*abort_flag != 0u) {
    if (threadIdx.x == 0) atomicExch(p.status, kStatusTimeout);
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 200000ull) {
    }
  }
  // the other CTAs may still read this one's partial sums
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, p.tmem_cols);
  }
}

// ---------------------------------------------------------------- many rows
//
// low[p] = scale[g] x[row(p)] . down[g] for the positions of a padded plan, as two 16-bit
// halves (the value rounded, and what that left, so that the pair kernel's product with
// `up` is exact to 16 bits and more).  A tile is up to 64 positions of one adapter: the
// rank fills the M side of the MMA (lanes beyond it hold what the stage happened to hold
// and are not stored), the positions its N side.  There are few tiles and K is long, so a
// cluster shares K as in the kernel above.  Rows are gathered by cp.async (see
// grouped_sm100.cuh); down comes by TMA.

struct LowTileParams {
  const int32_t *offsets, *order;  // the padded plan; groups of `groups` adapters
  int groups, positions;
  const uint8_t *x;
  long long x_pitch;     // bytes
  int src_rows, K, rank, split;
  int d_mn_major, bf16;
  int a_bytes;           // of down in a stage: 8192 up to rank 64, else 16384
  const float *scale;
  float alpha;           // 1 / what rows with an adapter are multiplied by at the end
  uint16_t *high, *low;  // [positions][pitch]
  int pitch;
  uint32_t *status;
  uint32_t wait_limit_us;
};

constexpr int kLowTile = 64, kLowStages = 4;
constexpr int kLowTileThreads = 224;
constexpr int kLowStageBytes = 16384 + kLowTile * 128;
constexpr int kLowTileSmem = 1024 + kLowStages * kLowStageBytes + (3 * kGroupedMaxGroups + 8) * 4;

// tmD: down, 3-D, in boxes of 64 x 64 (unit stride on the rank, or rank <= 64) or 64 x 128.
template <bool BF>
__global__ void __launch_bounds__(kLowTileThreads) adapter_low_tile_kernel(const __grid_constant__ CUtensorMap tmD,
                                                                           const LowTileParams p) {
  ptx::griddep_launch();
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full_bar[kLowStages], empty_bar[kLowStages], rows_bar[kLowStages], done_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_words[2];
  volatile uint32_t *abort_flag = abort_words;
  int *table_mem = reinterpret_cast<int *>(smem + kLowStages * kLowStageBytes);
  GroupedTable table{table_mem, table_mem + kGroupedMaxGroups + 2, table_mem + 2 * kGroupedMaxGroups + 4};
  float *partial = reinterpret_cast<float *>(smem);  // [kLowTile][128], over the ring
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.split;  // in the cluster
  const int want = static_cast<int>(blockIdx.x) / p.split;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kLowStages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 2);  // down's bytes, the rows
      ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&rows_bar[s]), 128);
    }
    ptx::mbar_init(ptx::smem_u32(&done_bar), 1);
    abort_flag[0] = 0u;
    abort_flag[1] = p.wait_limit_us;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&tmD);
  }
  if (warp == 1) {
    ptx::tmem_alloc<1>(ptx::smem_u32(&tmem_slot), 64);
    ptx::tmem_relinquish<1>();
  }
  if (warp == 0) build_tile_table(p.offsets, p.groups, p.positions, kLowTile, table, lane);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // this cluster's tile; clusters behind the last one only keep the barriers company
  const bool mine = want < table.first[p.groups];
  const int g = find_group(table, p.groups, want);
  const int at = (want - table.first[g]) * kLowTile;
  const int p0 = table.begin[g] + at, rows = mine ? min(kLowTile, table.count[g] - at) : 0;
  const int num_kb = (p.K + 63) / 64;
  const int kb0 = mine ? static_cast<int>(static_cast<long long>(rank) * num_kb / p.split) : 0;
  const int kb1 = mine ? static_cast<int>(static_cast<long long>(rank + 1) * num_kb / p.split) : 0;
  const int wide = round16(rows);

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!ptx::mbar_wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1u, abort_flag)) break;
        const uint32_t fb = ptx::smem_u32(&full_bar[stage]);
        const uint32_t dst = ptx::smem_u32(smem) + stage * kLowStageBytes;
        ptx::mbar_arrive_expect_tx(fb, p.a_bytes);
        if (p.d_mn_major) {
          ptx::tma_load_3d(dst, &tmD, fb, 0, kb * 64, g);
          if (p.a_bytes > 8192) ptx::tma_load_3d(dst + 8192, &tmD, fb, 64, kb * 64, g);
        } else {
          ptx::tma_load_3d(dst, &tmD, fb, kb * 64, 0, g);
        }
        if (++stage == kLowStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = ptx::make_idesc_f16(p.bf16, p.d_mn_major, 0, 128, mine ? wide : 16);
    const uint32_t a_lo_c = ((p.d_mn_major ? 8192u : 16u) >> 4) << 16;
    const uint32_t a_step = (p.d_mn_major ? 2048u : 32u) >> 4;
    constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&full_bar[stage]), phase, abort_flag))) {
        ok = false;
        break;
      }
      ptx::tc_fence_after();
      if (ptx::elect_one()) {
        const uint32_t base = (ptx::smem_u32(smem) + stage * kLowStageBytes) & 0x3ffffu;  // see adapter_decode_kernel
        const uint32_t a_lo = a_lo_c | (base >> 4), b_lo = (1u << 16) | ((base + 16384u) >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          ptx::umma_k<1, 0>(tmem, (static_cast<uint64_t>(hi) << 32) | (a_lo + k * a_step),
                            (static_cast<uint64_t>(hi) << 32) | (b_lo + k * 2u), idesc, (kb != kb0 || k != 0) ? 1u : 0u);
        ptx::umma_commit<1>(ptx::smem_u32(&empty_bar[stage]));
      }
      if (++stage == kLowStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (ok && mine && ptx::elect_one()) ptx::umma_commit<1>(ptx::smem_u32(&done_bar));
  } else if (warp == 6) {
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&rows_bar[stage]), phase, abort_flag))) break;
      ptx::fence_proxy_async_smem();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&full_bar[stage]));
      if (++stage == kLowStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  } else {
    const int tid = threadIdx.x - 64, piece = tid & 7, row0 = tid >> 3;  // 16 rows a pass
    const uint8_t *row[kLowTile / 16];
#pragma unroll
    for (int i = 0; i < kLowTile / 16; ++i) {
      row[i] = nullptr;
      if (row0 + 16 * i < rows) {
        const long long from = source_row(p.order, 1, p.src_rows, p0 + row0 + 16 * i);
        if (from >= 0) row[i] = p.x + from * p.x_pitch;
      }
    }
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1u, abort_flag))) {
        ok = false;
        break;
      }
      const int k = kb * 64 + piece * 8;
      const uint32_t bytes = static_cast<uint32_t>(max(0, min(16, (p.K - k) * 2)));
      const uint32_t dst =
          ptx::smem_u32(smem) + stage * kLowStageBytes + 16384u + row0 * 128 + ((piece ^ (row0 & 7)) << 4);
      const long long off = bytes ? k * 2ll : 0ll;
#pragma unroll
      for (int i = 0; i < kLowTile / 16; ++i)
        if (row0 + 16 * i < wide) cp_async16(dst + i * 2048, row[i] ? row[i] + off : p.x, row[i] ? bytes : 0u);
      cp_async_arrive(ptx::smem_u32(&rows_bar[stage]));
      if (++stage == kLowStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    cp_async_wait_all();
    if (mine) ok = ok && ptx::mbar_wait(ptx::smem_u32(&done_bar), 0u, abort_flag);
    ok = __all_sync(0xffffffffu, ok) != 0;
    ptx::tc_fence_after();
    if (ok && mine) {
      const int q = warp & 3;
      for (int c = 0; c < rows; c += 16) {
        uint32_t v[16];
        ptx::tmem_ld_32x16(tmem + (static_cast<uint32_t>(q * 32) << 16) + c, v);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) partial[(c + i) * 128 + q * 32 + lane] = __uint_as_float(v[i]);
      }
      ptx::tc_fence_before();
    }
  }
  __syncthreads();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (mine && warp >= 2 && warp < 6 && *abort_flag == 0u) {
    const int j = (warp & 3) * 32 + lane;
    const int r0 = rank * rows / p.split, r1 = (rank + 1) * rows / p.split;
    if (j < p.rank) {
      const float alpha = p.alpha * (p.scale ? p.scale[g] : 1.0f);
      constexpr int DT = BF ? KAPYB_BF16 : KAPYB_F16;
      constexpr int U = 8;
      for (int r = r0; r < r1; r += U) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = 0.0f;
        for (int c = 0; c < p.split; ++c) {
          const uint32_t from = ptx::mapa(ptx::smem_u32(partial + r * 128 + j), c);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (r + u < r1) v[u] += ld_shared_cluster(from + u * 512u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r + u >= r1) break;
          const float f = v[u] * alpha;
          const uint16_t high = cvt_f32_to_16(f, DT, 1);
          const long long to = static_cast<long long>(p0 + r + u) * p.pitch + j;
          p.high[to] = high;
          // an infinite product leaves nothing (inf - inf would make a NaN of it)
          const float held = cvt_16_to_f32(high, DT);
          p.low[to] = cvt_f32_to_16(isinf(held) ? 0.0f : f - held, DT, 1);
        }
      }
    }
  }
  __syncthreads();
  if (*abort_flag != 0u) {
    if (threadIdx.x == 0) atomicExch(p.status, kStatusTimeout);
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 200000ull) {
    }
  }
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, 64);
  }
}

}  // namespace kapyb
