// The products of rows that pick their weights, on CUDA cores: any strides and
// alignment, f16 / bf16 / f32 operands (f32 multiplied as f32), sums in 32 bits in
// ascending k.  What TMA can describe and the tensor cores multiply runs on the
// kernels of grouped_sm100.cuh instead; this is the path for the rest.
#pragma once

#include "common.cuh"

namespace kapyb {

// Row ranges of the groups as the device holds them: every offset is clamped to
// [0, rows], so that a broken plan cannot lead outside a tensor.
__device__ __forceinline__ void group_range(const int32_t *offsets, int g, int rows, int &begin, int &end) {
  begin = min(max(offsets[g], 0), rows);
  end = min(max(offsets[g + 1], 0), rows);
}

struct RowsSimtParams {
  const void *x;  // lhs [src_rows, K]
  long long x_s0, x_s1;
  int src_rows;
  const void *w;  // one group's [K, cols]
  long long w_s0, w_s1, w_group;
  int in_dtype;
  int groups, rows, K, cols;  // rows: positions of the plan; cols: output columns
  const int32_t *offsets, *order;
  int fan;
  int gated;  // w has 2 * cols columns: gate, then up
  void *out;
  long long out_s0, out_s1, out_group;
  int out_dtype;
  float alpha;
  const void *bias;
  int bias_dtype, activation, rounding;
  int cols_w;  // columns of one group's w (bias pitch)
};

// The source row of plan position p, or -1.
__device__ __forceinline__ long long source_row(const int32_t *order, int fan, int src_rows, long long p) {
  long long r = p;
  if (order) {
    const int o = order[p];
    if (o < 0) return -1;
    r = o / fan;
  }
  return r < src_rows ? r : -1;
}

// 32 x 32 outputs per block of 256 threads, four per thread (rows ty, ty+8, ...).
// blockIdx.y walks (group, row block) pairs: every block looks its pair up in the
// offsets, blocks behind the last pair leave.
__global__ void __launch_bounds__(256) rows_simt_kernel(const RowsSimtParams p) {
  __shared__ float xs[32][33], ws[32][33], us[32][33];
  __shared__ int sg, sp0, sp1;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n0 = blockIdx.x * 32;
  for (int want = blockIdx.y;; want += gridDim.y) {
    if (threadIdx.x == 0) {
      int left = want, high = 0;
      sg = -1;
      for (int g = 0; g < p.groups; ++g) {
        int b, e;
        group_range(p.offsets, g, p.rows, b, e);
        high = b = max(b, high);  // as in the tensor-core kernels, groups never overlap
        const int blocks = e > b ? (e - b + 31) / 32 : 0;
        if (left < blocks) {
          sg = g;
          sp0 = b + left * 32;
          sp1 = min(e, sp0 + 32);
          break;
        }
        left -= blocks;
      }
    }
    __syncthreads();
    if (sg < 0) return;
    const int g = sg, p0 = sp0, p1 = sp1;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, up[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < p.K; k0 += 32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = ty + 8 * i, k = k0 + tx;
        float v = 0.0f;
        if (p0 + r < p1 && k < p.K) {
          const long long src = source_row(p.order, p.fan, p.src_rows, p0 + r);
          if (src >= 0) v = load_as_f32(p.x, p.in_dtype, src * p.x_s0 + k * p.x_s1);
        }
        xs[r][tx] = v;
        const int kw = k0 + r, n = n0 + tx;
        float a = 0.0f, b = 0.0f;
        if (kw < p.K && n < p.cols) {
          a = load_as_f32(p.w, p.in_dtype, g * p.w_group + kw * p.w_s0 + n * p.w_s1);
          if (p.gated)
            b = load_as_f32(p.w, p.in_dtype, g * p.w_group + kw * p.w_s0 + (p.cols + n) * p.w_s1);
        }
        ws[r][tx] = a;
        us[r][tx] = b;
      }
      __syncthreads();
      const int kn = min(32, p.K - k0);
      for (int k = 0; k < kn; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[i] = fmaf(xs[ty + 8 * i][k], ws[k][tx], acc[i]);
          if (p.gated) up[i] = fmaf(xs[ty + 8 * i][k], us[k][tx], up[i]);
        }
      }
      __syncthreads();
    }
    const int n = n0 + tx;
    if (n < p.cols) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q = p0 + ty + 8 * i;
        if (q >= p1) continue;
        float v = acc[i] * p.alpha, u = up[i] * p.alpha;
        if (p.bias) {
          v += load_as_f32(p.bias, p.bias_dtype, static_cast<long long>(g) * p.cols_w + n);
          if (p.gated) u += load_as_f32(p.bias, p.bias_dtype, static_cast<long long>(g) * p.cols_w + p.cols + n);
        }
        v = apply_activation(p.activation, v);
        if (p.gated) v *= u;
        store_from_f32(p.out, p.out_dtype, q * p.out_s0 + n * p.out_s1, v, p.rounding);
      }
    }
    __syncthreads();
  }
}

// out[g][k][n] = alpha * sum over the group's positions of x[row][k] * grad[p][n].
// Here `w` is the gradient [rows, cols] and `out` one group's [K, cols].
__global__ void __launch_bounds__(256) rows_grad_simt_kernel(const RowsSimtParams p) {
  __shared__ float xs[32][33], gs[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n0 = blockIdx.x * 32, k0 = blockIdx.y * 32;
  for (int g = blockIdx.z; g < p.groups; g += gridDim.z) {
    int b, e;
    group_range(p.offsets, g, p.rows, b, e);
    // an offset below one in front of it counts as that one: as in the other kernels, groups
    // never overlap
    for (int i = tx; i < g; i += 32) b = max(b, min(p.offsets[i], p.rows));
    b = __reduce_max_sync(0xffffffffu, b);
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int q0 = b; q0 < e; q0 += 32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = ty + 8 * i, q = q0 + r;
        float xv = 0.0f, gv = 0.0f;
        if (q < e) {
          const long long src = source_row(p.order, p.fan, p.src_rows, q);
          if (src >= 0 && k0 + tx < p.K) xv = load_as_f32(p.x, p.in_dtype, src * p.x_s0 + (k0 + tx) * p.x_s1);
          if (src >= 0 && n0 + tx < p.cols) gv = load_as_f32(p.w, p.in_dtype, q * p.w_s0 + (n0 + tx) * p.w_s1);
        }
        xs[r][tx] = xv;
        gs[r][tx] = gv;
      }
      __syncthreads();
      const int qn = min(32, e - q0);
      for (int q = 0; q < qn; ++q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(xs[q][ty + 8 * i], gs[q][tx], acc[i]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = k0 + ty + 8 * i, n = n0 + tx;
      if (k < p.K && n < p.cols)
        store_from_f32(p.out, p.out_dtype, g * p.out_group + k * p.out_s0 + n * p.out_s1, acc[i] * p.alpha,
                       p.rounding);
    }
  }
}

// ------------------------------------------------------------------ adapters

struct AdapterSimtParams {
  const void *x;
  long long x_s0, x_s1;
  const void *w;
  long long w_s0, w_s1;
  const void *down, *up;  // one adapter's [K, r] and [r, cols]
  long long d_s0, d_s1, d_group, u_s0, u_s1, u_group;
  int in_dtype;
  int groups, rows, K, cols, rank;
  const int32_t *index;
  const float *scale;  // [groups] or nullptr
  float *low;          // [rows, rank]: scale * x . down of the row's adapter, 0 without one
  void *out;
  long long out_s0, out_s1;
  int out_dtype;
  float alpha;
  const void *bias;
  int bias_dtype, bias_axis, activation, rounding;
};

// low[t][j] for one row per block: threads split K, a tree joins them.
__global__ void __launch_bounds__(256) adapter_low_simt_kernel(const AdapterSimtParams p) {
  __shared__ float part[8];
  const long long t = blockIdx.x;
  const int i = p.index[t];
  const bool on = i >= 0 && i < p.groups;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int j = 0; j < p.rank; ++j) {
    float v = 0.0f;
    if (on)
      for (int k = threadIdx.x; k < p.K; k += 256)
        v = fmaf(load_as_f32(p.x, p.in_dtype, t * p.x_s0 + k * p.x_s1),
                 load_as_f32(p.down, p.in_dtype, i * p.d_group + k * p.d_s0 + j * p.d_s1), v);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if (lane == 0) part[w] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
      float s = 0.0f;
      for (int k = 0; k < 8; ++k) s += part[k];
      p.low[t * p.rank + j] = on ? s * (p.scale ? p.scale[i] : 1.0f) : 0.0f;
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(256) adapter_simt_kernel(const AdapterSimtParams p) {
  __shared__ float xs[32][33], ws[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n0 = blockIdx.x * 32, n = n0 + tx;
  for (long long t0 = static_cast<long long>(blockIdx.y) * 32; t0 < p.rows;
       t0 += static_cast<long long>(gridDim.y) * 32) {
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < p.K; k0 += 32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = ty + 8 * i;
        xs[r][tx] = t0 + r < p.rows && k0 + tx < p.K
                        ? load_as_f32(p.x, p.in_dtype, (t0 + r) * p.x_s0 + (k0 + tx) * p.x_s1)
                        : 0.0f;
        ws[r][tx] = k0 + r < p.K && n < p.cols
                        ? load_as_f32(p.w, p.in_dtype, (k0 + r) * p.w_s0 + n * p.w_s1)
                        : 0.0f;
      }
      __syncthreads();
      const int kn = min(32, p.K - k0);
      for (int k = 0; k < kn; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(xs[ty + 8 * i][k], ws[k][tx], acc[i]);
      }
      __syncthreads();
    }
    if (n < p.cols) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long t = t0 + ty + 8 * i;
        if (t >= p.rows) continue;
        float v = acc[i] * p.alpha;
        if (p.bias) v += load_as_f32(p.bias, p.bias_dtype, p.bias_axis == 1 ? n : t);
        const int a = p.index[t];
        if (a >= 0 && a < p.groups) {
          float d = 0.0f;
          for (int j = 0; j < p.rank; ++j)
            d = fmaf(p.low[t * p.rank + j], load_as_f32(p.up, p.in_dtype, a * p.u_group + j * p.u_s0 + n * p.u_s1), d);
          v += d;
        }
        store_from_f32(p.out, p.out_dtype, t * p.out_s0 + n * p.out_s1, apply_activation(p.activation, v),
                       p.rounding);
      }
    }
  }
}

}  // namespace kapyb
