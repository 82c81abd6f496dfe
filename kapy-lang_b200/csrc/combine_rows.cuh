// Weighted sum of a token's rows and its gradients.
//
//   out[t]          = sum_j w[t,j] rows[slots[t,j]]        (a slot < 0 adds nothing)
//   grad_rows[s]    = w[t,j] grad_out[t],  s = slots[t,j]
//   grad_weights[t,j] = <grad_out[t], rows[slots[t,j]]>     (0 for a slot < 0)
//
// Sums in 32 bits in ascending j, one rounding at the store.
#pragma once

#include "common.cuh"
#include "reduce.cuh"

namespace kapyb {

constexpr int kCombineMaxK = 32;

struct CombineParams {
  const void *rows;
  long long rows_s0, rows_s1;
  int rows_dtype, n_rows;
  const int32_t *slots;
  const float *weights;  // [tokens, k] or nullptr (all one)
  int tokens, k, cols;
  void *out;
  long long out_s0, out_s1;
  int out_dtype, rounding;
  // backward
  const void *grad_out;
  long long go_s0, go_s1;
  int go_dtype;
  void *grad_rows;  // may be nullptr
  long long gr_s0, gr_s1;
  int gr_dtype;
  float *grad_weights;  // may be nullptr
};

// 16 bytes of a row as f32 values (8 of a 16-bit type, 4 of f32)
template <int DT>
__device__ __forceinline__ void unpack16B(const uint4 &q, float (&f)[DT == KAPYB_F32 ? 4 : 8]) {
  const uint32_t ws[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (DT == KAPYB_F32)
      f[t] = __uint_as_float(ws[t]);
    else
      unpack2_16<DT>(ws[t], f[2 * t], f[2 * t + 1]);
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack16B(const float (&f)[DT == KAPYB_F32 ? 4 : 8]) {
  uint4 q;
  if constexpr (DT == KAPYB_F32)
    q = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    q = make_uint4(cvt_pack2_t<DT, 1>(f[0], f[1]), cvt_pack2_t<DT, 1>(f[2], f[3]),
                   cvt_pack2_t<DT, 1>(f[4], f[5]), cvt_pack2_t<DT, 1>(f[6], f[7]));
  return q;
}

// 32 bytes of a row (16 of a 16-bit type, 8 of f32).
template <int DT>
__device__ __forceinline__ void fma32B(const Vec32B &v, float w, float (&acc)[DT == KAPYB_F32 ? 8 : 16]) {
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    if constexpr (DT == KAPYB_F32) {
      acc[t] = fmaf(w, __uint_as_float(v.w[t]), acc[t]);
    } else {
      float lo, hi;
      unpack2_16<DT>(v.w[t], lo, hi);
      acc[2 * t] = fmaf(w, lo, acc[2 * t]);
      acc[2 * t + 1] = fmaf(w, hi, acc[2 * t + 1]);
    }
  }
}

// Rows and output of one type, in pieces of 32 bytes (WIDE) or 16: a thread owns one
// piece of one token and has the loads of four rows in flight before it adds them.
// A row's rows lie anywhere, but a warp reads 1 KB runs of each.
template <int DT, bool WIDE>
__global__ void __launch_bounds__(256) combine_vec_kernel(const CombineParams p, uint32_t pieces) {
  constexpr int esz = DT == KAPYB_F32 ? 4 : 2;
  constexpr int BYTES = WIDE ? 32 : 16, E = BYTES / esz, U = 4;
  const unsigned long long id = static_cast<unsigned long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long t = id / pieces;
  if (t >= p.tokens) return;
  const long long col = static_cast<long long>(id - t * static_cast<unsigned long long>(pieces)) * E;
  const char *base = static_cast<const char *>(p.rows) + col * esz;
  const long long pitch = p.rows_s0 * esz;
  float acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.0f;
  for (int j0 = 0; j0 < p.k; j0 += U) {
    Vec32B v[WIDE ? U : 1];
    uint4 q[WIDE ? 1 : U];
    float w[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      on[u] = false;
      if (j0 + u < p.k) {
        const int s = __ldg(p.slots + t * p.k + j0 + u);
        on[u] = s >= 0 && s < p.n_rows;
        w[u] = p.weights ? __ldg(p.weights + t * p.k + j0 + u) : 1.0f;
        if constexpr (WIDE) {
          if (on[u]) v[u] = ld_nc_v8(base + s * pitch);
        } else {
          if (on[u]) q[u] = __ldg(reinterpret_cast<const uint4 *>(base + s * pitch));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!on[u]) continue;
      if constexpr (WIDE) {
        fma32B<DT>(v[u], w[u], acc);
      } else {
        float f[E];
        unpack16B<DT>(q[u], f);
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = fmaf(w[u], f[i], acc[i]);
      }
    }
  }
  uint4 *out = reinterpret_cast<uint4 *>(static_cast<char *>(p.out) + (t * p.out_s0 + col) * esz);
#pragma unroll
  for (int h = 0; h < BYTES / 16; ++h) {
    float f[16 / esz];
#pragma unroll
    for (int i = 0; i < 16 / esz; ++i) f[i] = acc[h * (16 / esz) + i];
    __stcs(out + h, pack16B<DT>(f));
  }
}

// Any strides, types and alignment: one element per thread.
__global__ void __launch_bounds__(256) combine_any_kernel(const CombineParams p) {
  const unsigned long long id = static_cast<unsigned long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long t = id / static_cast<unsigned>(p.cols);
  if (t >= p.tokens) return;
  const long long col = id - t * static_cast<unsigned long long>(p.cols);
  float acc = 0.0f;
  for (int j = 0; j < p.k; ++j) {
    const int s = p.slots[t * p.k + j];
    if (s < 0 || s >= p.n_rows) continue;
    const float w = p.weights ? p.weights[t * p.k + j] : 1.0f;
    acc = fmaf(w, load_as_f32(p.rows, p.rows_dtype, s * p.rows_s0 + col * p.rows_s1), acc);
  }
  store_from_f32(p.out, p.out_dtype, t * p.out_s0 + col * p.out_s1, acc, p.rounding);
}

// Backward: one block per token.  A thread keeps its pieces of the output's gradient
// only for the row at hand; the k inner products meet in a warp tree and then in
// warp order, so a result is the same bits every time.
// VEC: 16-byte pieces of one type everywhere; otherwise element by element.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) combine_backward_kernel(const CombineParams p) {
  constexpr int E = VEC ? (DT == KAPYB_F32 ? 4 : 8) : 1;
  constexpr int esz = DT == KAPYB_F32 ? 4 : 2;
  constexpr int U = 4;  // rows in flight
  __shared__ float part[8][U];
  const long long t = blockIdx.x;
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
  for (int j0 = 0; j0 < p.k; j0 += U) {
    int s[U];
    float w[U], dot[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = -1;
      w[u] = 1.0f;
      dot[u] = 0.0f;
      if (j0 + u < p.k) {
        s[u] = p.slots[t * p.k + j0 + u];
        if (s[u] >= p.n_rows) s[u] = -1;
        if (p.weights) w[u] = p.weights[t * p.k + j0 + u];
      }
    }
    for (int c = threadIdx.x * E; c < p.cols; c += blockDim.x * E) {
      float g[E];
      if constexpr (VEC) {
        unpack16B<DT>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const char *>(p.grad_out) +
                                                            (t * p.go_s0 + c) * esz)), g);
      } else {
        g[0] = load_as_f32(p.grad_out, p.go_dtype, t * p.go_s0 + c * p.go_s1);
      }
      if (p.grad_weights) {
        float f[U][E];
        if constexpr (VEC) {
          uint4 q[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            q[u] = make_uint4(0u, 0u, 0u, 0u);
            if (s[u] >= 0)
              q[u] = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const char *>(p.rows) +
                                                            (s[u] * p.rows_s0 + c) * esz));
          }
#pragma unroll
          for (int u = 0; u < U; ++u) unpack16B<DT>(q[u], f[u]);
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u)
            f[u][0] = s[u] >= 0 ? load_as_f32(p.rows, p.rows_dtype, s[u] * p.rows_s0 + c * p.rows_s1) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (s[u] >= 0) {
#pragma unroll
            for (int i = 0; i < E; ++i) dot[u] = fmaf(g[i], f[u][i], dot[u]);
          }
      }
      if (p.grad_rows) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (s[u] < 0) continue;
          if constexpr (VEC) {
            float o[E];
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = w[u] * g[i];
            __stcs(reinterpret_cast<uint4 *>(static_cast<char *>(p.grad_rows) + (s[u] * p.gr_s0 + c) * esz),
                   pack16B<DT>(o));
          } else {
            store_from_f32(p.grad_rows, p.gr_dtype, s[u] * p.gr_s0 + c * p.gr_s1, w[u] * g[0], p.rounding);
          }
        }
      }
    }
    if (p.grad_weights) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], off);
        if (lane == 0) part[wp][u] = dot[u];
      }
      __syncthreads();
      if (threadIdx.x < U && j0 + threadIdx.x < p.k) {
        float v = 0.0f;
        for (int k = 0; k < n_warps; ++k) v += part[k][threadIdx.x];
        p.grad_weights[t * p.k + j0 + threadIdx.x] = v;
      }
      __syncthreads();
    }
  }
}

}  // namespace kapyb
