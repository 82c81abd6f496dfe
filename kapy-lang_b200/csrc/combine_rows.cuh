// Weighted sum of a token's rows and its gradients.
//
//   out[t]          = sum_j w[t,j] rows[slots[t,j]]        (a slot < 0 adds nothing)
//   grad_rows[s]    = w[t,j] grad_out[t],  s = slots[t,j]
//   grad_weights[t,j] = <grad_out[t], rows[slots[t,j]]>     (0 for a slot < 0)
//
// Sums in 32 bits in ascending j, one rounding at the store.
#pragma once

#include "common.cuh"
#include "ptx_sm100.cuh"
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

// 32 or 16 bytes of a row that the kernel in front may still be writing when this one is
// set up: ordinary loads (the .nc ones are for memory nothing writes while a kernel lives),
// kept behind the wait.
__device__ __forceinline__ Vec32B ld_behind_v8(const void *p) {
  Vec32B v;
  asm volatile("ld.global.L1::no_allocate.v8.u32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]),
                 "=r"(v.w[7])
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ uint4 ld_behind_v4(const void *p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// Rows and output of one type, in pieces of 32 bytes (WIDE) or 16: a thread owns one
// piece of one token and has the loads of four rows in flight before it adds them.
// A row's rows lie anywhere, but a warp reads 1 KB runs of each.
template <int DT, bool WIDE>
__global__ void __launch_bounds__(256) combine_vec_kernel(const CombineParams p, uint32_t pieces) {
  constexpr int esz = DT == KAPYB_F32 ? 4 : 2;
  constexpr int BYTES = WIDE ? 32 : 16, E = BYTES / esz, U = 4;
  ptx::griddep_wait();
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
        const int s = p.slots[t * p.k + j0 + u];  // an ordinary load stays behind the wait
        on[u] = s >= 0 && s < p.n_rows;
        w[u] = p.weights ? p.weights[t * p.k + j0 + u] : 1.0f;
        if constexpr (WIDE) {
          if (on[u]) v[u] = ld_behind_v8(base + s * pitch);
        } else {
          if (on[u]) q[u] = ld_behind_v4(base + s * pitch);
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

// An element as it lies in memory, zero where it is not wanted.  What bounds the kernels of
// single elements is the latency of their loads, so those of four rows are issued before
// the first is widened, in an order the compiler keeps (four of 8192 tokens' rows of 2047
// f16: 53 us, backward 84; an element at a time 117 and 129; rows of 2048 by pieces 39 and 59).
template <int DT>
struct RawOf {
  using type = uint16_t;
};
template <>
struct RawOf<KAPYB_F32> {
  using type = uint32_t;
};
template <int DT>
__device__ __forceinline__ typename RawOf<DT>::type raw_at(const char *at, bool wanted) {
  typename RawOf<DT>::type v;
  if constexpr (DT == KAPYB_F32)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.nc.u32 %0, [%1];\n\t}"
                 : "=r"(v)
                 : "l"(at), "r"(static_cast<int>(wanted)));
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\tmov.b16 %0, 0;\n\t@p ld.global.nc.u16 %0, [%1];\n\t}"
                 : "=h"(v)
                 : "l"(at), "r"(static_cast<int>(wanted)));
  return v;
}
template <int DT>
__device__ __forceinline__ float raw_to_f32(typename RawOf<DT>::type v) {
  if constexpr (DT == KAPYB_F32) return __uint_as_float(v);
  else return cvt_16_to_f32(v, DT);
}

// Any strides and alignment, the output in any type: a warp owns 32 * COLS columns of one
// token, a lane every 32nd of them, with four rows' loads in flight.  UNIT: the rows'
// columns are adjacent (offsets known to the compiler: the loop is bound by instructions).
template <int DT, int COLS, bool UNIT>
__global__ void __launch_bounds__(256) combine_any_kernel(const CombineParams p, uint32_t chunks) {
  constexpr int U = 4;
  const unsigned long long id = blockIdx.x * 8ull + (threadIdx.x >> 5);
  const long long t = id / chunks;
  if (t >= p.tokens) return;
  const int c0 = static_cast<int>(id - t * static_cast<unsigned long long>(chunks)) * (32 * COLS) + (threadIdx.x & 31);
  constexpr int esz = DT == KAPYB_F32 ? 4 : 2;
  const int out_esz = p.out_dtype == KAPYB_F32 ? 4 : 2;
  const char *base = static_cast<const char *>(p.rows) + c0 * (UNIT ? 1ll : p.rows_s1) * esz;
  char *out = static_cast<char *>(p.out) + (t * p.out_s0 + c0 * p.out_s1) * out_esz;
  const long long pitch = p.rows_s0 * esz, step = (UNIT ? 32ll : 32 * p.rows_s1) * esz;
  const long long out_step = 32 * p.out_s1 * out_esz;
  float acc[COLS];
#pragma unroll
  for (int i = 0; i < COLS; ++i) acc[i] = 0.0f;
  for (int j0 = 0; j0 < p.k; j0 += U) {
    typename RawOf<DT>::type raw[U][COLS];
    float w[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = j0 + u < p.k ? __ldg(p.slots + t * p.k + j0 + u) : -1;
      on[u] = s >= 0 && s < p.n_rows;
      w[u] = p.weights && j0 + u < p.k ? __ldg(p.weights + t * p.k + j0 + u) : 1.0f;
      const char *row = base + s * pitch;
#pragma unroll
      for (int i = 0; i < COLS; ++i) raw[u][i] = raw_at<DT>(row + i * step, on[u] && c0 + 32 * i < p.cols);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!on[u]) continue;
#pragma unroll
      for (int i = 0; i < COLS; ++i) acc[i] = fmaf(w[u], raw_to_f32<DT>(raw[u][i]), acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < COLS; ++i)
    if (c0 + 32 * i < p.cols) store_from_f32(out + i * out_step, p.out_dtype, 0, acc[i], p.rounding);
}

// Backward: one block per token.  A thread keeps its pieces of the output's gradient
// only for the row at hand; the k inner products meet in a warp tree and then in
// warp order, so a result is the same bits every time.
// VEC: 16-byte pieces of one type everywhere; otherwise a thread's elements lie a block
// apart, all of type DT or (DT negative) each tensor's own.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) combine_backward_kernel(const CombineParams p) {
  constexpr int E = VEC && DT != KAPYB_F32 ? 8 : 4;
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
    for (int c = threadIdx.x * (VEC ? E : 1); c < p.cols; c += blockDim.x * E) {
      float g[E];
      // !VEC: element i of this thread, of a row at element `first`, stride s1
      auto in_row = [&](int i) { return c + i * static_cast<int>(blockDim.x) < p.cols; };
      auto type = [](int own) { return DT < 0 ? own : DT; };
      auto bytes_at = [&](long long first, long long s1, int own) {
        return (first + c * s1) * (type(own) == KAPYB_F32 ? 4 : 2);
      };
      auto step_of = [&](long long s1, int own) { return blockDim.x * s1 * (type(own) == KAPYB_F32 ? 4 : 2); };
      if constexpr (VEC) {
        unpack16B<DT>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const char *>(p.grad_out) +
                                                            (t * p.go_s0 + c) * esz)), g);
      } else {
        const char *src = static_cast<const char *>(p.grad_out) + bytes_at(t * p.go_s0, p.go_s1, p.go_dtype);
        const long long step = step_of(p.go_s1, p.go_dtype);
        if constexpr (DT >= 0) {
          typename RawOf<DT>::type raw[E];
#pragma unroll
          for (int i = 0; i < E; ++i) raw[i] = raw_at<DT>(src + i * step, in_row(i));
#pragma unroll
          for (int i = 0; i < E; ++i) g[i] = raw_to_f32<DT>(raw[i]);
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) g[i] = in_row(i) ? load_as_f32(src + i * step, p.go_dtype, 0) : 0.0f;
        }
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
          const long long step = step_of(p.rows_s1, p.rows_dtype);
          auto row = [&](int u) {
            return static_cast<const char *>(p.rows) + bytes_at(s[u] * p.rows_s0, p.rows_s1, p.rows_dtype);
          };
          if constexpr (DT >= 0) {
            typename RawOf<DT>::type raw[U][E];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int i = 0; i < E; ++i) raw[u][i] = raw_at<DT>(row(u) + i * step, s[u] >= 0 && in_row(i));
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int i = 0; i < E; ++i) f[u][i] = raw_to_f32<DT>(raw[u][i]);
          } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int i = 0; i < E; ++i)
                f[u][i] = s[u] >= 0 && in_row(i) ? load_as_f32(row(u) + i * step, p.rows_dtype, 0) : 0.0f;
          }
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
            char *dst = static_cast<char *>(p.grad_rows) + bytes_at(s[u] * p.gr_s0, p.gr_s1, p.gr_dtype);
            const long long step = step_of(p.gr_s1, p.gr_dtype);
#pragma unroll
            for (int i = 0; i < E; ++i)
              if (in_row(i)) store_from_f32(dst + i * step, type(p.gr_dtype), 0, w[u] * g[i], p.rounding);
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
