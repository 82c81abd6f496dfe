// Routing of rows to experts: scores, choice of the top k, weights, and the
// gradient of the logits.
//
//   s = softmax(x) or sigmoid(x)        c = s + bias   (c only decides who is chosen)
//   w_j = scale * s_j [/ sum of the chosen s]
//
// One warp owns one row and keeps it in registers (expert e sits in lane e % 32),
// so the row is read once and nothing but k weights and k indices leaves the warp.
// A pick is two warp-wide integer reductions (redux.sync): the largest key, then
// the lowest index that has it, which is the rule for ties.
//
// Keys.  A choice between experts must not depend on how an exponential was
// rounded.  Without a bias the order of the scores is the order of the logits, so
// the logits themselves are the keys, which is exact.  With a bias (or with groups
// ranked by a sum of two scores) c is formed in 32 bits together with a bound on
// its error, and a row in which two neighbours of the ranking lie within that bound
// of one another is decided again in 64 bits (choose_f64).  On normally
// distributed logits that is about one row in a thousand.
#pragma once

#include "common.cuh"

namespace kapyb {

constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopK = 32;
constexpr int kRouteMaxGroups = 32;

struct RouteParams {
  const void *x;  // element (0, 0) of the logits
  long long x_s0, x_s1;
  int x_dtype;
  int rows, experts;
  const float *bias;  // [experts] or nullptr
  int sigmoid, top_k, n_groups, group_size, top_groups, group_best, renormalize;
  float scale;
  float *weights;  // [rows, top_k]
  int32_t *chosen;  // [rows, top_k]
  // backward
  const int32_t *picked;      // [rows, top_k]
  const float *grad_weights;  // [rows, top_k]
  void *grad;
  long long g_s0, g_s1;
  int g_dtype;
};

// Ranks as unsigned integers: 0 = masked (never chosen), 1 = NaN (behind every
// number), then the numbers in ascending order, both zeros alike.
__device__ __forceinline__ uint32_t rank_key(float c) {
  if (c != c) return 1u;
  const uint32_t b = __float_as_uint(c + 0.0f);
  return b & 0x80000000u ? ~b : (b | 0x80000000u);  // -inf -> 0x007fffff
}
__device__ __forceinline__ unsigned long long rank_key64(double c) {
  if (c != c) return 1ull;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(c + 0.0));
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  if (key == 1u) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(key & 0x80000000u ? (key & 0x7fffffffu) : ~key);
}

__device__ __forceinline__ unsigned long long warp_max64(unsigned long long v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, off);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {  // NaN is left out
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

__device__ __forceinline__ float route_logit(const RouteParams &p, long long row, int e) {
  return load_as_f32(p.x, p.x_dtype, row * p.x_s0 + e * p.x_s1);
}

// The kept groups of a row as a bit mask, from the lanes' group keys (lane q holds
// group q; 0 = the group has nothing to choose from).
template <class Key>
__device__ __forceinline__ uint32_t keep_groups(const RouteParams &p, Key key, int lane) {
  uint32_t kept = 0u;
  for (int i = 0; i < p.top_groups; ++i) {
    Key best;
    if constexpr (sizeof(Key) == 8)
      best = warp_max64(key);
    else
      best = __reduce_max_sync(0xffffffffu, key);
    if (best == 0) break;
    const int q = __ffs(__ballot_sync(0xffffffffu, key == best)) - 1;
    kept |= 1u << q;
    if (lane == q) key = 0;
  }
  return kept;
}

// One row's choice with every score in 64 bits: lane j < top_k returns the j-th
// choice, or -1.  Walks the row again per step instead of keeping it: rare.
__device__ __noinline__ int choose_f64(const RouteParams &p, long long row) {
  const int lane = threadIdx.x & 31;
  double top = -INFINITY, z = 1.0;
  if (!p.sigmoid) {
    float m = -INFINITY;
    for (int e = lane; e < p.experts; e += 32) m = fmaxf(m, route_logit(p, row, e));
    top = warp_max(m);
    double s = 0.0;
    for (int e = lane; e < p.experts; e += 32) {
      const float x = route_logit(p, row, e);
      if (x != -INFINITY) s += exp(static_cast<double>(x) - top);
    }
    z = warp_sum64(s);
  }
  // rank of expert e, 0 when it is masked
  auto key_of = [&](int e) -> unsigned long long {
    const float x = route_logit(p, row, e);
    if (x == -INFINITY) return 0ull;
    const double xd = x;
    double c = p.sigmoid ? 1.0 / (1.0 + exp(-xd)) : exp(xd - top) / z;
    if (p.bias) c += static_cast<double>(p.bias[e]);
    return rank_key64(c);
  };
  auto value_of = [&](unsigned long long key) -> double {
    if (key == 1ull) return __longlong_as_double(0x7fffffffffffffffll);
    return __longlong_as_double(static_cast<long long>(key >> 63 ? (key & 0x7fffffffffffffffull) : ~key));
  };
  uint32_t kept = 0xffffffffu;
  if (p.n_groups > 1) {
    unsigned long long mine = 0ull;
    for (int q = 0; q < p.n_groups; ++q) {
      unsigned long long k1 = 0ull, k2 = 0ull;  // this lane's two best
      for (int e = q * p.group_size + lane; e < (q + 1) * p.group_size; e += 32) {
        const unsigned long long k = key_of(e);
        if (k > k1) {
          k2 = k1;
          k1 = k;
        } else if (k > k2) {
          k2 = k;
        }
      }
      const unsigned long long g1 = warp_max64(k1);
      unsigned long long gk = g1;
      if (p.group_best == 2 && g1 != 0ull) {
        const int owner = __ffs(__ballot_sync(0xffffffffu, k1 == g1)) - 1;
        const unsigned long long g2 = warp_max64(lane == owner ? k2 : k1);
        if (g2 != 0ull) gk = rank_key64(value_of(g1) + value_of(g2));
      }
      if (lane == q) mine = gk;
    }
    kept = keep_groups(p, mine, lane);
  }
  int pick = -1;
  unsigned long long last = ~0ull;  // the previous choice's rank and index: the next one is behind it
  int last_e = -1;
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long best = 0ull;
    int best_e = 0x7fffffff;
    for (int e = lane; e < p.experts; e += 32) {
      if (p.n_groups > 1 && !((kept >> (e / p.group_size)) & 1u)) continue;
      const unsigned long long k = key_of(e);
      if (k == 0ull || k > last || (k == last && e <= last_e)) continue;
      if (k > best) {
        best = k;
        best_e = e;
      }
    }
    const unsigned long long top_key = warp_max64(best);
    if (top_key == 0ull) break;
    const int e = static_cast<int>(
        __reduce_min_sync(0xffffffffu, best == top_key ? static_cast<uint32_t>(best_e) : 0x7fffffffu));
    if (lane == j) pick = e;
    last = top_key;
    last_e = e;
  }
  return pick;
}

// exp(x - shift) and the like for the weights: full-precision expf and division,
// f32 throughout.
// VPT experts per lane.
template <int VPT>
__global__ void __launch_bounds__(256) route_kernel(const RouteParams p) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  for (long long row = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
       row < p.rows; row += warps) {
    float x[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = i * 32 + lane;
      x[i] = e < p.experts ? route_logit(p, row, e) : -INFINITY;
    }
    float top = 0.0f, z = 1.0f;
    const bool by_score = p.bias != nullptr || (p.n_groups > 1 && p.group_best > 1);
    if (!p.sigmoid) {
      float m = x[0];
#pragma unroll
      for (int i = 1; i < VPT; ++i) m = fmaxf(m, x[i]);
      top = warp_max(m);
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) s += x[i] == -INFINITY ? 0.0f : expf(x[i] - top);
      z = warp_sum(s);
    }
    // c and the bound on its error, from the 32-bit evaluation: a few roundings of
    // s (relative), the rounding of the exponent's argument (|x - top| 2^-24,
    // absolute in the exponent, so relative in s), one rounding of the sum with the bias
    auto score_of = [&](float xv, int e) -> float {
      float s = p.sigmoid ? 1.0f / (1.0f + expf(-xv)) : expf(xv - top) / z;
      return p.bias != nullptr ? s + p.bias[e] : s;
    };
    auto error_of = [&](float xv, float c) -> float {
      const float s = p.sigmoid ? 1.0f / (1.0f + expf(-xv)) : expf(xv - top) / z;
      const float rel = p.sigmoid ? 16.0f : 24.0f + fabsf(xv - top);
      return s * rel * 5.9604645e-8f + fabsf(c) * 1.1920929e-7f + 1e-37f;
    };
    uint32_t key[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = i * 32 + lane;
      key[i] = x[i] == -INFINITY ? 0u : rank_key(by_score ? score_of(x[i], e) : x[i]);
    }
    bool unsure = false;
    if (p.n_groups > 1) {
      uint32_t mine = 0u;
      float err = 0.0f;
      for (int q = 0; q < p.n_groups; ++q) {
        const int lo = q * p.group_size, hi = lo + p.group_size;
        uint32_t k1 = 0u, k2 = 0u;
        float e1 = 0.0f, e2 = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int e = i * 32 + lane;
          const uint32_t k = e >= lo && e < hi ? key[i] : 0u;
          const float er = by_score ? error_of(x[i], key_value(k)) : 0.0f;
          if (k > k1) {
            k2 = k1;
            e2 = e1;
            k1 = k;
            e1 = er;
          } else if (k > k2) {
            k2 = k;
            e2 = er;
          }
        }
        const uint32_t g1 = __reduce_max_sync(0xffffffffu, k1);
        uint32_t gk = g1;
        float ge = 0.0f;
        if (g1 != 0u) {
          const int owner = __ffs(__ballot_sync(0xffffffffu, k1 == g1)) - 1;
          ge = __shfl_sync(0xffffffffu, e1, owner);
          if (p.group_best == 2) {
            const uint32_t r1 = lane == owner ? k2 : k1;
            const float re = lane == owner ? e2 : e1;
            const uint32_t g2 = __reduce_max_sync(0xffffffffu, r1);
            if (g2 != 0u) {
              const int owner2 = __ffs(__ballot_sync(0xffffffffu, r1 == g2)) - 1;
              const float sum = key_value(g1) + key_value(g2);
              ge += __shfl_sync(0xffffffffu, re, owner2) + fabsf(sum) * 1.1920929e-7f;
              gk = rank_key(sum);
            }
          }
        }
        if (lane == q) {
          mine = gk;
          err = ge;
        }
      }
      const uint32_t kept = keep_groups(p, mine, lane);
      if (by_score && p.top_groups < p.n_groups) {
        // the weakest kept group against the strongest one left out
        const bool in = (kept >> lane) & 1u;
        const uint32_t low = __reduce_min_sync(0xffffffffu, in ? mine : 0xffffffffu);
        const uint32_t high = __reduce_max_sync(0xffffffffu, in ? 0u : mine);
        if (kept != 0u && high != 0u) {
          const float e_max = warp_max(err);
          unsure = !(key_value(low) - key_value(high) > 2.0f * e_max);
        }
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = i * 32 + lane;
        if (e < p.experts && !((kept >> (e / p.group_size)) & 1u)) key[i] = 0u;
      }
    }
    int pick = -1;
    float prev = 0.0f, prev_err = 0.0f;
    // with scores as keys one more rank is looked at: the best expert left out
    const int steps = by_score ? p.top_k + 1 : p.top_k;
    for (int j = 0; j < steps && !unsure; ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int i = 1; i < VPT; ++i) best = key[i] > best ? key[i] : best;
      const uint32_t g = __reduce_max_sync(0xffffffffu, best);
      if (g == 0u) break;
      uint32_t at = 0x7fffffffu;
      float er = 0.0f;
#pragma unroll
      for (int i = VPT - 1; i >= 0; --i)
        if (key[i] == g) at = static_cast<uint32_t>(i * 32 + lane);
      const int e = static_cast<int>(__reduce_min_sync(0xffffffffu, at));
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (i * 32 + lane == e) {
          if (by_score) er = error_of(x[i], key_value(g));
          key[i] = 0u;
        }
      }
      if (by_score) {
        er = __shfl_sync(0xffffffffu, er, e & 31);
        const float c = key_value(g);
        if (j > 0 && !(prev - c > prev_err + er)) unsure = true;
        prev = c;
        prev_err = er;
      }
      if (lane == j && j < p.top_k) pick = e;
    }
    if (unsure) pick = choose_f64(p, row);

    // weights of the choices, lane j the j-th
    const bool on = lane < p.top_k && pick >= 0;
    const float xv = on ? route_logit(p, row, pick) : -INFINITY;
    float w = 0.0f;
    if (p.renormalize) {
      // only ratios matter, so both scores are divided by e^shift, which keeps the
      // sum away from zero: softmax  exp(x - shift), sigmoid exp(x - shift) / (1 + exp(x))
      const float big = warp_max(xv);
      float r;
      if (p.sigmoid) {
        const float shift = fminf(big, 0.0f);
        r = xv > 0.0f ? 1.0f / (1.0f + expf(-xv)) : expf(xv - shift) / (1.0f + expf(xv));
        if (xv != xv) r = xv;
      } else {
        r = expf(xv - big) + (z - z);  // a row whose scores are NaN has NaN weights
      }
      if (!on) r = 0.0f;
      w = r / warp_sum(r);
    } else {
      w = p.sigmoid ? 1.0f / (1.0f + expf(-xv)) : expf(xv - top) / z;
    }
    if (lane < p.top_k) {
      p.weights[row * p.top_k + lane] = on ? w * p.scale : 0.0f;
      p.chosen[row * p.top_k + lane] = pick;
    }
  }
}

// Gradient of the logits.  With g the gradient of the weights, r_j = s_j / sum(s)
// over the row's choices:
//   renormalised softmax   dx_j = scale r_j (g_j - sum g r)            others 0
//   renormalised sigmoid   dx_j = scale r_j (1 - s_j)(g_j - sum g r)   others 0
//   plain sigmoid          dx_j = scale g_j s_j (1 - s_j)              others 0
//   plain softmax          dx_e = s_e (scale g_e [e chosen] - scale sum_j g_j s_j)
// (the softmax's own normaliser cancels in the renormalised form), so only the last
// one reads whole rows; the others read k logits a row and write the row once.
// A choice that names an expert twice counts twice; one outside 0..experts-1 not at
// all.  The sums run in lane order of a fixed tree: the same bits every time.
template <int VPT>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteParams p) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  for (long long row = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
       row < p.rows; row += warps) {
    int e = -1;
    float g = 0.0f;
    if (lane < p.top_k) {
      e = p.picked[row * p.top_k + lane];
      g = p.grad_weights[row * p.top_k + lane];
    }
    float xv = -INFINITY;
    if (e >= 0 && e < p.experts) xv = route_logit(p, row, e);
    if (xv == -INFINITY) {  // masked, or no expert: no part in anything
      e = -1;
      g = 0.0f;
    }
    float x[VPT];
    float top = 0.0f, z = 1.0f;
    const bool dense = !p.sigmoid && !p.renormalize;
    if (dense) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = i * 32 + lane;
        x[i] = c < p.experts ? route_logit(p, row, c) : -INFINITY;
      }
      float m = x[0];
#pragma unroll
      for (int i = 1; i < VPT; ++i) m = fmaxf(m, x[i]);
      top = warp_max(m);
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        x[i] = x[i] == -INFINITY ? 0.0f : expf(x[i] - top);
        s += x[i];
      }
      z = warp_sum(s);
    }
    float d = 0.0f;      // what lane j adds to the gradient of its expert
    float common = 0.0f;  // dense: subtracted from every expert's
    if (p.renormalize) {
      const float big = warp_max(xv);
      float r, one_minus = 1.0f;
      if (p.sigmoid) {
        const float shift = fminf(big, 0.0f);
        r = xv > 0.0f ? 1.0f / (1.0f + expf(-xv)) : expf(xv - shift) / (1.0f + expf(xv));
        if (xv != xv) r = xv;
        one_minus = 1.0f / (1.0f + expf(xv));
      } else {
        r = expf(xv - big);
      }
      if (e < 0) r = 0.0f;
      const float total = warp_sum(r);
      if (e >= 0) r /= total;
      const float mean = warp_sum(g * r);
      if (e >= 0) d = p.scale * r * one_minus * (g - mean);
    } else if (p.sigmoid) {
      if (e >= 0) d = p.scale * g / (1.0f + expf(-xv)) / (1.0f + expf(xv));
    } else {
      const float s = e >= 0 ? expf(xv - top) / z : 0.0f;
      common = p.scale * warp_sum(g * s);
      d = p.scale * g;
    }
    float out[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) out[i] = 0.0f;
    for (int j = 0; j < p.top_k; ++j) {
      const int ej = __shfl_sync(0xffffffffu, e, j);
      const float dj = __shfl_sync(0xffffffffu, d, j);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (ej == i * 32 + lane) out[i] += dj;
    }
    if (dense) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) out[i] = x[i] == 0.0f ? 0.0f : x[i] / z * (out[i] - common);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = i * 32 + lane;
      if (c < p.experts) store_from_f32(p.grad, p.g_dtype, row * p.g_s0 + c * p.g_s1, out[i], 1);
    }
  }
}

}  // namespace kapyb
