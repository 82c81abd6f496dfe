// Routing of rows to experts: scores, choice of the top k, weights, and the
// gradient of the logits.
//
//   s = softmax(x) or sigmoid(x)        c = s + bias   (c only decides who is chosen)
//   w_j = scale * s_j [/ sum of the chosen s]
//
// One warp owns one row and keeps it in registers, every lane a run of VPT adjacent
// experts (one vector load), so the row is read once and only k weights and k indices
// leave the warp.  A lane ranks its own two best; a pick is one redux.sync over the
// lanes' best, and the lowest lane that has it wins, which is the rule for ties.  A lane
// whose two best are gone looks for its next two (about one row in two, once).
//
// Keys.  A choice between experts must not depend on how an exponential was rounded.
// Without a bias the order of the scores is the order of the logits, so the logits
// themselves are the keys, which is exact.  With a bias (or with groups ranked by a sum
// of two scores) c is formed in 32 bits with a bound on its error, and a row in which
// two neighbours of the ranking lie within that bound of one another is put in order
// again with the candidates' scores in 64 bits, one per lane; a row whose choice of
// groups is that close, or with more than 32 candidates, is decided afresh (choose_f64).
// On normally distributed logits that is one row in some thousand and ten thousand.
// The bound for a sigmoid: with e = ex2.approx of a rounded product the relative error
// of e is (|x| + 4) 2^-24, so s = 1 / (1 + e) is off by s (1 - s) (|x| + 4) 2^-24 for e
// and 4 s 2^-24 for the sum and the reciprocal: s (1 - s) |x| is below 0.23 and s (1 - s) 4
// at most 1, so 6 2^-24 covers it.
// For a softmax: s = e / z, e off by (d + 4) 2^-24 relative, d = max - x; z by the mean of
// that over the row, at most ln(1024) + 4, and 37 roundings of its sum; s is at most 1 / z
// and (d + 4) exp(-d) at most 4, so 64 2^-24 / z covers it.  The sum with the bias adds one
// rounding of c.
#pragma once

#include "common.cuh"
#include "ptx_sm100.cuh"

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
  int bias_pieces;    // bias starts on 16 bytes
  int sigmoid, top_k, n_groups, group_size, top_groups, group_best, renormalize;
  int group_lanes;    // lanes a group's experts fill, 0 unless whole lanes and a power of two
  float scale;
  float *weights;  // [rows, top_k]
  int32_t *chosen;  // [rows, top_k]
  // backward
  const int32_t *picked;      // [rows, top_k]
  const float *grad_weights;  // [rows, top_k]
  void *grad;
  long long g_s0, g_s1;
  int g_dtype;
  int vec_out;  // grad: unit stride, four experts at a time on aligned addresses
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
  const uint32_t high = static_cast<uint32_t>(v >> 32), top = __reduce_max_sync(0xffffffffu, high);
  const uint32_t low = __reduce_max_sync(0xffffffffu, high == top ? static_cast<uint32_t>(v) : 0u);
  return static_cast<unsigned long long>(top) << 32 | low;
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

// A lane's VPT experts lane * VPT ..; experts that do not exist read as masked.  VEC: the
// row has unit stride, VPT * element size alignment and a multiple of VPT experts.
template <int VPT, bool VEC>
__device__ __forceinline__ void load_row(const RouteParams &p, long long row, int lane, float (&x)[VPT]) {
  const int e0 = lane * VPT;
  if constexpr (VEC) {
    if (e0 >= p.experts) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) x[i] = -INFINITY;
      return;
    }
    if (p.x_dtype == KAPYB_F32) {
      const float *src = static_cast<const float *>(p.x) + row * p.x_s0 + e0;
      if constexpr (VPT == 2) {
        const float2 v = __ldg(reinterpret_cast<const float2 *>(src));
        x[0] = v.x;
        x[1] = v.y;
      } else {
#pragma unroll
        for (int i = 0; i < VPT / 4; ++i) {
          const float4 v = __ldg(reinterpret_cast<const float4 *>(src) + i);
          x[4 * i] = v.x;
          x[4 * i + 1] = v.y;
          x[4 * i + 2] = v.z;
          x[4 * i + 3] = v.w;
        }
      }
    } else {
      const uint16_t *src = static_cast<const uint16_t *>(p.x) + row * p.x_s0 + e0;
      uint32_t w[VPT / 2];
      if constexpr (VPT == 2) {
        w[0] = __ldg(reinterpret_cast<const uint32_t *>(src));
      } else if constexpr (VPT == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(src));
        w[0] = v.x;
        w[1] = v.y;
      } else {
#pragma unroll
        for (int i = 0; i < VPT / 8; ++i) {
          const uint4 v = __ldg(reinterpret_cast<const uint4 *>(src) + i);
          w[4 * i] = v.x;
          w[4 * i + 1] = v.y;
          w[4 * i + 2] = v.z;
          w[4 * i + 3] = v.w;
        }
      }
      if (p.x_dtype == KAPYB_BF16) {
#pragma unroll
        for (int i = 0; i < VPT / 2; ++i) unpack2_16<KAPYB_BF16>(w[i], x[2 * i], x[2 * i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < VPT / 2; ++i) unpack2_16<KAPYB_F16>(w[i], x[2 * i], x[2 * i + 1]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) x[i] = e0 + i < p.experts ? route_logit(p, row, e0 + i) : -INFINITY;
  }
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

// One expert's selection score in 64 bits; top and z as for 32 bits, in 64.
__device__ __forceinline__ double score_f64(const RouteParams &p, float x, int e, double top, double z) {
  const double xd = x;
  double c = p.sigmoid ? 1.0 / (1.0 + exp(-xd)) : exp(xd - top) / z;
  if (p.bias) c += static_cast<double>(p.bias[e]);
  return c;
}

// A row's largest logit and the sum of its exponentials, in 64 bits.
__device__ __forceinline__ void normaliser_f64(const RouteParams &p, long long row, int lane, double &top, double &z) {
  float m = -INFINITY;
  for (int e = lane; e < p.experts; e += 32) m = fmaxf(m, route_logit(p, row, e));
  top = warp_max(m);
  double s = 0.0;
#pragma unroll 1
  for (int e = lane; e < p.experts; e += 32) {
    const float x = route_logit(p, row, e);
    if (x != -INFINITY) s += exp(static_cast<double>(x) - top);
  }
  z = warp_sum64(s);
}

// Candidates of a row, lane j < n holding the j-th, in the order of their scores in 64
// bits: lane j gets the j-th of them.
__device__ __noinline__ int reorder_f64(const RouteParams &p, long long row, int n, int pick) {
  const int lane = threadIdx.x & 31;
  double top = 0.0, z = 1.0;
  if (!p.sigmoid) normaliser_f64(p, row, lane, top, z);
  unsigned long long key = 0ull;
  if (lane < n) key = rank_key64(score_f64(p, route_logit(p, row, pick), pick, top, z));
  int ahead = 0;
  for (int i = 0; i < n; ++i) {
    const unsigned long long k = __shfl_sync(0xffffffffu, key, i);
    const int e = __shfl_sync(0xffffffffu, pick, i);
    ahead += k > key || (k == key && e < pick);
  }
  int out = -1;
  for (int i = 0; i < n; ++i) {
    const int place = __shfl_sync(0xffffffffu, ahead, i), e = __shfl_sync(0xffffffffu, pick, i);
    if (place == lane) out = e;
  }
  return out;
}

// One row's choice with every score in 64 bits: lane j < top_k returns the j-th choice, or
// -1.  Rare, so its code is kept short: a lane's scores are formed one after the other.
template <int VPT>
__device__ __noinline__ int choose_f64(const RouteParams &p, long long row) {
  const int lane = threadIdx.x & 31;
  const int e0 = lane * VPT;
  unsigned long long key[VPT];  // rank of expert e0 + i, 0 when it is masked
  {
    double top = 0.0, z = 1.0;
    if (!p.sigmoid) normaliser_f64(p, row, lane, top, z);
#pragma unroll 1
    for (int i = 0; i < VPT; ++i) {
      const float x = e0 + i < p.experts ? route_logit(p, row, e0 + i) : -INFINITY;
      key[i] = x == -INFINITY ? 0ull : rank_key64(score_f64(p, x, e0 + i, top, z));
    }
  }
  auto value_of = [](unsigned long long k) -> double {
    if (k == 1ull) return __longlong_as_double(0x7fffffffffffffffll);
    return __longlong_as_double(static_cast<long long>(k >> 63 ? (k & 0x7fffffffffffffffull) : ~k));
  };
  if (p.n_groups > 1) {
    unsigned long long mine = 0ull;
    for (int q = 0; q < p.n_groups; ++q) {
      const int lo = q * p.group_size, hi = lo + p.group_size;
      unsigned long long k1 = 0ull, k2 = 0ull;  // this lane's two best of the group
#pragma unroll 1
      for (int i = 0; i < VPT; ++i) {
        const unsigned long long k = e0 + i >= lo && e0 + i < hi ? key[i] : 0ull;
        k2 = k > k1 ? k1 : k > k2 ? k : k2;
        k1 = k > k1 ? k : k1;
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
    const uint32_t kept = keep_groups(p, mine, lane);
#pragma unroll 1
    for (int i = 0; i < VPT; ++i)
      if (e0 + i < p.experts && !((kept >> ((e0 + i) / p.group_size)) & 1u)) key[i] = 0ull;
  }
  int pick = -1;
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long best = 0ull;
    int at = -1;
#pragma unroll 1
    for (int i = 0; i < VPT; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    const unsigned long long g = warp_max64(best);
    if (g == 0ull) break;
    const int w = __ffs(__ballot_sync(0xffffffffu, best == g)) - 1;
    const int i_w = __shfl_sync(0xffffffffu, at, w);
    if (lane == j) pick = w * VPT + i_w;
    if (lane == w) key[at] = 0ull;
  }
  return pick;
}

// A lane's two best of what is behind (bound, index) in the ranking (ALL: of everything).
struct LaneBest {
  uint32_t k1, k2;
  int i1, i2;
};
template <int VPT, bool ALL>
__device__ __forceinline__ LaneBest two_best(const uint32_t (&key)[VPT], uint32_t bound = 0u, int behind = 0) {
  LaneBest b{0u, 0u, 0, 0};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const uint32_t k = ALL || key[i] < bound || (key[i] == bound && i > behind) ? key[i] : 0u;
    const bool first = k > b.k1, second = k > b.k2;
    b.k2 = first ? b.k1 : second ? k : b.k2;
    b.i2 = first ? b.i1 : second ? i : b.i2;
    b.k1 = first ? k : b.k1;
    b.i1 = first ? i : b.i1;
  }
  return b;
}

// Approximations for the 32-bit selection scores only (their error is bounded above, and
// results below 2^-126, which they flush, are covered by its smallest term).
__device__ __forceinline__ float exp_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fmul_rn(x, 1.4426950408889634f)));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// rank_key of a number that is not NaN.
__device__ __forceinline__ uint32_t number_key(float c) {
  const int b = __float_as_int(c + 0.0f);
  return static_cast<uint32_t>(b ^ ((b >> 31) | static_cast<int>(0x80000000u)));
}

// Weights from full-precision expf and division, f32 throughout.  SCORED: experts (or
// groups) are ranked by their scores, not by their logits.  The kernel is bound by the
// instructions it issues (some 1450 a row of 256 experts in eight groups before, 70 % of
// the issue slots): rows without a mask, NaN or infinity take the short forms of the keys,
// the bias comes in 16-byte pieces, and a logit that served as key is its own copy.
template <int VPT, bool SCORED, bool VEC>
__global__ void __launch_bounds__(256) route_kernel(const RouteParams p) {
  ptx::griddep_launch();
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int e0 = lane * VPT;
  uint32_t key[VPT];
  float top = 0.0f, z = 1.0f, err = 0.0f;
  bool bad = false;  // a NaN or +inf among the logits: softmax weights are NaN
  {
    float x[VPT];
    load_row<VPT, VEC>(p, row, lane, x);
    float odd = 0.0f;  // NaN as soon as one of the logits is not finite
#pragma unroll
    for (int i = 0; i < VPT; ++i) odd = fmaf(x[i], 0.0f, odd);
    // (experts that do not exist read as masked, so a short last lane counts as odd)
    const bool plain = __all_sync(0xffffffffu, odd == odd);
    if (!plain) {
      bool off = false;
#pragma unroll
      for (int i = 0; i < VPT; ++i) off |= !(x[i] < INFINITY);
      bad = __any_sync(0xffffffffu, off);
    }
    if (!p.sigmoid && (SCORED || !p.renormalize)) {
      float m = x[0];
#pragma unroll
      for (int i = 1; i < VPT; ++i) m = fmaxf(m, x[i]);
      top = warp_max(m);
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) s += x[i] == -INFINITY ? 0.0f : kapy_exp(x[i] - top);
      z = warp_sum(s);
    }
    if constexpr (SCORED) {
      err = (p.sigmoid ? 6.0f : 64.0f / z) * 5.9604645e-8f + 1e-37f;
      float bias[VPT];
      if (p.bias != nullptr && VEC && p.bias_pieces) {
#pragma unroll
        for (int i = 0; i < VPT; i += 4) {
          const float4 v = e0 < p.experts ? __ldg(reinterpret_cast<const float4 *>(p.bias + e0 + i))
                                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          bias[i] = v.x;
          bias[i + 1] = v.y;
          if (VPT > 2) {
            bias[(i + 2) % VPT] = v.z;
            bias[(i + 3) % VPT] = v.w;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) bias[i] = p.bias != nullptr && e0 + i < p.experts ? __ldg(p.bias + e0 + i) : 0.0f;
      }
      float c[VPT];
      if (p.sigmoid) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) c[i] = rcp_fast(1.0f + exp_fast(-x[i])) + bias[i];
      } else {
        const float rz = 1.0f / z;
#pragma unroll
        for (int i = 0; i < VPT; ++i) c[i] = fmaf(exp_fast(x[i] - top), rz, bias[i]);
      }
      float nan = 0.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) nan = fmaf(c[i], 0.0f, nan);
      if (plain && __all_sync(0xffffffffu, nan == nan)) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) key[i] = number_key(c[i]);
      } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) key[i] = x[i] == -INFINITY ? 0u : rank_key(c[i]);
      }
    } else {
      if (plain) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) key[i] = number_key(x[i]);
      } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) key[i] = x[i] == -INFINITY ? 0u : rank_key(x[i]);
      }
    }
  }
  bool unsure = false;
  LaneBest b = two_best<VPT, true>(key);
  if (p.n_groups > 1) {
    uint32_t mine = 0u;
    float slack = 0.0f;  // error of this lane's group
    auto sum_key = [&](uint32_t g1, uint32_t g2, uint32_t &gk, float &ge) {
      gk = g1;
      ge = 0.0f;
      if (SCORED && g1 != 0u) {
        ge = err + fabsf(key_value(g1)) * 1.1920929e-7f;
        if (p.group_best == 2 && g2 != 0u) {
          const float sum = key_value(g1) + key_value(g2);
          ge += err + (fabsf(key_value(g2)) + fabsf(sum)) * 1.1920929e-7f;
          gk = rank_key(sum);
        }
      }
    };
    // lanes per group, when every lane's experts belong to one group
    const int lanes = p.group_lanes;
    if (lanes) {
      // every lane's two best belong to one group: join them over its lanes
      uint32_t k1 = b.k1, k2 = b.k2;
      for (int off = 1; off < lanes; off <<= 1) {
        const uint32_t o1 = __shfl_xor_sync(0xffffffffu, k1, off), o2 = __shfl_xor_sync(0xffffffffu, k2, off);
        k2 = max(min(k1, o1), max(k2, o2));
        k1 = max(k1, o1);
      }
      uint32_t gk;
      float ge;
      sum_key(k1, k2, gk, ge);
      const int from = lane * lanes;  // a lane of group `lane`
      mine = __shfl_sync(0xffffffffu, gk, from & 31);
      slack = __shfl_sync(0xffffffffu, ge, from & 31);
      if (lane >= p.n_groups) {
        mine = 0u;
        slack = 0.0f;
      }
    } else {
      for (int q = 0; q < p.n_groups; ++q) {
        const int lo = q * p.group_size - e0, hi = lo + p.group_size;
        uint32_t k1 = 0u, k2 = 0u;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const uint32_t k = i >= lo && i < hi ? key[i] : 0u;
          k2 = max(min(k, k1), k2);
          k1 = max(k1, k);
        }
        const uint32_t g1 = __reduce_max_sync(0xffffffffu, k1);
        const uint32_t owners = __ballot_sync(0xffffffffu, k1 == g1);
        const uint32_t g2 = __reduce_max_sync(0xffffffffu, lane == __ffs(owners) - 1 ? k2 : k1);
        uint32_t gk;
        float ge;
        sum_key(g1, g2, gk, ge);
        if (lane == q) {
          mine = gk;
          slack = ge;
        }
      }
    }
    const uint32_t kept = keep_groups(p, mine, lane);
    if (SCORED && p.top_groups < p.n_groups) {
      // the weakest kept group against the strongest one left out
      const bool in = (kept >> lane) & 1u;
      const uint32_t low = __reduce_min_sync(0xffffffffu, in ? mine : 0xffffffffu);
      const uint32_t high = __reduce_max_sync(0xffffffffu, in ? 0u : mine);
      // (errors are not negative, so their bits order like they do; a NaN is the largest)
      const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(slack) & 0x7fffffffu));
      if (kept != 0u && high != 0u) unsure = !(key_value(low) - key_value(high) > 2.0f * most);
    }
    if (lanes) {
      // all of a lane's experts are kept or none
      if (e0 < p.experts && !((kept >> (e0 / p.group_size)) & 1u)) {
        b = LaneBest{0u, 0u, 0, 0};
#pragma unroll
        for (int i = 0; i < VPT; ++i) key[i] = 0u;
      }
    } else {
      int q = e0 / p.group_size, next = (q + 1) * p.group_size - e0;  // group of expert e0 + i
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        while (i >= next) {
          ++q;
          next += p.group_size;
        }
        if (q < 32 && !((kept >> q) & 1u)) key[i] = 0u;
      }
      b = two_best<VPT, true>(key);
    }
  }
  int pick = -1;
  uint32_t pick_key = 0u;
  float prev = 0.0f, last = 0.0f;  // scores: of the pick before, and of the top_k-th
  bool spent = false;  // this lane's second best is its candidate already
  bool close = false;  // two neighbours are within the error of one another
  int found = 0;
  // c is clearly behind `above`: by more than both errors, 2 err + (|above| + |c|) 2^-23,
  // where |above| is at most |c| and the difference
  const float err2 = 2.1f * err;
  const auto apart = [&](float above, float c) { return above - c > fmaf(fabsf(c), 2.5e-7f, err2); };
  // with scores as keys the candidates go on until one is clearly behind the top_k-th
  for (int j = 0; j < (SCORED ? 32 : p.top_k) && !unsure; ++j) {
    const uint32_t g = __reduce_max_sync(0xffffffffu, b.k1);
    if (g == 0u) break;
    const int w = __ffs(__ballot_sync(0xffffffffu, b.k1 == g)) - 1;
    const int i_w = __shfl_sync(0xffffffffu, b.i1, w);
    if constexpr (SCORED) {
      const float c = key_value(g);
      if (j >= p.top_k && apart(last, c)) break;
      if (j > 0 && !apart(prev, c)) close = true;
      if (j == 31 && p.top_k <= 31) unsure = true;  // more candidates than lanes
      prev = c;
      if (j < p.top_k) last = c;
      found = j + 1;
    }
    if (lane == j) {
      pick = w * VPT + i_w;
      pick_key = g;
    }
    if (lane == w) {
      if (spent) {
        b = two_best<VPT, false>(key, g, i_w);
        spent = false;
      } else {
        b.k1 = b.k2;
        b.i1 = b.i2;
        spent = true;
      }
    }
    __syncwarp();
  }
  if constexpr (SCORED) {
    // 32 picks of a top 32: the one left out has not been looked at
    if (p.top_k == 32 && found == 32) {
      const uint32_t g = __reduce_max_sync(0xffffffffu, b.k1);
      if (g != 0u && !apart(last, key_value(g))) unsure = true;
    }
    if (unsure) pick = choose_f64<VPT>(p, row);
    else if (close) pick = reorder_f64(p, row, found, pick);
  }

  // weights of the choices, lane j the j-th
  const bool on = lane < p.top_k && pick >= 0;
  float xv = -INFINITY;
  if (on) xv = SCORED ? route_logit(p, row, pick) : key_value(pick_key);
  float w = 0.0f;
  if (p.renormalize) {
    // only ratios matter, so both scores are divided by e^shift, which keeps the sum away
    // from zero: softmax  exp(x - shift), sigmoid  exp(x - shift) / (1 + exp(x))
    const float big = warp_max(xv);
    float r;
    if (p.sigmoid) {
      const float shift = fminf(big, 0.0f);
      r = xv > 0.0f ? 1.0f / (1.0f + expf(-xv)) : expf(xv - shift) / (1.0f + expf(xv));
      if (xv != xv) r = xv;
    } else {
      r = bad ? __uint_as_float(0x7fffffffu) : expf(xv - big);
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

// Gradient of the logits.  With g the gradient of the weights, r_j = s_j / sum(s)
// over the row's choices:
//   renormalised softmax   dx_j = scale r_j (g_j - sum g r)            others 0
//   renormalised sigmoid   dx_j = scale r_j (1 - s_j)(g_j - sum g r)   others 0
//   plain sigmoid          dx_j = scale g_j s_j (1 - s_j)              others 0
//   plain softmax          dx_e = s_e (scale g_e [e chosen] - scale sum_j g_j s_j)
// (the softmax's own normaliser cancels in the renormalised form), so only the last
// one reads whole rows; the others read k logits a row and write the row once, put
// together in shared memory.  A choice that names an expert twice counts twice: its
// terms are summed in the order of the choices by the lane of its first mention.  One
// outside 0..experts-1 does not count.  No atomics: the same bits every time.
template <int VPT, bool VEC>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteParams p) {
  __shared__ __align__(16) float rows_mem[8][VPT * 32];
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  float *mem = rows_mem[threadIdx.x >> 5];
  int e = -1;
  float g = 0.0f;
  if (lane < p.top_k) {
    e = p.picked[row * p.top_k + lane];
    g = p.grad_weights[row * p.top_k + lane];
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) mem[i * 32 + lane] = 0.0f;
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
    load_row<VPT, VEC>(p, row, lane, x);
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
  float d = 0.0f;       // what lane j adds to the gradient of its expert
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
  float total_d = 0.0f;
  bool first = e >= 0;
  for (int j = 0; j < p.top_k; ++j) {
    const int ej = __shfl_sync(0xffffffffu, e, j);
    const float dj = __shfl_sync(0xffffffffu, d, j);
    if (ej == e) {
      total_d += dj;
      if (j < lane) first = false;
    }
  }
  __syncwarp();
  if (first) mem[e] = total_d;
  __syncwarp();
  if (dense) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      mem[lane * VPT + i] = x[i] == 0.0f ? 0.0f : x[i] / z * (mem[lane * VPT + i] - common);
    __syncwarp();
  }
  if (p.vec_out) {
    // four experts per lane and step: 16 bytes of f32, 8 of a 16-bit type
    for (int c = lane * 4; c < p.experts; c += 128) {
      const float4 v = *reinterpret_cast<const float4 *>(mem + c);
      if (p.g_dtype == KAPYB_F32) {
        __stcs(reinterpret_cast<float4 *>(static_cast<float *>(p.grad) + row * p.g_s0 + c), v);
      } else {
        uint2 w;
        if (p.g_dtype == KAPYB_BF16)
          w = make_uint2(cvt_pack2_t<KAPYB_BF16, 1>(v.x, v.y), cvt_pack2_t<KAPYB_BF16, 1>(v.z, v.w));
        else
          w = make_uint2(cvt_pack2_t<KAPYB_F16, 1>(v.x, v.y), cvt_pack2_t<KAPYB_F16, 1>(v.z, v.w));
        __stcs(reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.grad) + row * p.g_s0 + c), w);
      }
    }
  } else {
    for (int c = lane; c < p.experts; c += 32)
      store_from_f32(p.grad, p.g_dtype, row * p.g_s0 + c * p.g_s1, mem[c], 1);
  }
}

}  // namespace kapyb
