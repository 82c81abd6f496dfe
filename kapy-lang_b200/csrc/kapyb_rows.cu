// C ABI of the operators whose rows pick their weights (include/kapyb.h): argument
// checks, choice of kernel and launch.  The arithmetic lives in route.cuh,
// plan_rows.cuh, combine_rows.cuh, rows_simt.cuh and grouped_sm100.cuh.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>

#include "../../include/kapyb.h"
#include "adapters_sm100.cuh"
#include "combine_rows.cuh"
#include "context.cuh"
#include "grouped_sm100.cuh"
#include "plan_rows.cuh"
#include "route.cuh"
#include "rows_simt.cuh"

using namespace kapyb;

namespace {

// Launches go to the handle's device; the caller's current device comes back on the
// way out.
class OnDevice {
 public:
  explicit OnDevice(kapyb_handle h) {
    error_ = cudaGetDevice(&before_);
    if (error_ == cudaSuccess && before_ != h->device) {
      error_ = cudaSetDevice(h->device);
      moved_ = error_ == cudaSuccess;
    }
  }
  ~OnDevice() {
    if (moved_) cudaSetDevice(before_);
  }
  cudaError_t error() const { return error_; }

 private:
  int before_ = 0;
  bool moved_ = false;
  cudaError_t error_ = cudaSuccess;
};

// The arguments are checked before the handle, so that the checks need no GPU.
#define HAVE_HANDLE(h) \
  if (!h) return fail(nullptr, KAPYB_INVALID_ARG, "%s: NULL handle", call)

#define ON_DEVICE(h)       \
  HAVE_HANDLE(h);          \
  OnDevice on_device_(h);  \
  CUDA_TRY(h, on_device_.error())

#define TRY(expr)                          \
  do {                                     \
    const kapyb_status st_ = (expr);       \
    if (st_ != KAPYB_OK) return st_;       \
  } while (0)

// Lets a kernel use `bytes` of dynamic shared memory, once per device.
template <auto Kernel>
kapyb_status allow_smem(kapyb_handle h, int bytes) {
  static std::atomic<bool> done[kMaxDevices];
  if (!done[h->device].load()) {
    CUDA_TRY(h, cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done[h->device].store(true);
  }
  return KAPYB_OK;
}

kapyb_status launched(kapyb_handle h, const char *name) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(h, KAPYB_CUDA_ERROR, "%s: launch failed: %s", name, cudaGetErrorString(e));
  h->last_kernel = name;
  h->launches += 1;
  return KAPYB_OK;
}

constexpr int32_t kMaxSize = 1 << 30;  // rows and columns: the kernels' index arithmetic adds to them

bool empty(const kapyb_tensor2d *t) { return t->size0 == 0 || t->size1 == 0; }

kapyb_status check_tensor(kapyb_handle h, const char *call, const char *what, const kapyb_tensor2d *t) {
  if (!t) return fail(h, KAPYB_INVALID_ARG, "%s: %s is NULL", call, what);
  if (t->size0 < 0 || t->size1 < 0 || t->stride0 < 0 || t->stride1 < 0 || t->offset_elems < 0)
    return fail(h, KAPYB_INVALID_ARG, "%s: %s has a negative size, stride or offset", call, what);
  if (t->size0 > kMaxSize || t->size1 > kMaxSize)
    return fail(h, KAPYB_UNSUPPORTED, "%s: %s has more than 2^30 rows or columns", call, what);
  if (!valid_dtype(t->dtype))
    return fail(h, KAPYB_INVALID_ARG, "%s: %s must have f16, bf16 or f32 element type", call, what);
  if (!t->ptr && !empty(t)) return fail(h, KAPYB_INVALID_ARG, "%s: %s has no data pointer", call, what);
  if (reinterpret_cast<uintptr_t>(t->ptr) % dtype_size(t->dtype) != 0)
    return fail(h, KAPYB_INVALID_ARG, "%s: %s is not aligned to its element size", call, what);
  if (!valid_cache(t->cache))
    return fail(h, KAPYB_INVALID_ARG, "%s: %s has an unknown cache operator or eviction priority", call, what);
  return KAPYB_OK;
}

kapyb_status check_output(kapyb_handle h, const char *call, const char *what, const kapyb_tensor2d *t) {
  const kapyb_status st = check_tensor(h, call, what, t);
  if (st != KAPYB_OK) return st;
  // two elements of an output must not share an address
  const bool a = t->size0 > 1 && t->stride0 == 0, b = t->size1 > 1 && t->stride1 == 0;
  if (a || b) return fail(h, KAPYB_INVALID_ARG, "%s: %s has a stride of 0", call, what);
  return KAPYB_OK;
}

bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// First and last byte behind a descriptor repeated `batch` times.
struct Span {
  uintptr_t lo, hi;
};
Span span_of(const kapyb_tensor2d *t, int64_t batch = 1, int64_t batch_stride = 0) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(elem_ptr(t));
  if (empty(t) || batch == 0) return {lo, lo};
  const int64_t last = (t->size0 - 1ll) * t->stride0 + (t->size1 - 1ll) * t->stride1 + (batch - 1) * batch_stride;
  return {lo, lo + static_cast<uintptr_t>(last + 1) * dtype_size(t->dtype)};
}
Span span_of(const void *p, size_t bytes) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  return {lo, p ? lo + bytes : lo};
}
bool meet(const Span &a, const Span &b) { return a.lo < a.hi && b.lo < b.hi && a.lo < b.hi && b.lo < a.hi; }

bool rounding_ok(int r) { return r == KAPYB_RZ || r == KAPYB_RN; }

kapyb_status check_epilogue(kapyb_handle h, const char *call, const kapyb_epilogue *ep) {
  if (!ep) return KAPYB_OK;
  if (ep->bias && !valid_dtype(ep->bias_dtype))
    return fail(h, KAPYB_INVALID_ARG, "%s: bias must have f16, bf16 or f32 element type", call);
  if (ep->bias_axis != 0 && ep->bias_axis != 1) return fail(h, KAPYB_INVALID_ARG, "%s: bias_axis must be 0 or 1", call);
  if (ep->activation < KAPYB_ACT_NONE || ep->activation > KAPYB_ACT_SILU)
    return fail(h, KAPYB_INVALID_ARG, "%s: unknown activation %d", call, ep->activation);
  if (!rounding_ok(ep->rounding))
    return fail(h, KAPYB_INVALID_ARG, "%s: rounding mode must be set for down cast", call);
  return KAPYB_OK;
}

const kapyb_epilogue kPlainEpilogue = {1.0f, nullptr, KAPYB_F32, 1, KAPYB_ACT_NONE, KAPYB_RN};

// Launches.  A step is a chain of short kernels, so plan, products, weighted sums and the
// adapters' second kernels are launched with programmatic serialization: they are set up
// while the kernel in front ends, and every one of them waits for its end
// (griddepcontrol.wait) before it reads or writes what another kernel may hold.  Each such
// kernel has a thread that waits, so one that has ended vouches for all in front of it.
// (In replayed graphs: plan and product of 5331 rows 30.3 -> 28.6 us; a layer of one token x 2
// of 8 experts 29.8 -> 29.0, 64 x 2 of 8 32.7 -> 32.5, 512 x 2 of 16 65.3 -> 64.4; adapters of
// one row 14.5 -> 11.4.)

// ------------------------------------------------------------------- routing

kapyb_status check_routing(kapyb_handle h, const char *call, const kapyb_tensor2d *logits, const kapyb_routing *r) {
  if (!r) return fail(h, KAPYB_INVALID_ARG, "%s: routing is NULL", call);
  const int experts = logits->size1;
  if (experts < 1 || experts > kRouteMaxExperts)
    return fail(h, experts < 1 ? KAPYB_INVALID_ARG : KAPYB_UNSUPPORTED, "%s: 1 to %d experts (got %d)", call,
                kRouteMaxExperts, experts);
  if (r->score != KAPYB_SCORE_SOFTMAX && r->score != KAPYB_SCORE_SIGMOID)
    return fail(h, KAPYB_INVALID_ARG, "%s: unknown score %d", call, r->score);
  if (r->top_k < 1 || r->top_k > kRouteMaxTopK || r->top_k > experts)
    return fail(h, KAPYB_INVALID_ARG, "%s: top_k must be 1 to %d and at most the number of experts (got %d of %d)",
                call, kRouteMaxTopK, r->top_k, experts);
  if (r->n_groups < 1 || r->n_groups > kRouteMaxGroups || experts % r->n_groups != 0)
    return fail(h, KAPYB_INVALID_ARG, "%s: n_groups must be 1 to %d and divide the number of experts (got %d of %d)",
                call, kRouteMaxGroups, r->n_groups, experts);
  if (r->top_groups < 1 || r->top_groups > r->n_groups)
    return fail(h, KAPYB_INVALID_ARG, "%s: top_groups must be 1 to n_groups (got %d of %d)", call, r->top_groups,
                r->n_groups);
  if (r->group_best != 1 && r->group_best != 2)
    return fail(h, KAPYB_INVALID_ARG, "%s: group_best must be 1 or 2 (got %d)", call, r->group_best);
  return KAPYB_OK;
}

RouteParams route_params(const kapyb_tensor2d *logits, const kapyb_routing *r) {
  RouteParams p{};
  p.x = elem_ptr(logits);
  p.x_s0 = logits->stride0;
  p.x_s1 = logits->stride1;
  p.x_dtype = logits->dtype;
  p.rows = logits->size0;
  p.experts = logits->size1;
  p.sigmoid = r->score == KAPYB_SCORE_SIGMOID;
  p.top_k = r->top_k;
  p.n_groups = r->n_groups;
  p.group_size = logits->size1 / r->n_groups;
  p.top_groups = r->top_groups;
  p.group_best = r->group_best;
  p.renormalize = r->renormalize != 0;
  p.scale = r->scale;
  return p;
}

// Experts per lane, rounded up to a compiled width; VEC: a lane's experts are one aligned
// run that exists as a whole.
template <int VPT>
bool row_vec_ok(const RouteParams &p) {
  const int64_t esz = dtype_size(p.x_dtype);
  const int64_t align = std::min<int64_t>(16, VPT * esz);
  return p.x_s1 == 1 && p.experts % VPT == 0 && reinterpret_cast<uintptr_t>(p.x) % align == 0 &&
         (p.x_s0 * esz) % align == 0;
}
template <int VPT>
void launch_route(RouteParams p, int grid, cudaStream_t s) {
  const int lanes = p.group_size / VPT;
  p.group_lanes = lanes * VPT == p.group_size && (lanes & (lanes - 1)) == 0 && lanes <= 32 ? lanes : 0;
  p.bias_pieces = VPT % 4 == 0 && aligned16(p.bias);
  const bool scored = p.bias != nullptr || (p.n_groups > 1 && p.group_best > 1);
  const bool vec = row_vec_ok<VPT>(p);
  if (scored && vec) route_kernel<VPT, true, true><<<grid, 256, 0, s>>>(p);
  else if (scored) route_kernel<VPT, true, false><<<grid, 256, 0, s>>>(p);
  else if (vec) route_kernel<VPT, false, true><<<grid, 256, 0, s>>>(p);
  else route_kernel<VPT, false, false><<<grid, 256, 0, s>>>(p);
}
template <int VPT>
void launch_route_backward(const RouteParams &p, int grid, cudaStream_t s) {
  if (row_vec_ok<VPT>(p)) route_backward_kernel<VPT, true><<<grid, 256, 0, s>>>(p);
  else route_backward_kernel<VPT, false><<<grid, 256, 0, s>>>(p);
}

int warp_grid(int rows) { return static_cast<int>((rows + 7ll) / 8); }

}  // namespace

extern "C" KAPYB_API kapyb_status kapyb_route(kapyb_handle h, const kapyb_tensor2d *logits, const float *bias,
                                              const kapyb_routing *routing, float *weights, int32_t *experts,
                                              void *stream) {
  const char *call = "route";
  TRY(check_tensor(h, "route", "logits", logits));
  TRY(check_routing(h, "route", logits, routing));
  if (logits->size0 == 0) {
    HAVE_HANDLE(h);
    return KAPYB_OK;
  }
  if (!weights || !experts) return fail(h, KAPYB_INVALID_ARG, "route: weights or experts is NULL");
  if (!aligned4(weights) || !aligned4(experts) || !aligned4(bias))
    return fail(h, KAPYB_INVALID_ARG, "route: bias, weights and experts must be 4-byte aligned");
  const size_t bytes = static_cast<size_t>(logits->size0) * routing->top_k * 4;
  const Span w = span_of(weights, bytes), e = span_of(experts, bytes), x = span_of(logits),
             b = span_of(bias, static_cast<size_t>(logits->size1) * 4);
  if (meet(w, e) || meet(w, x) || meet(e, x) || meet(w, b) || meet(e, b))
    return fail(h, KAPYB_INVALID_ARG, "route: an output overlaps another tensor of the call");
  ON_DEVICE(h);
  RouteParams p = route_params(logits, routing);
  p.bias = bias;
  p.weights = weights;
  p.chosen = experts;
  const int grid = warp_grid(p.rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.experts <= 64) launch_route<2>(p, grid, s);
  else if (p.experts <= 128) launch_route<4>(p, grid, s);
  else if (p.experts <= 256) launch_route<8>(p, grid, s);
  else if (p.experts <= 512) launch_route<16>(p, grid, s);
  else launch_route<32>(p, grid, s);
  return launched(h, "route");
}

extern "C" KAPYB_API kapyb_status kapyb_route_backward(kapyb_handle h, const kapyb_tensor2d *logits,
                                                       const kapyb_routing *routing, const int32_t *experts,
                                                       const float *grad_weights, const kapyb_tensor2d *grad_logits,
                                                       void *stream) {
  const char *call = "route_backward";
  TRY(check_tensor(h, "route_backward", "logits", logits));
  TRY(check_routing(h, "route_backward", logits, routing));
  TRY(check_output(h, "route_backward", "grad_logits", grad_logits));
  if (grad_logits->size0 != logits->size0 || grad_logits->size1 != logits->size1)
    return fail(h, KAPYB_INVALID_ARG, "route_backward: grad_logits must have the shape of logits");
  if (logits->size0 == 0) {
    HAVE_HANDLE(h);
    return KAPYB_OK;
  }
  if (!experts || !grad_weights) return fail(h, KAPYB_INVALID_ARG, "route_backward: experts or grad_weights is NULL");
  if (!aligned4(experts) || !aligned4(grad_weights))
    return fail(h, KAPYB_INVALID_ARG, "route_backward: experts and grad_weights must be 4-byte aligned");
  const size_t bytes = static_cast<size_t>(logits->size0) * routing->top_k * 4;
  const Span out = span_of(grad_logits);
  if (meet(out, span_of(logits)) || meet(out, span_of(experts, bytes)) || meet(out, span_of(grad_weights, bytes)))
    return fail(h, KAPYB_INVALID_ARG, "route_backward: grad_logits overlaps an input");
  ON_DEVICE(h);
  RouteParams p = route_params(logits, routing);
  p.picked = experts;
  p.grad_weights = grad_weights;
  p.grad = const_cast<void *>(elem_ptr(grad_logits));
  p.g_s0 = grad_logits->stride0;
  p.g_s1 = grad_logits->stride1;
  p.g_dtype = grad_logits->dtype;
  const int64_t esz = dtype_size(p.g_dtype);
  p.vec_out = p.g_s1 == 1 && p.experts % 4 == 0 && p.g_s0 % 4 == 0 &&
              reinterpret_cast<uintptr_t>(p.grad) % (4 * esz) == 0;
  const int grid = warp_grid(p.rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.experts <= 64) launch_route_backward<2>(p, grid, s);
  else if (p.experts <= 128) launch_route_backward<4>(p, grid, s);
  else if (p.experts <= 256) launch_route_backward<8>(p, grid, s);
  else if (p.experts <= 512) launch_route_backward<16>(p, grid, s);
  else launch_route_backward<32>(p, grid, s);
  return launched(h, "route_backward");
}

// ---------------------------------------------------------------------- plan

namespace {

kapyb_status launch_plan(kapyb_handle h, const PlanParams &p, cudaStream_t stream) {
  const size_t smem = plan_smem_bytes(p.groups);
  TRY(allow_smem<plan_rows_kernel>(h, static_cast<int>(plan_smem_bytes(kPlanMaxGroups + 1))));
  // A warp's piece is a whole number of 32-entry steps.  One CTA takes up to two steps a
  // warp; beyond that the work is spread over the cluster.
  int ctas = 1;
  while (ctas < kPlanMaxCtas && static_cast<long long>(p.n) > ctas * kPlanWarps * 64ll) ctas *= 2;
  if (ctas > 8)
    CUDA_TRY(h, cudaFuncSetAttribute(plan_rows_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(ctas, 1, 1);
  cfg.blockDim = dim3(kPlanWarps * 32, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  CUDA_TRY(h, cudaLaunchKernelEx(&cfg, plan_rows_kernel, p));
  return launched(h, "plan_rows");
}

}  // namespace

extern "C" KAPYB_API kapyb_status kapyb_plan_rows(kapyb_handle h, const int32_t *index, int32_t n, int32_t groups,
                                                  int32_t *order, int32_t *offsets, int32_t *slots, void *stream) {
  const char *call = "plan_rows";
  if (n < 0) return fail(h, KAPYB_INVALID_ARG, "plan_rows: n is negative");
  if (groups < 1 || groups > kPlanMaxGroups)
    return fail(h, groups < 1 ? KAPYB_INVALID_ARG : KAPYB_UNSUPPORTED, "plan_rows: 1 to %d groups (got %d)",
                kPlanMaxGroups, groups);
  if (!offsets || (n > 0 && (!index || !order)))
    return fail(h, KAPYB_INVALID_ARG, "plan_rows: index, order or offsets is NULL");
  if (!aligned4(index) || !aligned4(order) || !aligned4(offsets) || !aligned4(slots))
    return fail(h, KAPYB_INVALID_ARG, "plan_rows: arrays must be 4-byte aligned");
  const size_t bytes = static_cast<size_t>(n) * 4;
  const Span s[4] = {span_of(index, bytes), span_of(order, bytes), span_of(offsets, (groups + 1ull) * 4),
                     span_of(slots, bytes)};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (meet(s[i], s[j])) return fail(h, KAPYB_INVALID_ARG, "plan_rows: two arrays of the call overlap");
  ON_DEVICE(h);
  return launch_plan(h, PlanParams{index, n, groups, order, offsets, slots, n, 1, 0},
                     static_cast<cudaStream_t>(stream));
}

// ------------------------------------------------------------------- products

namespace {

constexpr int kMaxRowGroups = kGroupedMaxGroups;

// 2-D map over 16-bit rows of `inner` unit-stride elements, boxes of 64 elements x box_rows.
kapyb_status make_row_tmap(kapyb_handle h, CUtensorMap *map, const void *base, int dtype, uint64_t inner,
                           uint64_t rows, uint64_t ld, uint32_t box_rows) {
  cuuint64_t dims[2] = {inner, rows};
  cuuint64_t strides[1] = {ld * 2};
  cuuint32_t box[2] = {64, box_rows}, step[2] = {1, 1};
  const CUresult r = h->encode(map, tmap_dtype(dtype), 2, const_cast<void *>(base), dims, strides, box, step,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(h, KAPYB_CUDA_ERROR, "cuTensorMapEncodeTiled failed (%d): rows of %llu, %llu of them, ld %llu", (int)r,
                (unsigned long long)inner, (unsigned long long)rows, (unsigned long long)ld);
  return KAPYB_OK;
}

bool half_type(int dtype) { return dtype == KAPYB_F16 || dtype == KAPYB_BF16; }

constexpr int64_t kMaxRowPitch = 1 << 26;  // bytes between output rows on the tcgen05 paths

// Two neighbouring 16-bit columns of the output may be written as one aligned word, four
// f32 ones as 16 bytes.
bool wide_stores_ok(const void *out, int dtype, int64_t s0, int64_t group) {
  const int64_t n = half_type(dtype) ? 2 : 4;
  return reinterpret_cast<uintptr_t>(out) % (n * dtype_size(dtype)) == 0 && s0 % n == 0 && group % n == 0;
}

PairParams pair_params(const GroupedParams &gp, const kapyb_tensor2d *lhs, bool gather) {
  PairParams pp{};
  pp.g = gp;
  pp.gather = gather;
  pp.lhs = static_cast<const uint8_t *>(elem_ptr(lhs));
  pp.lhs_pitch = lhs->stride0 * 2ll;
  pp.div_fan = FastDiv::make(static_cast<uint32_t>(gp.fan));
  pp.entries = static_cast<uint32_t>(std::min<int64_t>(static_cast<int64_t>(gp.src_rows) * gp.fan, 1ll << 31));
  return pp;
}

// The pair kernel: `tiles` pairs of CTAs at most, as many as the device holds at once
// (the tile loop is statically strided).
template <int MODE>
kapyb_status launch_pairs(kapyb_handle h, const CUtensorMap &tmA, const CUtensorMap &tmB, const CUtensorMap &tmR,
                          const CUtensorMap &tmU, const PairParams &pp, long long tiles, cudaStream_t stream) {
  using Cfg = PairCfg;
  auto kern = grouped_pair_kernel<MODE>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see "Launches" above
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static std::atomic<int> resident[kMaxDevices];  // 0: not asked yet
  int pairs = resident[h->device].load();
  if (pairs == 0) {
    CUDA_TRY(h, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
    cfg.gridDim = dim3(2 * (h->sm_count / 2), 1, 1);
    if (cudaOccupancyMaxActiveClusters(&pairs, kern, &cfg) != cudaSuccess || pairs < 1) {
      cudaGetLastError();
      pairs = h->sm_count / 2;
    }
    pairs = std::min(pairs, h->sm_count / 2);
    resident[h->device].store(pairs);
  }
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min<long long>(tiles, pairs)), 1, 1);
  cfg.numAttrs = 2;
  CUDA_TRY(h, cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmR, tmU, pp));
  return launched(h, MODE == PAIR_GRADIENT   ? "grouped_grad_pair"
                     : MODE == PAIR_ADAPTERS ? "adapters_pair"
                                             : "grouped_pair");
}

// Rows of lhs as TMA can fetch them: 16-bit, unit stride along K, 16-byte rows.
bool rows_tma_ok(const kapyb_tensor2d *t) {
  return half_type(t->dtype) && t->stride1 == 1 && tma_ok(elem_ptr(t), t->dtype, t->size1, t->size0, t->stride0, 1, 0);
}

// The tensor-core path of kapyb_matmul_grouped; *taken = false when the operands are
// not for it.
kapyb_status grouped_on_tcgen05(kapyb_handle h, const kapyb_tensor2d *lhs, const kapyb_tensor2d *rhs, int groups,
                                int64_t group_stride, const int32_t *offsets, const int32_t *order, int fan,
                                const kapyb_tensor2d *out, const kapyb_epilogue &ep, bool gated, cudaStream_t stream,
                                bool *taken) {
  *taken = false;
  if (!rows_tma_ok(lhs) || out->stride1 != 1) return KAPYB_OK;
  const int64_t pitch = static_cast<int64_t>(out->stride0) * dtype_size(out->dtype);
  if (pitch >= kMaxRowPitch) return KAPYB_OK;
  const bool mn = rhs->stride1 == 1;
  if (!mn && rhs->stride0 != 1) return KAPYB_OK;
  const int64_t unit = mn ? rhs->size1 : rhs->size0, other = mn ? rhs->size0 : rhs->size1;
  const int64_t ld = mn ? rhs->stride0 : rhs->stride1;
  if (!tma_ok(elem_ptr(rhs), rhs->dtype, unit, other, ld, groups, group_stride)) return KAPYB_OK;
  // the up columns' tiles start at column cols: a TMA start on 16 bytes
  if (gated && mn && out->size1 % 8 != 0) return KAPYB_OK;
  GroupedParams gp{};
  gp.groups = groups;
  gp.rows = out->size0;
  gp.cols = out->size1;
  gp.K = lhs->size1;
  gp.n_tiles = gated ? (gp.cols + 127) / 128 : (gp.cols + 255) / 256;
  gp.num_kb = (gp.K + 63) / 64;
  gp.offsets = offsets;
  gp.order = order;
  gp.fan = order ? fan : 1;
  gp.src_rows = lhs->size0;
  gp.a_mn_major = mn;
  gp.bf16 = lhs->dtype == KAPYB_BF16;
  gp.out = const_cast<void *>(elem_ptr(out));
  gp.row_pitch = static_cast<uint32_t>(pitch);
  gp.out_dtype = out->dtype;
  gp.wide_stores = wide_stores_ok(gp.out, out->dtype, out->stride0, 0);
  gp.alpha = ep.alpha;
  gp.bias = ep.bias;
  gp.bias_dtype = ep.bias_dtype;
  gp.bias_cols = rhs->size1;
  gp.activation = ep.activation;
  gp.rounding = ep.rounding;
  gp.status = h->status;
  gp.wait_limit_us = h->wait_limit_us;
  const long long busy = std::min(groups, gp.rows);
  const long long tiles = ((gp.rows + PairCfg::BT - 1ll) / PairCfg::BT + busy) * gp.n_tiles;
  if (tiles >= (1ll << 30)) return KAPYB_OK;
  const int64_t lhs_ld = lhs->size0 > 1 ? lhs->stride0 : (lhs->size1 + 7) / 8 * 8;
  CUtensorMap tmA;
  TRY(make_tmap(h, &tmA, elem_ptr(rhs), rhs->dtype, unit, other, groups, ld, group_stride, 64, mn || gated ? 64 : 128));
  CUtensorMap box[3] = {tmA, tmA, tmA};  // rows in plan order come in boxes of 128, 64 and 32, others without
  for (int i = 0; i < 3 && !order; ++i)
    TRY(make_row_tmap(h, &box[i], elem_ptr(lhs), lhs->dtype, lhs->size1, lhs->size0, lhs_ld, 128 >> i));
  *taken = true;
  const PairParams pp = pair_params(gp, lhs, order != nullptr);
  return gated ? launch_pairs<PAIR_GATED>(h, tmA, box[0], box[1], box[2], pp, tiles, stream)
               : launch_pairs<PAIR_FORWARD>(h, tmA, box[0], box[1], box[2], pp, tiles, stream);
}

kapyb_status grouped_grad_on_tcgen05(kapyb_handle h, const kapyb_tensor2d *lhs, const kapyb_tensor2d *grad,
                                     int groups, const int32_t *offsets, const int32_t *order, int fan,
                                     const kapyb_tensor2d *out, int64_t out_group_stride, float alpha, int rounding,
                                     cudaStream_t stream, bool *taken) {
  *taken = false;
  if (!rows_tma_ok(lhs) || !rows_tma_ok(grad) || out->stride1 != 1) return KAPYB_OK;
  const int64_t pitch = static_cast<int64_t>(out->stride0) * dtype_size(out->dtype);
  if (pitch >= kMaxRowPitch) return KAPYB_OK;
  GroupedParams gp{};
  gp.groups = groups;
  gp.rows = grad->size0;
  gp.cols = out->size1;
  gp.K = out->size0;
  gp.n_tiles = (gp.cols + 255) / 256;
  gp.k_tiles = (gp.K + 255) / 256;
  gp.offsets = offsets;
  gp.order = order;
  gp.fan = order ? fan : 1;
  gp.src_rows = lhs->size0;
  gp.bf16 = lhs->dtype == KAPYB_BF16;
  gp.out = const_cast<void *>(elem_ptr(out));
  gp.row_pitch = static_cast<uint32_t>(pitch);
  gp.group_bytes = groups > 1 ? out_group_stride * dtype_size(out->dtype) : 0;
  gp.out_dtype = out->dtype;
  gp.wide_stores = wide_stores_ok(gp.out, out->dtype, out->stride0, groups > 1 ? out_group_stride : 0);
  gp.alpha = alpha;
  gp.activation = KAPYB_ACT_NONE;
  gp.rounding = rounding;
  gp.status = h->status;
  gp.wait_limit_us = h->wait_limit_us;
  const long long tiles = static_cast<long long>(groups) * gp.n_tiles * gp.k_tiles;
  if (tiles >= (1ll << 30)) return KAPYB_OK;
  CUtensorMap tmA;
  TRY(make_row_tmap(h, &tmA, elem_ptr(grad), grad->dtype, grad->size1, grad->size0,
                    grad->size0 > 1 ? grad->stride0 : (grad->size1 + 7) / 8 * 8, 64));
  *taken = true;
  PairParams pp = pair_params(gp, lhs, true);
  pp.grad = static_cast<const uint8_t *>(elem_ptr(grad));
  pp.grad_pitch = grad->stride0 * 2ll;
  pp.piece_kb = out->dtype == KAPYB_F32 ? 16 : 1 << 30;
  return launch_pairs<PAIR_GRADIENT>(h, tmA, tmA, tmA, tmA, pp, tiles, stream);
}

// What the two grouped products check alike.
kapyb_status check_grouped(kapyb_handle h, const char *call, const kapyb_tensor2d *lhs, const kapyb_tensor2d *other,
                           int groups, const int32_t *offsets, const int32_t *order, int fan) {
  if (lhs->dtype != other->dtype)
    return fail(h, KAPYB_INVALID_ARG, "%s: operands must have same element type", call);
  if (lhs->padding != KAPYB_PAD_ZERO || other->padding != KAPYB_PAD_ZERO)
    return fail(h, KAPYB_UNSUPPORTED, "%s: operands are padded with zeros only", call);
  if (groups < 1 || groups > kMaxRowGroups)
    return fail(h, groups < 1 ? KAPYB_INVALID_ARG : KAPYB_UNSUPPORTED, "%s: 1 to %d groups (got %d)", call,
                kMaxRowGroups, groups);
  if (!offsets) return fail(h, KAPYB_INVALID_ARG, "%s: offsets is NULL", call);
  if (order && fan < 1) return fail(h, KAPYB_INVALID_ARG, "%s: fan must be at least 1", call);
  if (!aligned4(offsets) || !aligned4(order))
    return fail(h, KAPYB_INVALID_ARG, "%s: offsets and order must be 4-byte aligned", call);
  return KAPYB_OK;
}

}  // namespace

extern "C" KAPYB_API kapyb_status kapyb_matmul_grouped(kapyb_handle h, const kapyb_tensor2d *lhs,
                                                       const kapyb_tensor2d *rhs, int32_t groups,
                                                       int64_t group_stride, const int32_t *offsets,
                                                       const int32_t *order, int32_t fan, const kapyb_tensor2d *out,
                                                       const kapyb_epilogue *epilogue, int32_t gated, void *stream) {
  const char *call = "matmul_grouped";
  TRY(check_tensor(h, call, "lhs", lhs));
  TRY(check_tensor(h, call, "rhs", rhs));
  TRY(check_output(h, call, "out", out));
  TRY(check_grouped(h, call, lhs, rhs, groups, offsets, order, fan));
  TRY(check_epilogue(h, call, epilogue));
  if (epilogue && epilogue->bias && epilogue->bias_axis != 1)
    return fail(h, KAPYB_UNSUPPORTED, "%s: bias_axis must be 1 (one value per column of each group)", call);
  if (group_stride < 0) return fail(h, KAPYB_INVALID_ARG, "%s: group_stride is negative", call);
  if (lhs->size1 != rhs->size0)
    return fail(h, KAPYB_INVALID_ARG, "%s: number of columns of lhs must be equal to number of rows of rhs", call);
  const int64_t cols_w = static_cast<int64_t>(out->size1) * (gated ? 2 : 1);
  if (rhs->size1 != cols_w)
    return fail(h, KAPYB_INVALID_ARG, "%s: rhs must have %s columns of out", call, gated ? "twice the" : "the");
  if (!order && lhs->size0 != out->size0)
    return fail(h, KAPYB_INVALID_ARG, "%s: without order lhs must have as many rows as out", call);
  if (empty(out)) {
    HAVE_HANDLE(h);
    return KAPYB_OK;
  }
  const Span o = span_of(out);
  if (meet(o, span_of(lhs)) || meet(o, span_of(rhs, groups, group_stride)) ||
      meet(o, span_of(offsets, (groups + 1ull) * 4)) || meet(o, span_of(order, order ? out->size0 * 4ull : 0)) ||
      (epilogue && meet(o, span_of(epilogue->bias, groups * cols_w * dtype_size(epilogue->bias_dtype)))))
    return fail(h, KAPYB_INVALID_ARG, "%s: out overlaps an input", call);
  ON_DEVICE(h);
  const kapyb_epilogue &ep = epilogue ? *epilogue : kPlainEpilogue;
  bool taken = false;
  const kapyb_status st = grouped_on_tcgen05(h, lhs, rhs, groups, group_stride, offsets, order, fan, out, ep,
                                             gated != 0, static_cast<cudaStream_t>(stream), &taken);
  if (taken || st != KAPYB_OK) return st;
  RowsSimtParams p{};
  p.x = elem_ptr(lhs);
  p.x_s0 = lhs->stride0;
  p.x_s1 = lhs->stride1;
  p.src_rows = lhs->size0;
  p.w = elem_ptr(rhs);
  p.w_s0 = rhs->stride0;
  p.w_s1 = rhs->stride1;
  p.w_group = group_stride;
  p.in_dtype = lhs->dtype;
  p.groups = groups;
  p.rows = out->size0;
  p.K = lhs->size1;
  p.cols = out->size1;
  p.cols_w = rhs->size1;
  p.offsets = offsets;
  p.order = order;
  p.fan = fan;
  p.gated = gated != 0;
  p.out = const_cast<void *>(elem_ptr(out));
  p.out_s0 = out->stride0;
  p.out_s1 = out->stride1;
  p.out_dtype = out->dtype;
  p.alpha = ep.alpha;
  p.bias = ep.bias;
  p.bias_dtype = ep.bias_dtype;
  p.activation = ep.activation;
  p.rounding = ep.rounding;
  const long long blocks = (p.rows + 31ll) / 32 + std::min(groups, p.rows);
  const dim3 grid((p.cols + 31) / 32, static_cast<unsigned>(std::min<long long>(blocks, 65535)));
  rows_simt_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return launched(h, "grouped_simt");
}

extern "C" KAPYB_API kapyb_status kapyb_matmul_grouped_grad(kapyb_handle h, const kapyb_tensor2d *lhs,
                                                            const kapyb_tensor2d *grad, int32_t groups,
                                                            const int32_t *offsets, const int32_t *order, int32_t fan,
                                                            const kapyb_tensor2d *out, int64_t out_group_stride,
                                                            float alpha, int32_t rounding, void *stream) {
  const char *call = "matmul_grouped_grad";
  TRY(check_tensor(h, call, "lhs", lhs));
  TRY(check_tensor(h, call, "grad", grad));
  TRY(check_output(h, call, "out", out));
  TRY(check_grouped(h, call, lhs, grad, groups, offsets, order, fan));
  if (!rounding_ok(rounding))
    return fail(h, KAPYB_INVALID_ARG, "%s: rounding mode must be set for down cast", call);
  if (out->size0 != lhs->size1 || out->size1 != grad->size1)
    return fail(h, KAPYB_INVALID_ARG, "%s: out must have a row per column of lhs and a column per column of grad", call);
  if (!order && lhs->size0 != grad->size0)
    return fail(h, KAPYB_INVALID_ARG, "%s: without order lhs must have as many rows as grad", call);
  if (empty(out)) {
    HAVE_HANDLE(h);
    return KAPYB_OK;
  }
  // groups of the output must not share addresses: behind one another, or interleaved
  // by whole rows / columns that another group cannot reach
  const int64_t extent = (out->size0 - 1ll) * out->stride0 + (out->size1 - 1ll) * out->stride1 + 1;
  if (groups > 1 && out_group_stride < extent)
    return fail(h, KAPYB_INVALID_ARG, "%s: out_group_stride (%lld) lets the groups of out overlap", call,
                static_cast<long long>(out_group_stride));
  const Span o = span_of(out, groups, out_group_stride);
  if (meet(o, span_of(lhs)) || meet(o, span_of(grad)) || meet(o, span_of(offsets, (groups + 1ull) * 4)) ||
      meet(o, span_of(order, order ? grad->size0 * 4ull : 0)))
    return fail(h, KAPYB_INVALID_ARG, "%s: out overlaps an input", call);
  ON_DEVICE(h);
  bool taken = false;
  const kapyb_status st = grouped_grad_on_tcgen05(h, lhs, grad, groups, offsets, order, fan, out, out_group_stride,
                                                  alpha, rounding, static_cast<cudaStream_t>(stream), &taken);
  if (taken || st != KAPYB_OK) return st;
  RowsSimtParams p{};
  p.x = elem_ptr(lhs);
  p.x_s0 = lhs->stride0;
  p.x_s1 = lhs->stride1;
  p.src_rows = lhs->size0;
  p.w = elem_ptr(grad);
  p.w_s0 = grad->stride0;
  p.w_s1 = grad->stride1;
  p.in_dtype = lhs->dtype;
  p.groups = groups;
  p.rows = grad->size0;
  p.K = lhs->size1;
  p.cols = grad->size1;
  p.offsets = offsets;
  p.order = order;
  p.fan = fan;
  p.out = const_cast<void *>(elem_ptr(out));
  p.out_s0 = out->stride0;
  p.out_s1 = out->stride1;
  p.out_group = out_group_stride;
  p.out_dtype = out->dtype;
  p.alpha = alpha;
  p.rounding = rounding;
  const int k_blocks = (p.K + 31) / 32;
  if (k_blocks > 65535)
    return fail(h, KAPYB_UNSUPPORTED, "%s: more than %d columns of lhs on the CUDA-core path", call, 65535 * 32);
  const dim3 grid((p.cols + 31) / 32, k_blocks, groups);
  rows_grad_simt_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return launched(h, "grouped_grad_simt");
}

// -------------------------------------------------------------------- combine

namespace {

// Whole pieces of `bytes`: unit column stride, base and row pitch aligned to them
bool pieces_ok(const kapyb_tensor2d *t, int bytes) {
  const int64_t esz = dtype_size(t->dtype);
  return t->stride1 == 1 && reinterpret_cast<uintptr_t>(elem_ptr(t)) % bytes == 0 && (t->stride0 * esz) % bytes == 0 &&
         (t->size1 * esz) % bytes == 0;
}

template <int DT>
void launch_combine_vec(const CombineParams &p, bool wide, uint32_t per_row, int grid, cudaStream_t s) {
  auto kern = wide ? combine_vec_kernel<DT, true> : combine_vec_kernel<DT, false>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, p, per_row);
}

template <int DT>
void launch_combine_any(const CombineParams &p, bool wide, uint32_t chunks, int grid, cudaStream_t s) {
  const bool unit = p.rows_s1 == 1;
  if (wide && unit) combine_any_kernel<DT, 8, true><<<grid, 256, 0, s>>>(p, chunks);
  else if (wide) combine_any_kernel<DT, 8, false><<<grid, 256, 0, s>>>(p, chunks);
  else if (unit) combine_any_kernel<DT, 2, true><<<grid, 256, 0, s>>>(p, chunks);
  else combine_any_kernel<DT, 2, false><<<grid, 256, 0, s>>>(p, chunks);
}

kapyb_status check_slots(kapyb_handle h, const char *call, const int32_t *slots, int k, const float *weights) {
  if (k < 1 || k > kCombineMaxK)
    return fail(h, KAPYB_INVALID_ARG, "%s: k must be 1 to %d (got %d)", call, kCombineMaxK, k);
  if (!slots) return fail(h, KAPYB_INVALID_ARG, "%s: slots is NULL", call);
  if (!aligned4(slots) || !aligned4(weights))
    return fail(h, KAPYB_INVALID_ARG, "%s: slots and weights must be 4-byte aligned", call);
  return KAPYB_OK;
}

}  // namespace

extern "C" KAPYB_API kapyb_status kapyb_combine_rows(kapyb_handle h, const kapyb_tensor2d *rows, const int32_t *slots,
                                                     int32_t k, const float *weights, const kapyb_tensor2d *out,
                                                     void *stream) {
  const char *call = "combine_rows";
  TRY(check_tensor(h, call, "rows", rows));
  TRY(check_output(h, call, "out", out));
  if (rows->size1 != out->size1)
    return fail(h, KAPYB_INVALID_ARG, "%s: rows and out must have as many columns", call);
  if (empty(out)) {
    HAVE_HANDLE(h);
    return KAPYB_OK;
  }
  TRY(check_slots(h, call, slots, k, weights));
  const size_t entries = static_cast<size_t>(out->size0) * k;
  const Span o = span_of(out);
  if (meet(o, span_of(rows)) || meet(o, span_of(slots, entries * 4)) || meet(o, span_of(weights, entries * 4)))
    return fail(h, KAPYB_INVALID_ARG, "%s: out overlaps an input", call);
  ON_DEVICE(h);
  CombineParams p{};
  p.rows = elem_ptr(rows);
  p.rows_s0 = rows->stride0;
  p.rows_s1 = rows->stride1;
  p.rows_dtype = rows->dtype;
  p.n_rows = rows->size0;
  p.slots = slots;
  p.weights = weights;
  p.tokens = out->size0;
  p.k = k;
  p.cols = out->size1;
  p.out = const_cast<void *>(elem_ptr(out));
  p.out_s0 = out->stride0;
  p.out_s1 = out->stride1;
  p.out_dtype = out->dtype;
  p.rounding = KAPYB_RN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool vec = rows->dtype == out->dtype && pieces_ok(rows, 16) && pieces_ok(out, 16);
  const bool wide = vec ? pieces_ok(rows, 32) : p.cols > 128;
  // threads of a token: one per piece, or whole warps of 8 (few columns: 2) elements a lane
  const int any = wide ? 256 : 64;
  const uint32_t per_row =
      vec ? static_cast<uint32_t>(static_cast<int64_t>(p.cols) * dtype_size(rows->dtype) / (wide ? 32 : 16))
          : (p.cols + any - 1) / any;
  const unsigned long long threads = static_cast<unsigned long long>(p.tokens) * per_row * (vec ? 1 : 32);
  const unsigned long long blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffull) return fail(h, KAPYB_UNSUPPORTED, "%s: output too large", call);
  const int grid = static_cast<int>(blocks);
  if (!vec && rows->dtype == KAPYB_F32)
    launch_combine_any<KAPYB_F32>(p, wide, per_row, grid, s);
  else if (!vec && rows->dtype == KAPYB_BF16)
    launch_combine_any<KAPYB_BF16>(p, wide, per_row, grid, s);
  else if (!vec)
    launch_combine_any<KAPYB_F16>(p, wide, per_row, grid, s);
  else if (rows->dtype == KAPYB_F32)
    launch_combine_vec<KAPYB_F32>(p, wide, per_row, grid, s);
  else if (rows->dtype == KAPYB_BF16)
    launch_combine_vec<KAPYB_BF16>(p, wide, per_row, grid, s);
  else
    launch_combine_vec<KAPYB_F16>(p, wide, per_row, grid, s);
  return launched(h, vec ? "combine_vec" : "combine_any");
}

extern "C" KAPYB_API kapyb_status kapyb_combine_rows_backward(kapyb_handle h, const kapyb_tensor2d *rows,
                                                              const int32_t *slots, int32_t k, const float *weights,
                                                              const kapyb_tensor2d *grad_out,
                                                              const kapyb_tensor2d *grad_rows, float *grad_weights,
                                                              void *stream) {
  const char *call = "combine_rows_backward";
  TRY(check_tensor(h, call, "grad_out", grad_out));
  if (grad_weights && !rows) return fail(h, KAPYB_INVALID_ARG, "%s: grad_weights needs rows", call);
  if (rows) TRY(check_tensor(h, call, "rows", rows));
  if (grad_rows) TRY(check_output(h, call, "grad_rows", grad_rows));
  if ((rows && rows->size1 != grad_out->size1) || (grad_rows && grad_rows->size1 != grad_out->size1))
    return fail(h, KAPYB_INVALID_ARG, "%s: rows, grad_out and grad_rows must have as many columns", call);
  if (rows && grad_rows && rows->size0 != grad_rows->size0)
    return fail(h, KAPYB_INVALID_ARG, "%s: grad_rows must have the shape of rows", call);
  if (grad_out->size0 == 0 || (!grad_rows && !grad_weights)) {
    HAVE_HANDLE(h);
    return KAPYB_OK;
  }
  TRY(check_slots(h, call, slots, k, weights));
  if (!aligned4(grad_weights)) return fail(h, KAPYB_INVALID_ARG, "%s: grad_weights must be 4-byte aligned", call);
  const size_t bytes = static_cast<size_t>(grad_out->size0) * k * 4;
  const Span gw = span_of(grad_weights, bytes);
  const Span gr = grad_rows ? span_of(grad_rows) : Span{0, 0};
  const Span in[4] = {rows ? span_of(rows) : Span{0, 0}, span_of(slots, bytes), span_of(weights, bytes),
                      span_of(grad_out)};
  if (meet(gw, gr)) return fail(h, KAPYB_INVALID_ARG, "%s: grad_weights overlaps grad_rows", call);
  for (const Span &i : in)
    if (meet(gw, i) || meet(gr, i)) return fail(h, KAPYB_INVALID_ARG, "%s: an output overlaps an input", call);
  ON_DEVICE(h);
  CombineParams p{};
  if (rows) {
    p.rows = elem_ptr(rows);
    p.rows_s0 = rows->stride0;
    p.rows_s1 = rows->stride1;
    p.rows_dtype = rows->dtype;
  }
  p.n_rows = rows ? rows->size0 : grad_rows->size0;
  p.slots = slots;
  p.weights = weights;
  p.tokens = grad_out->size0;
  p.k = k;
  p.cols = grad_out->size1;
  p.grad_out = elem_ptr(grad_out);
  p.go_s0 = grad_out->stride0;
  p.go_s1 = grad_out->stride1;
  p.go_dtype = grad_out->dtype;
  p.rounding = KAPYB_RN;
  if (grad_rows) {
    p.grad_rows = const_cast<void *>(elem_ptr(grad_rows));
    p.gr_s0 = grad_rows->stride0;
    p.gr_s1 = grad_rows->stride1;
    p.gr_dtype = grad_rows->dtype;
  }
  p.grad_weights = grad_weights;
  const int dt = grad_out->dtype;
  const bool same = (!rows || rows->dtype == dt) && (!grad_rows || grad_rows->dtype == dt);
  const bool vec = same && pieces_ok(grad_out, 16) && (!rows || pieces_ok(rows, 16)) &&
                   (!grad_rows || pieces_ok(grad_rows, 16));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long units = vec ? static_cast<long long>(p.cols) * dtype_size(dt) / 16 : (p.cols + 3ll) / 4;
  const int threads = static_cast<int>(std::min(256ll, std::max(32ll, (units + 31) / 32 * 32)));
  if (!same)
    combine_backward_kernel<-1, false><<<p.tokens, threads, 0, s>>>(p);
  else if (!vec && dt == KAPYB_F32)
    combine_backward_kernel<KAPYB_F32, false><<<p.tokens, threads, 0, s>>>(p);
  else if (!vec && dt == KAPYB_BF16)
    combine_backward_kernel<KAPYB_BF16, false><<<p.tokens, threads, 0, s>>>(p);
  else if (!vec)
    combine_backward_kernel<KAPYB_F16, false><<<p.tokens, threads, 0, s>>>(p);
  else if (dt == KAPYB_F32)
    combine_backward_kernel<KAPYB_F32, true><<<p.tokens, threads, 0, s>>>(p);
  else if (dt == KAPYB_BF16)
    combine_backward_kernel<KAPYB_BF16, true><<<p.tokens, threads, 0, s>>>(p);
  else
    combine_backward_kernel<KAPYB_F16, true><<<p.tokens, threads, 0, s>>>(p);
  return launched(h, vec ? "combine_backward_vec" : "combine_backward_any");
}

// ------------------------------------------------------------------- adapters

namespace {

constexpr int kMaxAdapterRank = 128;

size_t up256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// Scratch of the call: f32 products for few rows and the CUDA-core path, else the plan
// (order, offsets) and the products' two 16-bit halves.
struct AdapterScratch {
  int64_t positions;   // of the padded plan: groups start at multiples of 32
  size_t order, offsets, low, total;
  AdapterScratch(int rows, int groups, int rank) {
    positions = (rows + 31ll * std::min(groups + 1, rows) + 31) / 32 * 32;
    order = 0;
    offsets = up256(static_cast<size_t>(positions) * 4);
    low = offsets + up256((groups + 2ull) * 4);
    const size_t halves = static_cast<size_t>(positions) * ((rank + 7) / 8 * 8) * 2 * 2;
    total = std::max(low + halves, static_cast<size_t>(rows) * rank * sizeof(float));
  }
};

struct AdapterCall {
  const kapyb_tensor2d *lhs, *rhs, *down, *up, *out;
  int groups;
  int64_t down_stride, up_stride;
  const int32_t *index;
  const float *scale;
  const kapyb_epilogue &ep;
  void *scratch;
};

// One matrix of a stack as TMA can fetch it; `mn`: unit stride on the second axis.
bool stack_tma_ok(const kapyb_tensor2d *t, int groups, int64_t stride, bool &mn, int64_t &unit, int64_t &other,
                  int64_t &ld) {
  mn = t->stride1 == 1;
  if (!half_type(t->dtype) || (!mn && t->stride0 != 1)) return false;
  unit = mn ? t->size1 : t->size0;
  other = mn ? t->size0 : t->size1;
  ld = mn ? t->stride0 : t->stride1;
  return tma_ok(elem_ptr(t), t->dtype, unit, other, ld, groups, stride);
}

// At most 256 rows: the weight stream with the adapters' part beside it.
kapyb_status adapters_decode(kapyb_handle h, const AdapterCall &c, cudaStream_t stream, bool *taken) {
  *taken = false;
  bool mn;
  int64_t unit, other, ld;
  if (c.lhs->size0 > kDecodeMaxRows || !rows_tma_ok(c.lhs) || !stack_tma_ok(c.rhs, 1, 0, mn, unit, other, ld))
    return KAPYB_OK;
  const int rows = c.lhs->size0, rank = c.down->size1;
  const uint16_t *down = static_cast<const uint16_t *>(elem_ptr(c.down));
  float *low = static_cast<float *>(c.scratch);
  const bool bf = c.lhs->dtype == KAPYB_BF16;

  const int wide = (rows + 15) / 16 * 16, num_kb = (c.lhs->size1 + 63) / 64;
  // CTAs per column block.  Up to 64 rows two CTAs fit an SM (the ring is kept below half
  // of its shared memory), so that one streams while the other starts or ends, and a CTA
  // by itself streams some 50 GB/s at most.  The share of those places that is used, over
  // whole waves, decides; more CTAs must gain a fifth.  Each keeps at least four K blocks.
  const int tiles = (c.out->size1 + 127) / 128;
  const int per_sm = wide <= 64 ? 2 : 1;
  const int places = h->sm_count * per_sm;
  int split = 1;
  double best = 0.0;
  for (int s = 1; s <= 8 && s * 4 <= std::max(4, num_kb); s *= 2) {
    const long long units = static_cast<long long>(tiles) * s;
    const long long waves = (units + places - 1) / places;
    const double used = static_cast<double>(units) / (waves * places);
    if (used > best * 1.2) {
      best = used;
      split = s;
    }
  }
  const int stage_bytes = 16384 + wide * 128;
  int delta = 0, stages = 0;
  for (;; split *= 2) {  // rows of a CTA's share of the output, in f32, beside the ring
    delta = (rows + split - 1) / split * 512;
    const int budget = 232448 / per_sm - 3 * 1024 - delta;
    stages = std::min(8, budget / stage_bytes);
    // the ring also takes the partial sums
    if (stages >= 3 && stages * stage_bytes >= wide * 512) break;
    if (split >= 8) return KAPYB_OK;
  }
  const int smem = 1024 + stages * stage_bytes + delta;

  // low = scale * x . down
  const bool d_aligned = aligned16(down) && c.down_stride % 8 == 0;
  const bool d_k = c.down->stride0 == 1 && c.down->stride1 % 8 == 0 && d_aligned;
  const bool d_r = c.down->stride1 == 1 && c.down->stride0 % 8 == 0 && d_aligned && rank % 8 == 0;
  if (d_k || d_r) {
    const LowParams lp{static_cast<const uint16_t *>(elem_ptr(c.lhs)), c.lhs->stride0, down, c.down->stride0,
                       c.down->stride1, c.down_stride, bf, c.groups, rows, c.lhs->size1, rank, c.index, c.scale, low,
                       // few rows share their K between CTAs: two blocks of 512 threads an SM at most
                       rows <= h->sm_count / 2 ? kLowMaxSplit : rows <= h->sm_count ? 2 : 1};
    auto kern = d_r ? (bf ? adapter_low_kernel<true, false> : adapter_low_kernel<false, false>)
                    : (bf ? adapter_low_kernel<true, true> : adapter_low_kernel<false, true>);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(static_cast<unsigned>(rows) * lp.split, 1, 1);
    cfg.blockDim = dim3(kLowThreads, 1, 1);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = lp.split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CUDA_TRY(h, cudaLaunchKernelEx(&cfg, kern, lp));
  } else {
    AdapterSimtParams sp{};
    sp.x = elem_ptr(c.lhs);
    sp.x_s0 = c.lhs->stride0;
    sp.x_s1 = c.lhs->stride1;
    sp.down = down;
    sp.d_s0 = c.down->stride0;
    sp.d_s1 = c.down->stride1;
    sp.d_group = c.down_stride;
    sp.in_dtype = c.lhs->dtype;
    sp.groups = c.groups;
    sp.rows = rows;
    sp.K = c.lhs->size1;
    sp.rank = rank;
    sp.index = c.index;
    sp.scale = c.scale;
    sp.low = low;
    adapter_low_simt_kernel<<<rows, 256, 0, stream>>>(sp);
  }
  TRY(launched(h, "adapter_low"));

  DecodeParams p{};
  p.rows = rows;
  p.wide = wide;
  p.cols = c.out->size1;
  p.num_kb = num_kb;
  p.stages = stages;
  p.stage_bytes = stage_bytes;
  p.w_mn_major = mn;
  p.bf16 = bf;
  p.tmem_cols = 32;
  while (static_cast<int>(p.tmem_cols) < p.wide) p.tmem_cols *= 2;
  p.low = low;
  p.index = c.index;
  p.groups = c.groups;
  p.rank = rank;
  p.up = static_cast<const uint16_t *>(elem_ptr(c.up));
  p.u_s0 = c.up->stride0;
  p.u_s1 = c.up->stride1;
  p.u_group = c.up_stride;
  const bool u_aligned = aligned16(p.up) && c.up_stride % 8 == 0;
  p.up_form = u_aligned && p.u_s1 == 1 && p.u_s0 % 8 == 0 && p.cols % 8 == 0 ? 1
              : u_aligned && p.u_s0 == 1 && p.u_s1 % 8 == 0 && rank % 8 == 0 ? 2
                                                                             : 0;
  p.out = const_cast<void *>(elem_ptr(c.out));
  p.out_s0 = c.out->stride0;
  p.out_s1 = c.out->stride1;
  p.out_dtype = c.out->dtype;
  p.alpha = c.ep.alpha;
  p.bias = c.ep.bias;
  p.bias_dtype = c.ep.bias_dtype;
  p.bias_axis = c.ep.bias_axis;
  p.activation = c.ep.activation;
  p.rounding = c.ep.rounding;
  p.status = h->status;
  p.wait_limit_us = h->wait_limit_us;
  CUtensorMap tmW, tmX;
  TRY(make_tmap(h, &tmW, elem_ptr(c.rhs), c.rhs->dtype, unit, other, 1, ld, 0, 64, mn ? 64 : 128));
  TRY(make_row_tmap(h, &tmX, elem_ptr(c.lhs), c.lhs->dtype, c.lhs->size1, rows,
                    rows > 1 ? c.lhs->stride0 : (c.lhs->size1 + 7) / 8 * 8, p.wide));
  auto kern = bf ? adapter_decode_kernel<true> : adapter_decode_kernel<false>;
  TRY(bf ? allow_smem<adapter_decode_kernel<true>>(h, 232448 - 512)
         : allow_smem<adapter_decode_kernel<false>>(h, 232448 - 512));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>(tiles) * split, 1, 1);
  cfg.blockDim = dim3(192, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see adapters_sm100.cuh
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  *taken = true;
  CUDA_TRY(h, cudaLaunchKernelEx(&cfg, kern, tmW, tmX, p));
  return launched(h, "adapters_decode");
}

// More rows: sorted by adapter, products down on the pair kernel, then one pass over the
// shared weights that takes the adapters' K blocks along.
kapyb_status adapters_pairs(kapyb_handle h, const AdapterCall &c, cudaStream_t stream, bool *taken) {
  *taken = false;
  bool w_mn, d_mn, u_mn;
  int64_t w_unit, w_other, w_ld, d_unit, d_other, d_ld, u_unit, u_other, u_ld;
  const int rank = c.down->size1, K = c.lhs->size1, rows = c.lhs->size0;
  const int64_t pitch = static_cast<int64_t>(c.out->stride0) * dtype_size(c.out->dtype);
  if (!rows_tma_ok(c.lhs) || c.out->stride1 != 1 || pitch >= kMaxRowPitch ||
      !stack_tma_ok(c.rhs, 1, 0, w_mn, w_unit, w_other, w_ld) ||
      !stack_tma_ok(c.down, c.groups, c.down_stride, d_mn, d_unit, d_other, d_ld) ||
      !stack_tma_ok(c.up, c.groups, c.up_stride, u_mn, u_unit, u_other, u_ld))
    return KAPYB_OK;
  // the adapters' part is divided by alpha (or, in f16, by its mantissa), which needs an
  // alpha that division does not push out of the 16-bit types' ranges
  const float size = std::fabs(c.ep.alpha);
  if (!(size >= 0.00390625f && size <= 256.0f)) return KAPYB_OK;
  // f16: alpha = adapter_alpha 2^-shift, see grouped_sm100.cuh
  int shift = 0;
  if (c.lhs->dtype == KAPYB_F16 && size < 1.0f) {
    std::frexp(size, &shift);  // size = fraction 2^shift, fraction in [1/2, 1)
    shift = 1 - shift;
  }
  const float adapter_alpha = std::ldexp(c.ep.alpha, shift);
  const AdapterScratch sc(rows, c.groups, rank);
  const int n_tiles = (c.out->size1 + 255) / 256;
  if (sc.positions >= (1ll << 30) || (sc.positions / 256 + 1) * n_tiles >= (1ll << 30)) return KAPYB_OK;
  char *scratch = static_cast<char *>(c.scratch);
  int32_t *order = reinterpret_cast<int32_t *>(scratch + sc.order);
  int32_t *offsets = reinterpret_cast<int32_t *>(scratch + sc.offsets);
  const int low_pitch = (rank + 7) / 8 * 8;
  const int positions = static_cast<int>(sc.positions);

  *taken = true;
  TRY(launch_plan(h, PlanParams{c.index, rows, c.groups + 1, order, offsets, nullptr, positions, 32, 1}, stream));

  // the rows' products with their adapter's down, in two halves
  CUtensorMap tmD, tmW, tmU, tmL, tmR;
  LowTileParams lp{};
  lp.offsets = offsets;
  lp.order = order;
  lp.groups = c.groups;
  lp.positions = positions;
  lp.x = static_cast<const uint8_t *>(elem_ptr(c.lhs));
  lp.x_pitch = c.lhs->stride0 * 2ll;
  lp.src_rows = rows;
  lp.K = K;
  lp.rank = rank;
  lp.d_mn_major = d_mn;
  lp.bf16 = c.lhs->dtype == KAPYB_BF16;
  lp.a_bytes = rank <= 64 ? 8192 : 16384;
  lp.scale = c.scale;
  lp.alpha = 1.0f / adapter_alpha;
  lp.high = reinterpret_cast<uint16_t *>(scratch + sc.low);
  lp.low = lp.high + static_cast<size_t>(positions) * low_pitch;
  lp.pitch = low_pitch;
  lp.status = h->status;
  lp.wait_limit_us = h->wait_limit_us;
  TRY(make_tmap(h, &tmD, elem_ptr(c.down), c.down->dtype, d_unit, d_other, c.groups, d_ld, c.down_stride, 64,
                d_mn || rank <= 64 ? 64 : 128));
  // tiles at most; CTAs per tile until two an SM are busy, each keeping four K blocks
  const long long low_tiles = (positions + kLowTile - 1ll) / kLowTile + std::min(c.groups, rows);
  const int num_kb = (K + 63) / 64;
  lp.split = 1;
  while (lp.split < 8 && low_tiles * lp.split < 2 * h->sm_count && lp.split * 8 <= num_kb) lp.split *= 2;
  {
    auto kern = lp.bf16 ? adapter_low_tile_kernel<true> : adapter_low_tile_kernel<false>;
    TRY(lp.bf16 ? allow_smem<adapter_low_tile_kernel<true>>(h, kLowTileSmem)
                : allow_smem<adapter_low_tile_kernel<false>>(h, kLowTileSmem));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(static_cast<unsigned>(low_tiles) * lp.split, 1, 1);
    cfg.blockDim = dim3(kLowTileThreads, 1, 1);
    cfg.dynamicSmemBytes = kLowTileSmem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = lp.split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CUDA_TRY(h, cudaLaunchKernelEx(&cfg, kern, tmD, lp));
    TRY(launched(h, "adapter_low_tile"));
  }

  GroupedParams gp{};
  gp.rows = positions;
  gp.K = K;
  gp.num_kb = num_kb;
  gp.offsets = offsets;
  gp.order = order;
  gp.fan = 1;
  gp.src_rows = rows;
  gp.bf16 = lp.bf16;
  gp.status = h->status;
  gp.wait_limit_us = h->wait_limit_us;
  gp.groups = c.groups + 1;
  gp.cols = c.out->size1;
  gp.n_tiles = n_tiles;
  gp.a_mn_major = w_mn;
  gp.out = const_cast<void *>(elem_ptr(c.out));
  gp.row_pitch = static_cast<uint32_t>(pitch);
  gp.out_dtype = c.out->dtype;
  gp.wide_stores = wide_stores_ok(gp.out, c.out->dtype, c.out->stride0, 0);
  gp.alpha = c.ep.alpha;
  gp.bias = c.ep.bias;
  gp.bias_dtype = c.ep.bias_dtype;
  gp.bias_axis = c.ep.bias_axis;
  gp.activation = c.ep.activation;
  gp.rounding = c.ep.rounding;
  PairParams pp = pair_params(gp, c.lhs, true);
  pp.rank = rank;
  pp.up_mn_major = u_mn;
  pp.low_rows = positions;
  pp.adapter_alpha = adapter_alpha;
  pp.adapter_shift = shift;
  TRY(make_tmap(h, &tmW, elem_ptr(c.rhs), c.rhs->dtype, w_unit, w_other, 1, w_ld, 0, 64, w_mn ? 64 : 128));
  TRY(make_tmap(h, &tmU, elem_ptr(c.up), c.up->dtype, u_unit, u_other, c.groups, u_ld, c.up_stride, 64,
                u_mn ? 64 : 128));
  TRY(make_row_tmap(h, &tmL, scratch + sc.low, c.lhs->dtype, rank, 2ull * positions, low_pitch, PairCfg::BT / 2));
  TRY(make_row_tmap(h, &tmR, scratch + sc.low, c.lhs->dtype, rank, 2ull * positions, low_pitch, 16));
  return launch_pairs<PAIR_ADAPTERS>(h, tmW, tmL, tmR, tmU, pp, (positions / 256 + 1ll) * n_tiles, stream);
}

}  // namespace

extern "C" KAPYB_API size_t kapyb_matmul_adapters_scratch(int32_t rows, int32_t groups, int32_t rank) {
  if (rows <= 0 || groups <= 0 || rank <= 0) return 0;
  return AdapterScratch(rows, groups, rank).total;
}

extern "C" KAPYB_API kapyb_status kapyb_matmul_adapters(kapyb_handle h, const kapyb_tensor2d *lhs,
                                                        const kapyb_tensor2d *rhs, int32_t groups,
                                                        const kapyb_tensor2d *down, int64_t down_stride,
                                                        const kapyb_tensor2d *up, int64_t up_stride,
                                                        const int32_t *index, const float *scale,
                                                        const kapyb_tensor2d *out, const kapyb_epilogue *epilogue,
                                                        void *scratch, size_t scratch_bytes, void *stream) {
  const char *call = "matmul_adapters";
  TRY(check_tensor(h, call, "lhs", lhs));
  TRY(check_tensor(h, call, "rhs", rhs));
  TRY(check_tensor(h, call, "down", down));
  TRY(check_tensor(h, call, "up", up));
  TRY(check_output(h, call, "out", out));
  TRY(check_epilogue(h, call, epilogue));
  if (lhs->dtype != rhs->dtype || lhs->dtype != down->dtype || lhs->dtype != up->dtype)
    return fail(h, KAPYB_INVALID_ARG, "%s: lhs, rhs, down and up must have same element type", call);
  for (const kapyb_tensor2d *t : {lhs, rhs, down, up})
    if (t->padding != KAPYB_PAD_ZERO)
      return fail(h, KAPYB_UNSUPPORTED, "%s: operands are padded with zeros only", call);
  if (groups < 1 || groups > kMaxRowGroups)
    return fail(h, groups < 1 ? KAPYB_INVALID_ARG : KAPYB_UNSUPPORTED, "%s: 1 to %d adapters (got %d)", call,
                kMaxRowGroups, groups);
  if (down_stride < 0 || up_stride < 0)
    return fail(h, KAPYB_INVALID_ARG, "%s: down_stride or up_stride is negative", call);
  if (lhs->size1 != rhs->size0)
    return fail(h, KAPYB_INVALID_ARG, "%s: number of columns of lhs must be equal to number of rows of rhs", call);
  if (out->size0 != lhs->size0 || out->size1 != rhs->size1)
    return fail(h, KAPYB_INVALID_ARG, "%s: out must have the rows of lhs and the columns of rhs", call);
  if (down->size0 != lhs->size1 || up->size1 != rhs->size1 || down->size1 != up->size0)
    return fail(h, KAPYB_INVALID_ARG, "%s: down must be [columns of lhs, rank] and up [rank, columns of rhs]", call);
  if (down->size1 < 1 || down->size1 > kMaxAdapterRank)
    return fail(h, down->size1 < 1 ? KAPYB_INVALID_ARG : KAPYB_UNSUPPORTED, "%s: rank must be 1 to %d (got %d)", call,
                kMaxAdapterRank, down->size1);
  if (empty(out)) {
    HAVE_HANDLE(h);
    return KAPYB_OK;
  }
  if (!index) return fail(h, KAPYB_INVALID_ARG, "%s: index is NULL", call);
  if (!aligned4(index) || !aligned4(scale))
    return fail(h, KAPYB_INVALID_ARG, "%s: index and scale must be 4-byte aligned", call);
  const size_t need = kapyb_matmul_adapters_scratch(lhs->size0, groups, down->size1);
  if (!scratch || scratch_bytes < need || reinterpret_cast<uintptr_t>(scratch) % 256 != 0)
    return fail(h, KAPYB_INVALID_ARG, "%s: scratch must be %zu bytes, 256-byte aligned", call, need);
  const kapyb_epilogue &ep = epilogue ? *epilogue : kPlainEpilogue;
  const Span o = span_of(out), sc = span_of(scratch, need);
  const Span in[8] = {span_of(lhs), span_of(rhs), span_of(down, groups, down_stride), span_of(up, groups, up_stride),
                      span_of(index, lhs->size0 * 4ull), span_of(scale, scale ? groups * 4ull : 0),
                      span_of(ep.bias, static_cast<size_t>(ep.bias_axis == 1 ? out->size1 : out->size0) *
                                           dtype_size(ep.bias_dtype)),
                      Span{0, 0}};
  if (meet(o, sc)) return fail(h, KAPYB_INVALID_ARG, "%s: out overlaps scratch", call);
  for (const Span &i : in)
    if (meet(o, i) || meet(sc, i)) return fail(h, KAPYB_INVALID_ARG, "%s: out or scratch overlaps an input", call);
  ON_DEVICE(h);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (lhs->size1 > 0) {
    const AdapterCall c{lhs, rhs, down, up, out, groups, down_stride, up_stride, index, scale, ep, scratch};
    bool taken = false;
    kapyb_status st = adapters_decode(h, c, s, &taken);
    if (st != KAPYB_OK || taken) return st;
    st = adapters_pairs(h, c, s, &taken);
    if (st != KAPYB_OK || taken) return st;
  }
  AdapterSimtParams p{};
  p.x = elem_ptr(lhs);
  p.x_s0 = lhs->stride0;
  p.x_s1 = lhs->stride1;
  p.w = elem_ptr(rhs);
  p.w_s0 = rhs->stride0;
  p.w_s1 = rhs->stride1;
  p.down = elem_ptr(down);
  p.d_s0 = down->stride0;
  p.d_s1 = down->stride1;
  p.d_group = down_stride;
  p.up = elem_ptr(up);
  p.u_s0 = up->stride0;
  p.u_s1 = up->stride1;
  p.u_group = up_stride;
  p.in_dtype = lhs->dtype;
  p.groups = groups;
  p.rows = lhs->size0;
  p.K = lhs->size1;
  p.cols = rhs->size1;
  p.rank = down->size1;
  p.index = index;
  p.scale = scale;
  p.low = static_cast<float *>(scratch);
  p.out = const_cast<void *>(elem_ptr(out));
  p.out_s0 = out->stride0;
  p.out_s1 = out->stride1;
  p.out_dtype = out->dtype;
  p.alpha = ep.alpha;
  p.bias = ep.bias;
  p.bias_dtype = ep.bias_dtype;
  p.bias_axis = ep.bias_axis;
  p.activation = ep.activation;
  p.rounding = ep.rounding;
  adapter_low_simt_kernel<<<p.rows, 256, 0, s>>>(p);
  TRY(launched(h, "adapter_low_simt"));
  const dim3 grid((p.cols + 31) / 32, static_cast<unsigned>(std::min((p.rows + 31ll) / 32, 65535ll)));
  adapter_simt_kernel<<<grid, 256, 0, s>>>(p);
  return launched(h, "adapter_simt");
}
