// What the library's translation units share on the host side: the handle, error
// reporting, descriptor checks and tensor-map construction.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "common.cuh"

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                  const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

enum MatmulPath { PATH_AUTO = 0, PATH_1CTA, PATH_2CTA, PATH_SKINNY, PATH_SIMT };
constexpr int kMaxDevices = 64;

struct kapyb_context {
  int device = 0;
  int sm_count = 0;
  uint32_t *status = nullptr;  // device word written by kernels that give up
  void *workspace = nullptr;
  size_t workspace_bytes = 0;
  EncodeTiledFn encode = nullptr;
  std::string last_error;
  const char *last_kernel = "none";
  int64_t launches = 0;
  int forced_path = PATH_AUTO;
  int forced_bn = 0;
  int debug = 0;
  uint32_t wait_limit_us = 0;
  int forced_epi = 0;  // 0: by K; 4 or 8: that many epilogue warps (single-CTA kernels)
  int skinny_stages = 0;  // 0: the default depth
  uint32_t skinny_epoch = 0;  // number of the last decode-kernel launch that used the workspace
  int forced_group_m = 0; // 0: the default raster group (row blocks walked together); else that many
  int skinny_split = -1;  // -1: by shape; 0: whole weight tiles only; 1: split leftover tiles between SMs
  int tile_split = -1;    // tcgen05 kernels, the same three choices for the last wave's tiles
  void *split_scratch = nullptr;  // their partial accumulators and flag words
  size_t split_scratch_bytes = 0;
  uint32_t split_epoch = 0;       // number of the last launch that used them
  // host-buffer calls: copy streams and events for the chunked pipeline
  cudaStream_t copy_in = nullptr, copy_out = nullptr;
  cudaEvent_t ev[2 * 16 + 2] = {};
  bool pipe_ready = false;
  // sharded host-buffer calls: the stream that forwards this rank's rows to its peers
  cudaStream_t push = nullptr;
  cudaEvent_t ev_push[16 + 1] = {};
  bool push_ready = false;
};

// Error text of calls without a handle (one per thread and library).
inline thread_local std::string g_create_error;

inline kapyb_status fail(kapyb_handle h, kapyb_status st, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  if (h)
    h->last_error = buf;
  else
    g_create_error = buf;
  return st;
}

#define CUDA_TRY(h, expr)                                                                  \
  do {                                                                                     \
    cudaError_t e_ = (expr);                                                               \
    if (e_ != cudaSuccess)                                                                 \
      return fail(h, KAPYB_CUDA_ERROR, "%s failed: %s", #expr, cudaGetErrorString(e_));    \
  } while (0)

// kapyb_tensor2d.cache: cache operator 0..7, eviction priority 0..4, volatile bit
inline bool valid_cache(int c) {
  return (c & ~0x1ffff) == 0 && (c & 0xff) <= KAPYB_CACHE_CV && ((c >> 8) & 0xff) <= KAPYB_NO_ALLOCATE;
}

inline bool valid_dtype(int d) { return d == KAPYB_F16 || d == KAPYB_BF16 || d == KAPYB_F32; }
inline bool is_fp8(int d) { return d == KAPYB_F8E4M3 || d == KAPYB_F8E5M2; }
inline bool valid_operand_dtype(int d) { return valid_dtype(d) || is_fp8(d); }

inline const char *dtype_name(int d) {
  return d == KAPYB_F16     ? "f16"
         : d == KAPYB_BF16  ? "bf16"
         : d == KAPYB_F32   ? "f32"
         : d == KAPYB_F8E4M3 ? "f8E4M3"
         : d == KAPYB_F8E5M2 ? "f8E5M2"
         : d == KAPYB_I1     ? "i1"
                             : "?";
}

inline const void *elem_ptr(const kapyb_tensor2d *t) {
  return static_cast<const char *>(t->ptr) + t->offset_elems * kapyb::dtype_size(t->dtype);
}

inline CUtensorMapDataType tmap_dtype(int dtype) {
  return dtype == KAPYB_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : dtype == KAPYB_F16  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
         : dtype == KAPYB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                               : CU_TENSOR_MAP_DATA_TYPE_UINT8;
}

// 3-D map over a matrix whose unit-stride axis has `inner` elements and whose
// other axis has `outer` rows `ld` elements apart, repeated `batch` times.
inline kapyb_status make_tmap(kapyb_handle h, CUtensorMap *map, const void *base, int dtype,
                              uint64_t inner, uint64_t outer, uint64_t batch, uint64_t ld,
                              uint64_t batch_stride, uint32_t box_inner, uint32_t box_outer,
                              bool swizzle_32b_units = false) {
  const uint64_t esz = kapyb::dtype_size(dtype);
  cuuint64_t dims[3] = {inner, outer, batch};
  uint64_t bs = batch_stride * esz;
  if (batch <= 1 || bs == 0) bs = ((std::max<uint64_t>(outer, 1) * ld * esz) + 15) / 16 * 16;
  cuuint64_t strides[2] = {ld * esz, bs};
  cuuint32_t box[3] = {box_inner, box_outer, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = h->encode(map, tmap_dtype(dtype), 3, const_cast<void *>(base), dims, strides, box,
                         estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle_32b_units ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B
                                           : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(h, KAPYB_CUDA_ERROR,
                "cuTensorMapEncodeTiled failed (%d): dims=%llu,%llu,%llu ld=%llu box=%u,%u", (int)r,
                (unsigned long long)inner, (unsigned long long)outer, (unsigned long long)batch,
                (unsigned long long)ld, box_inner, box_outer);
  return KAPYB_OK;
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A 2-D operand is TMA-describable when one stride is 1, its base is 16-byte
// aligned and the other stride (and the batch stride) are multiples of 16 bytes.
inline bool tma_ok(const void *base, int dtype, int64_t unit_extent, int64_t other_extent,
                   int64_t ld, int64_t batch, int64_t batch_stride) {
  const int64_t esz = kapyb::dtype_size(dtype);
  if (!aligned16(base)) return false;
  if (unit_extent <= 0 || other_extent <= 0) return false;
  if (other_extent > 1 && ((ld * esz) % 16 != 0 || ld < unit_extent)) return false;
  if (other_extent == 1 && (ld * esz) % 16 != 0) return false;
  if (batch > 1 && ((batch_stride * esz) % 16 != 0 || batch_stride <= 0)) return false;
  if (ld * esz >= (1ll << 40)) return false;
  return true;
}

