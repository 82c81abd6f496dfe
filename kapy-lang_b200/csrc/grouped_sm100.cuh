// Products of rows that pick their weights, on tcgen05:
//   forward   out[p, n]    = epilogue( sum_k lhs[row(p), k] * rhs[g(p)][k, n] )
//   gradient  out[g][k, n] = alpha * sum over p of group g  lhs[row(p), k] * grad[p, n]
//   adapters  out[t, n]    = epilogue( lhs[t] . rhs ) + low[t] . up[i(t)]
//
// Two CTAs of a cluster share a tile of 256 output columns and up to 256 rows through
// tcgen05.mma.cta_group::2.  The output columns n always fill the M side of the MMA (TMEM
// lanes, 128 in each CTA) and the output rows its N side:  D[n, r] = sum A[n, .] B[r, .].
// The N side of a pair's MMA is any multiple of 32 up to 256, so a group of three rows
// costs a 32-wide MMA and not a tile of 256 rows, and one kernel serves a decode step (a
// few rows per group, bound by streaming the weights) and a prompt (hundreds of rows,
// bound by the tensor cores).  A group's rows are dealt out in equal tiles.
// (A kernel of single CTAs with tiles of 64 rows, for few rows a group, was 2% quicker at
// best, 301 us against 308 for 8 groups of 4 rows, 4096 x 14336 gated.  64 groups of 2048 x
// 2048 took it 115 us against 103 at 8 rows a group, 168 against 104 at 32.)
//
// Rows named by a plan are fetched where they lie, so no permuted copy of lhs is written.
// Rows outside lhs, and the K tail of both operands, arrive as zeros.  A tile's rows
// behind the end of its group may be those of the next group: they only reach output
// rows that are not stored.  In the gradient the rows are the contraction, so there
// everything behind a group's end, and every position whose entry names no row, is fetched
// as zeros on both sides (a zero on one side alone would still let a NaN through).
//
// Persistent CTAs; warp 0 fetches columns, warp 1 issues the MMAs, warps 6..14 fetch rows
// (below), warps 2..5 and 15..18 drain: two accumulator slots in TMEM let the drain of one
// tile run under the next one's main loop.  A drain is bound by latency, some 700 clocks
// for 32 rows of 32 columns, twice that with gate and up; with four warps it took longer
// than 16 K blocks of MMAs (64 gradients of 2048 x 2048 from 64 rows each: 251 us, with
// eight 188; K of 256, gated, 16384 x 4096: 122 and 89).
//
// The table of tiles depends on the plan, which only the device knows: every CTA
// builds it in shared memory from the offsets (a scan over at most 1024 groups).
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "gemm_sm100.cuh"
#include "ptx_sm100.cuh"
#include "rows_simt.cuh"

namespace kapyb {

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void *tmap, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      :
      : "r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

struct GroupedParams {
  int groups, rows;      // rows: positions of the plan
  int cols;              // output columns (of one group)
  int K;                 // forward: contraction length; gradient: output rows of one group
  int n_tiles;           // column blocks of 256 (gated: 128)
  int k_tiles;           // gradient: ceil(K / BT)
  int num_kb;            // forward: ceil(K / 64)
  const int32_t *offsets, *order;
  int fan, src_rows;     // row(p) = order[p] / fan (order may be nullptr: p); rows of lhs
  int a_mn_major;        // forward: rhs has its unit stride on n
  int bf16;
  void *out;
  uint32_t row_pitch;           // bytes between output rows, below 2^26; unit stride on n
  long long group_bytes;        // gradient: bytes between groups
  int out_dtype, wide_stores;   // wide_stores: two 16-bit columns may be stored as one word,
                                // or four f32 ones added to as 16 bytes
  float alpha;
  const void *bias;      // [groups, bias_cols]; adapters: [cols], or [source rows] with bias_axis 0
  int bias_dtype, bias_cols, bias_axis, activation, rounding;
  uint32_t *status;
  uint32_t wait_limit_us;
};

constexpr int kGroupedMaxGroups = 1024;

// One output tile.
struct GroupedTile {
  int g;        // group
  int n0;       // first output column
  int r0;       // forward: first position; gradient: first output row
  int rows;     // output rows of the tile
  int wide;     // the MMA's N: rows rounded up to 32
  int num_kb;   // K blocks
  int p0, p1;   // gradient: the group's positions
};

// Which of a group's tiles (`tiles` row tiles x n_tiles column blocks) is number `in`:
// row tiles next to one another, eight at a time, so that CTAs running at the same time
// share rows and columns in L2 (eight row tiles and some nine column blocks at once
// instead of all row tiles of a long group and one or two column blocks).
__device__ __forceinline__ void raster(int in, int tiles, int n_tiles, int &m, int &n) {
  const int block = in / (8 * n_tiles), first = block * 8;
  const int high = min(8, tiles - first);
  const int r = in - block * 8 * n_tiles;
  n = r / high;
  m = first + r - n * high;
}

// The tile table in shared memory: first[g] = tiles of output rows in front of group
// g, begin[g] / count[g] its positions.
struct GroupedTable {
  int *first, *begin, *count;
};

// Builds the table from the plan's offsets; one warp.  An offset below one in front of it
// counts as that one, so that groups never overlap, whatever the memory holds: the number
// of tiles stays below the bound the host has checked.
__device__ __forceinline__ void build_tile_table(const int32_t *offsets, int groups, int rows, int tile_rows,
                                                 const GroupedTable &table, int lane) {
  int before = 0, high = 0;
  for (int g0 = 0; g0 < groups; g0 += 32) {
    const int g = g0 + lane;
    int b = 0, e = 0;
    if (g < groups) group_range(offsets, g, rows, b, e);
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, b, off);
      if (lane >= off) b = max(b, o);
    }
    b = max(b, high);
    high = __shfl_sync(0xffffffffu, b, 31);
    const int cnt = max(0, e - b);
    const int tiles = (cnt + tile_rows - 1) / tile_rows;
    int scan = tiles;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, scan, off);
      if (lane >= off) scan += o;
    }
    if (g < groups) {
      table.first[g] = before + scan - tiles;
      table.begin[g] = b;
      table.count[g] = cnt;
    }
    before += __shfl_sync(0xffffffffu, scan, 31);
  }
  if (lane == 0) table.first[groups] = before;
}

// The group that row tile q belongs to.
__device__ __forceinline__ int find_group(const GroupedTable &t, int groups, int q) {
  int lo = 0, hi = groups;  // first[lo] <= q < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= q) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int R>
__device__ __forceinline__ void grouped_activation(int activation, float (&f)[R]) {
  switch (activation) {
  case KAPYB_ACT_RELU:
#pragma unroll
    for (int i = 0; i < R; ++i) f[i] = apply_activation_t<KAPYB_ACT_RELU>(f[i]);
    break;
  case KAPYB_ACT_GELU_TANH:
#pragma unroll
    for (int i = 0; i < R; ++i) f[i] = apply_activation_t<KAPYB_ACT_GELU_TANH>(f[i]);
    break;
  case KAPYB_ACT_SILU:
#pragma unroll
    for (int i = 0; i < R; ++i) f[i] = apply_activation_t<KAPYB_ACT_SILU>(f[i]);
    break;
  default: break;
  }
}

// Scale, bias and activation of 32 values of one output column.
__device__ __forceinline__ void grouped_finish32(const GroupedParams &p, float (&f)[32], float alpha, float bias) {
#pragma unroll
  for (int i = 0; i < 32; ++i) f[i] = f[i] * alpha + bias;
  grouped_activation(p.activation, f);
}

// 16-bit values of one column per lane (rows 2i, 2i + 1 in w[i]) -> words of two adjacent
// columns: of every four rows the even lane of two neighbours gets the first two and the
// odd lane the others, one exchange for four stores.
template <int WORDS>
__device__ __forceinline__ void join_columns16(uint32_t (&w)[WORDS], int lane) {
  const bool odd = lane & 1;
  const uint32_t first = odd ? 0x1054u : 0x5410u, second = odd ? 0x3276u : 0x7632u;
#pragma unroll
  for (int i = 0; i < WORDS; i += 2) {
    const uint32_t keep = odd ? w[i + 1] : w[i];
    const uint32_t take = __shfl_xor_sync(0xffffffffu, odd ? w[i] : w[i + 1], 1);
    w[i] = __byte_perm(keep, take, first);
    w[i + 1] = __byte_perm(keep, take, second);
  }
}

// R output rows of one column per lane -> memory.  `at` points at (first row, column n),
// rows are `pitch` bytes apart, `left` of them exist (ALL: all of them).
// The common case (32 rows, 32 columns) carries no conditions and 32-bit row offsets: the
// drain of a short main loop is bound by the latency of this loop, one warp a scheduler.
template <int DT, int RN, bool ALL, int R>
__device__ __forceinline__ void store_pairs16(char *at, uint32_t pitch, const float (&f)[R], int left, int lane,
                                              bool both) {
  uint32_t w[R / 2];
#pragma unroll
  for (int i = 0; i < R / 2; ++i) w[i] = cvt_pack2_t<DT, RN>(f[2 * i], f[2 * i + 1]);
  join_columns16(w, lane);
  const int skip = lane & 1 ? 2 : 0;
  char *base = lane & 1 ? at - 2 + 2 * pitch : at;  // (first row + skip, even column)
  uint32_t off = 0u;
#pragma unroll
  for (int i = 0; i < R / 2; i += 2) {
    if (ALL || (both && 2 * i + skip < left)) *reinterpret_cast<uint32_t *>(base + off) = w[i];
    if (ALL || (both && 2 * i + skip + 1 < left)) *reinterpret_cast<uint32_t *>(base + off + pitch) = w[i + 1];
    off += 4u * pitch;
  }
}
template <int DT, int RN, int R>
__device__ __forceinline__ void store_single16(char *at, uint32_t pitch, const float (&f)[R], int left, bool on) {
  if (!on) return;
#pragma unroll
  for (int j = 0; j < R; ++j)
    if (j < left)
      *reinterpret_cast<uint16_t *>(at + static_cast<unsigned long long>(j) * pitch) =
          static_cast<uint16_t>(cvt_pack2_t<DT, RN>(f[j], 0.0f) & 0xffffu);
}
template <int DT, int RN, int R>
__device__ __forceinline__ void store_rows16(char *at, uint32_t pitch, const float (&f)[R], int left, int lane,
                                             bool mine, bool both, bool pairs) {
  if (!pairs) {
    store_single16<DT, RN>(at, pitch, f, left, mine);
  } else if (left >= R && __all_sync(0xffffffffu, both)) {
    store_pairs16<DT, RN, true>(at, pitch, f, left, lane, both);
  } else {
    store_pairs16<DT, RN, false>(at, pitch, f, left, lane, both);
    store_single16<DT, RN>(at, pitch, f, left, mine && !both);  // the last of an odd number of columns
  }
}

// Four rows of four neighbouring lanes' columns: lane l (of four) goes from rows 0..3 of its
// own column to all four columns of row l.  Two exchanges, two values each.
__device__ __forceinline__ float4 transpose4(float a0, float a1, float a2, float a3, int lane) {
  const bool odd = lane & 1, high = lane & 2;
  const float s0 = __shfl_xor_sync(0xffffffffu, odd ? a0 : a1, 1), s1 = __shfl_xor_sync(0xffffffffu, odd ? a2 : a3, 1);
  // rows 0 and 2 in even lanes, 1 and 3 in odd ones, columns (even, odd) of the pair
  const float lo0 = odd ? s0 : a0, hi0 = odd ? a1 : s0, lo1 = odd ? s1 : a2, hi1 = odd ? a3 : s1;
  const float t0 = __shfl_xor_sync(0xffffffffu, high ? lo0 : lo1, 2);
  const float t1 = __shfl_xor_sync(0xffffffffu, high ? hi0 : hi1, 2);
  return high ? make_float4(t0, t1, lo1, hi1) : make_float4(lo0, hi0, t0, t1);
}

// f32 rows added to memory, in 16-byte pieces where addresses and columns allow.  One
// thread alone adds to an element, and its additions to one address keep their order, so
// the sum is the same bits on every run.
__device__ __forceinline__ void add_rows32(char *at, uint32_t pitch, const float (&f)[32], int left, int lane,
                                           bool mine, bool pieces) {
  if (pieces && __all_sync(0xffffffffu, mine)) {
    char *base = at - (lane & 3) * 4 + (lane & 3) * static_cast<unsigned long long>(pitch);
    uint32_t off = 0u;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 v = transpose4(f[j], f[j + 1], f[j + 2], f[j + 3], lane);
      if (j + (lane & 3) < left)
        asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(base + off), "f"(v.x),
                     "f"(v.y), "f"(v.z), "f"(v.w)
                     : "memory");
      off += 4u * pitch;
    }
  } else if (mine) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < left)
        asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(at + static_cast<unsigned long long>(j) * pitch),
                     "f"(f[j])
                     : "memory");
  }
}

// p.row_pitch (bytes) is below 2^26, so 32 rows span less than 2^31.
template <int R>
__device__ __forceinline__ void grouped_store(const GroupedParams &p, char *at, const float (&f)[R], int left,
                                              int lane, bool mine, bool both) {
  const uint32_t pitch = p.row_pitch;
  if (p.out_dtype == KAPYB_F32) {
    if (left >= R && __all_sync(0xffffffffu, mine)) {
      uint32_t off = 0u;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        *reinterpret_cast<float *>(at + off) = f[j];
        off += pitch;
      }
    } else if (mine) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (j < left) *reinterpret_cast<float *>(at + static_cast<unsigned long long>(j) * pitch) = f[j];
    }
    return;
  }
  const bool pairs = p.wide_stores != 0;
  if (p.out_dtype == KAPYB_BF16) {
    if (p.rounding) store_rows16<KAPYB_BF16, 1>(at, pitch, f, left, lane, mine, both, pairs);
    else store_rows16<KAPYB_BF16, 0>(at, pitch, f, left, lane, mine, both, pairs);
  } else {
    if (p.rounding) store_rows16<KAPYB_F16, 1>(at, pitch, f, left, lane, mine, both, pairs);
    else store_rows16<KAPYB_F16, 0>(at, pitch, f, left, lane, mine, both, pairs);
  }
}

// The same rows to places of their own: lane j of the warp holds the output row of f[j],
// -1 for none.
template <int DT, int RN>
__device__ __forceinline__ void scatter_rows16(char *col, uint32_t pitch, const float (&f)[32], int to, int lane,
                                               bool mine, bool both, bool pairs) {
  if (pairs) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = cvt_pack2_t<DT, RN>(f[2 * i], f[2 * i + 1]);
    join_columns16(w, lane);
    char *even = lane & 1 ? col - 2 : col;  // the even column of the two
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = __shfl_sync(0xffffffffu, to, (i & ~1) * 2 + (i & 1) + (lane & 1) * 2);
      if (both && row >= 0) *reinterpret_cast<uint32_t *>(even + static_cast<long long>(row) * pitch) = w[i];
    }
    if (!__any_sync(0xffffffffu, mine && !both)) return;
  }
  const bool on = mine && !(pairs && both);
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const int row = __shfl_sync(0xffffffffu, to, j);
    if (on && row >= 0)
      *reinterpret_cast<uint16_t *>(col + static_cast<long long>(row) * pitch) =
          static_cast<uint16_t>(cvt_pack2_t<DT, RN>(f[j], 0.0f) & 0xffffu);
  }
}
__device__ __forceinline__ void grouped_scatter32(const GroupedParams &p, char *col, const float (&f)[32], int to,
                                                  int lane, bool mine, bool both) {
  const uint32_t pitch = p.row_pitch;
  const bool pairs = p.wide_stores != 0;
  if (p.out_dtype == KAPYB_F32) {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const int row = __shfl_sync(0xffffffffu, to, j);
      if (mine && row >= 0) *reinterpret_cast<float *>(col + static_cast<long long>(row) * pitch) = f[j];
    }
  } else if (p.out_dtype == KAPYB_BF16) {
    if (p.rounding) scatter_rows16<KAPYB_BF16, 1>(col, pitch, f, to, lane, mine, both, pairs);
    else scatter_rows16<KAPYB_BF16, 0>(col, pitch, f, to, lane, mine, both, pairs);
  } else {
    if (p.rounding) scatter_rows16<KAPYB_F16, 1>(col, pitch, f, to, lane, mine, both, pairs);
    else scatter_rows16<KAPYB_F16, 0>(col, pitch, f, to, lane, mine, both, pairs);
  }
}

// ------------------------------------------------------------------- CTA pairs
//
// Each CTA holds 128 of the tile's 256 output columns (its M half) and fetches half of
// its rows (its half of the N side), so a row is pulled from L2 once per 256 columns and
// an SM reads a third fewer operand bytes from shared memory per flop than alone.
//
// Gathered rows.  tile::gather4 costs about 70 clocks per four rows here (measured:
// 37 ns with every lane of a warp issuing), four times the MMA time of the tile they
// feed, so eight more warps gather with 16-byte cp.async, eight lanes a row, straight
// into the swizzled layout, as far ahead as there are free stages.  Their copies
// complete on a barrier of their CTA (cp.async.mbarrier.arrive); one more warp waits
// there, fences the generic proxy that wrote the rows against the async proxy the MMA
// reads them through, and arrives on the leader's barrier, whichever CTA it sits in.
// What has to be ordered are finished copies into an SM's shared memory against the
// tensor core's reads of the same memory, and the proxy fence does that; the arrival
// itself carries the default semantics.  (With a release at cluster scope it waited for
// all copies in flight, 1 to 1.5 us a stage, three times the whole kernel's time.)  Four
// warps fetch 16 KB a stage in 1070 clocks, twice the MMA's time for it (8192 x 4096 x
// 4096 as one group: 259 us); eight nearly keep up.
//
// In the gradient the rows are the contraction: lhs is always gathered (zeros behind
// the group's end and for entries that name no row); grad lies in plan order and comes by
// TMA, but for blocks of 64 positions that have such a place: those the gathering warps
// bring as well, with zeros where lhs has them.  Both roles look at the block's entries.
// The tensor core's f32 additions truncate: a sum loses about 1e-9 of itself per row (9e-6
// over 8192 rows, measured; rounded sums 2e-7).  So an f32 gradient is accumulated 1024
// rows at a time (1e-6 at any length): the epilogue joins two such pieces, one from each
// accumulator slot, rounded to nearest, and adds further pairs to what it has stored.  That
// addition is what it costs: reductions in L2 run at 1.8 TB/s, so 8192 rows of 4096 x 4096
// take 248 us in f32 and 196 in bf16; reading, adding and storing in their place took 1.4 times
// as long.  A group of up to 2048 rows needs none of it.  What is rounded to 16 bits in the end
// stays in one accumulator.

// Adapters: the rows are a plan sorted by adapter whose groups start at multiples of 32
// (gaps and rows without an adapter included), and the tile's main loop over the shared
// weights is followed by more K blocks, for each adapter that has rows in the tile: its
// `up` block times the rows' low-rank products (scale x . down, computed before), into
// exactly the accumulator columns those rows own.  (The kernel is launched with
// programmatic serialization behind the one that computes the products and only waits for
// it there: the plan and everything else it reads were complete when that one started.)
// The products come in two 16-bit
// halves, so the second factor is exact to 16 bits and more.  Nothing is added twice to
// memory and one rounding remains; what a broken adapter produces stays in its own rows.
//
// The accumulator is scaled as a whole at the end, so the products are divided by that
// scale when they are stored.  f16 has no room for a quotient larger than the product, so a
// scale of m 2^-s with 1 <= m < 2 and s > 0 is applied in two steps: the first MMA of an
// adapter's blocks takes 2^-s of what its rows have accumulated (exact), the products are
// divided by m only, and the end multiplies by m.  Rows without an adapter take the whole
// scale at the end; a chunk of 32 rows has the one or the other.

// Gated products: the 128 columns a CTA holds are 64 gate columns and the 64 up columns
// that go with them, so the tile keeps its 256-wide MMA (two sets of columns beside one
// another would take two 128-wide ones and a quarter more operand bytes).  Gate and up
// of one output then sit 64 TMEM lanes apart, in two epilogue warps: they swap half of a
// chunk's rows through shared memory and each finishes 16.

enum PairMode { PAIR_FORWARD = 0, PAIR_GRADIENT = 1, PAIR_ADAPTERS = 2, PAIR_GATED = 3 };

struct PairParams {
  GroupedParams g;
  int gather;            // rows of lhs by cp.async: a plan's order, and always the gradient
  const uint8_t *lhs;    // element (0, 0)
  long long lhs_pitch;   // bytes between rows
  const uint8_t *grad;   // gradient: the same of grad
  long long grad_pitch;
  int piece_kb;          // gradient: K blocks to an accumulator
  FastDiv div_fan;
  uint32_t entries;      // entries of the plan below this name a row of lhs
  // adapters: g.groups = adapters + 1 (the last group: rows without one)
  int rank, up_mn_major;
  int low_rows;          // rows of one half of the low-rank products
  float adapter_alpha;   // what rows with an adapter are multiplied by at the end,
  int adapter_shift;     // and how often their shared part is halved before
};

constexpr int kPairThreads = 192 + 256 + 32 + 128;

struct PairCfg {
  static constexpr int BT = 256;             // rows of a tile
  static constexpr int A_BYTES = 128 * 128;  // per CTA: 128 columns x 64 of the contraction
  static constexpr int B_BYTES = BT / 2 * 128;  // per CTA: half of the tile's rows
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int CTRL_BYTES = 1024;
  static constexpr int TABLE_BYTES = (3 * kGroupedMaxGroups + 8) * 4;
  static constexpr int SWAP_BYTES = 4 * 2 * 16 * 32 * 4;  // warp pairs, directions x 16 rows x 32 lanes
  static constexpr int SMEM_LIMIT = 232448;
  static constexpr int STAGES = (SMEM_LIMIT - 1024 - CTRL_BYTES - TABLE_BYTES - SWAP_BYTES) / STAGE_BYTES;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + CTRL_BYTES + TABLE_BYTES + SWAP_BYTES;
  static constexpr int TMEM_COLS = 2 * BT;   // two accumulator slots
  static_assert(STAGES >= 4, "pipeline too shallow");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Arrives on `bar` once every cp.async this thread has issued so far is complete.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void *tmap, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];"
      :
      : "r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ int round32(int v) { return (v + 31) & ~31; }

// Tile number idx.
template <int MODE>
__device__ __forceinline__ GroupedTile pair_tile(const GroupedParams &p, const GroupedTable &t, int idx) {
  constexpr int BT = PairCfg::BT;
  constexpr int COLS = MODE == PAIR_GATED ? 128 : 256;  // output columns of a tile
  GroupedTile r;
  if constexpr (MODE == PAIR_ADAPTERS) {
    const int all = t.begin[p.groups];  // positions, gaps included
    int m, n;
    raster(idx, (all + BT - 1) / BT, p.n_tiles, m, n);
    r.g = 0;
    r.n0 = n * COLS;
    r.r0 = m * BT;
    r.rows = min(BT, all - r.r0);
    r.num_kb = p.num_kb;
    r.p0 = r.p1 = 0;
  } else if constexpr (MODE == PAIR_GRADIENT) {
    const int per = p.n_tiles * p.k_tiles;
    r.g = idx / per;
    const int in = idx - r.g * per;
    const int n = in / p.k_tiles;
    r.r0 = (in - n * p.k_tiles) * BT;
    r.n0 = n * COLS;
    r.rows = min(BT, p.K - r.r0);
    r.p0 = t.begin[r.g];
    r.p1 = r.p0 + t.count[r.g];
    r.num_kb = (t.count[r.g] + 63) >> 6;
  } else {
    const int q = idx / p.n_tiles;
    const int lo = find_group(t, p.groups, q);
    r.g = lo;
    const int tiles = t.first[lo + 1] - t.first[lo];
    const int in = idx - t.first[lo] * p.n_tiles;
    int m, n;
    raster(in, tiles, p.n_tiles, m, n);
    const int cnt = t.count[lo];
    const int each = round32((cnt + tiles - 1) / tiles);
    r.n0 = n * COLS;
    r.r0 = t.begin[lo] + m * each;
    r.rows = min(each, cnt - m * each);
    r.num_kb = p.num_kb;
    r.p0 = r.p1 = 0;
  }
  r.wide = round32(r.rows);
  return r;
}

// The adapters that have rows in [c0, c1): f(g, first position, last position + 1) for
// each; returns false as soon as f does.
template <class F>
__device__ __forceinline__ bool each_adapter(const GroupedTable &t, int adapters, int c0, int c1, F &&f) {
  int lo = 0, hi = adapters;  // the first adapter that ends behind c0
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (t.begin[mid + 1] > c0) hi = mid;
    else lo = mid + 1;
  }
  for (int g = lo; g < adapters && t.begin[g] < c1; ++g) {
    const int s0 = max(t.begin[g], c0), s1 = min(t.begin[g + 1], c1);
    if (s1 > s0 && !f(g, s0, s1)) return false;
  }
  return true;
}

// tmA: forward: rhs, 3-D (unit axis, other axis, group), boxes of 64 x 128 (K-major) or
// 64 x 64 (MN-major, gated); gradient: grad [positions, cols] in boxes of 64 x 64.
// Rows that come by TMA: lhs in plan order in boxes of 64 x 128 (tmB), 64 x 64 (tmR) and
// 64 x 32 (tmU); adapters: the low-rank products, both halves behind one another, in boxes
// of 64 x 128 (tmB) and 64 x 16 (tmR), and tmU up, 3-D as rhs.
template <int MODE>
__global__ void __launch_bounds__(kPairThreads, 1)
grouped_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmU,
                    const PairParams pp) {
  using Cfg = PairCfg;
  constexpr int STAGES = Cfg::STAGES, BT = Cfg::BT;
  constexpr bool GRAD = MODE == PAIR_GRADIENT, ADAPT = MODE == PAIR_ADAPTERS, GATED = MODE == PAIR_GATED;
  const GroupedParams &p = pp.g;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  uint8_t *sA = smem;
  uint8_t *sB = sA + STAGES * Cfg::A_BYTES;
  uint64_t *bars = reinterpret_cast<uint64_t *>(sB + STAGES * Cfg::B_BYTES);
  uint64_t *full_bar = bars, *empty_bar = bars + STAGES, *tfull_bar = bars + 2 * STAGES, *tempty_bar = tfull_bar + 2;
  uint64_t *rows_bar = tempty_bar + 2;
  uint64_t *swap_bar = rows_bar + STAGES;  // [warp pair][written, read]
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(swap_bar + 8);
  volatile uint32_t *abort_flag = tmem_slot + 1;  // two words
  int *table_mem = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(bars) + Cfg::CTRL_BYTES);
  GroupedTable table{table_mem, table_mem + kGroupedMaxGroups + 2, table_mem + 2 * kGroupedMaxGroups + 4};

  float *swap_mem = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(table_mem) + Cfg::TABLE_BYTES);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int unit = blockIdx.x >> 1, units = gridDim.x >> 1;
  const bool gather = GRAD || ADAPT || pp.gather;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      // the columns' expect_tx in the leader, and the rows': another one there, or with a
      // gather one arrival from each CTA
      ptx::mbar_init(ptx::smem_u32(&full_bar[s]), gather ? 3 : 2);
      ptx::mbar_init(ptx::smem_u32(&rows_bar[s]), 128);  // every thread of a gathering team
      ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(ptx::smem_u32(&tfull_bar[a]), 1);
      ptx::mbar_init(ptx::smem_u32(&tempty_bar[a]), 16);  // eight epilogue warps of each CTA
    }
    for (int i = 0; i < 8; ++i) ptx::mbar_init(ptx::smem_u32(&swap_bar[i]), 2);  // both warps
    abort_flag[0] = 0u;
    abort_flag[1] = p.wait_limit_us;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&tmA);
    ptx::prefetch_tensormap(&tmB);
  }
  if (warp == 1) {
    ptx::tmem_alloc<2>(ptx::smem_u32(tmem_slot), Cfg::TMEM_COLS);
    ptx::tmem_relinquish<2>();
  }
  if constexpr (!ADAPT) {
    // the set-up above ran under the end of the kernel in front; what follows reads its results
    // (with ordinary loads: the compiler may move those marked read-only across the wait)
    ptx::griddep_wait();
    ptx::griddep_launch();
  }
  if constexpr (ADAPT) {
    // group starts only, made ascending as in build_tile_table
    if (warp == 0) {
      int high = 0;
      for (int g0 = 0; g0 <= p.groups; g0 += 32) {
        const int g = g0 + lane;
        int b = g <= p.groups ? min(max(p.offsets[g], 0), p.rows) & ~31 : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, b, off);
          if (lane >= off) b = max(b, o);
        }
        b = max(b, high);
        if (g <= p.groups) table.begin[g] = b;
        high = __shfl_sync(0xffffffffu, b, 31);
      }
    }
  } else if (warp == 0) {
    build_tile_table(p.offsets, p.groups, p.rows, BT, table, lane);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total = GRAD    ? p.groups * p.n_tiles * p.k_tiles
                    : ADAPT ? (table.begin[p.groups] + BT - 1) / BT * p.n_tiles
                            : table.first[p.groups] * p.n_tiles;
  const int low_blocks = ADAPT ? (pp.rank + 63) >> 6 : 0;  // K blocks of an adapter, each twice
  // adapters: K blocks of a tile behind its main loop
  auto extra = [&](const GroupedTile &t) {
    int n = 0;
    if constexpr (ADAPT)
      each_adapter(table, p.groups - 1, t.r0, t.r0 + t.rows, [&](int, int, int) {
        n += 2 * low_blocks;
        return true;
      });
    return n;
  };
  const uint32_t full0 = ptx::mapa(ptx::smem_u32(full_bar), 0);  // the leader's barriers
  auto leader = [](const void *bar) { return ptx::mapa(ptx::smem_u32(bar), 0); };

  // whether a plan entry (a position, without an order) names a row of lhs
  auto names_row = [&](int entry) { return static_cast<uint32_t>(entry) < pp.entries; };

  if (GRAD && warp == 0) {
    // ---------------------------------------------- TMA: the columns' side, gradient
    // The warp loads the entries of four blocks while those in front are fetched.
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int idx = unit; ok && idx < total; idx += units) {
      const GroupedTile t = pair_tile<MODE>(p, table, idx);
      const int n0 = t.n0 + rank * 128;
      int entry[8];
      auto fetch = [&](int kb) {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int q = t.p0 + kb * 64 + 32 * u + lane;
          entry[u] = q >= t.p1 ? -1 : p.order ? p.order[q] : q;
        }
      };
      fetch(0);
      for (int kb0 = 0; ok && kb0 < t.num_kb; kb0 += 4) {
        uint32_t holes = 0u;  // of these four blocks: a position without a row
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (__any_sync(0xffffffffu, !names_row(entry[u]))) holes |= 1u << (u >> 1);
        fetch(kb0 + 4);
        if (lane == 0) {
          for (int kb = kb0; kb < min(kb0 + 4, t.num_kb); ++kb) {
            if (!ptx::mbar_wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1u, abort_flag)) {
              ok = false;
              break;
            }
            const bool whole = !((holes >> (kb - kb0)) & 1u);
            if (rank == 0) {
              if (whole) ptx::mbar_arrive_expect_tx(ptx::smem_u32(&full_bar[stage]), 2u * Cfg::A_BYTES);
              else ptx::mbar_arrive(ptx::smem_u32(&full_bar[stage]));
            }
            if (whole) {
              const uint32_t fb = full0 + stage * 8u;
              const uint32_t a_dst = ptx::smem_u32(sA) + stage * Cfg::A_BYTES;
              tma_load_2d_pair(a_dst, &tmA, fb, n0, t.p0 + kb * 64);
              tma_load_2d_pair(a_dst + 8192, &tmA, fb, n0 + 64, t.p0 + kb * 64);
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0) != 0;
      }
    }
  } else if (!GRAD && warp == 0) {
    // -------------------------------------------------- TMA: the columns' side
    // One lane walks the loop: a load issued by several lanes at once is serialised with
    // its operands moved to uniform registers lane by lane, some 150 clocks each, and at
    // 512 clocks of MMA a stage this role's own time is what the pipeline waits for.
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      // a free stage, its barrier told to expect `bytes` from both CTAs together
      auto open = [&](uint32_t bytes) -> bool {
        if (!ptx::mbar_wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1u, abort_flag)) return false;
        if (rank == 0) ptx::mbar_arrive_expect_tx(ptx::smem_u32(&full_bar[stage]), bytes);
        return true;
      };
      auto advance = [&]() {
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      };
      for (int idx = unit; ok && idx < total; idx += units) {
        const GroupedTile t = pair_tile<MODE>(p, table, idx);
        const int n0 = t.n0 + rank * (GATED ? 64 : 128);
        const int second = GATED ? p.cols : 64;  // from the first 64 columns to the other 64
        for (int kb = 0; kb < t.num_kb; ++kb) {
          if (!open(2u * Cfg::A_BYTES)) {
            ok = false;
            break;
          }
          const uint32_t fb = full0 + stage * 8u;
          const uint32_t a_dst = ptx::smem_u32(sA) + stage * Cfg::A_BYTES;
          if (p.a_mn_major) {
            ptx::tma_load_3d_pair(a_dst, &tmA, fb, n0, kb * 64, t.g);
            ptx::tma_load_3d_pair(a_dst + 8192, &tmA, fb, n0 + second, kb * 64, t.g);
          } else if (GATED) {
            ptx::tma_load_3d_pair(a_dst, &tmA, fb, kb * 64, n0, t.g);
            ptx::tma_load_3d_pair(a_dst + 8192, &tmA, fb, kb * 64, n0 + second, t.g);
          } else {
            ptx::tma_load_3d_pair(a_dst, &tmA, fb, kb * 64, n0, t.g);
          }
          advance();
        }
        if constexpr (ADAPT) {
          if (!ok) break;
          if (idx == unit) ptx::griddep_wait();  // the low-rank products, of the kernel ahead
          ok = each_adapter(table, p.groups - 1, t.r0, t.r0 + t.rows, [&](int g, int s0, int s1) {
            const int mine = (s1 - s0) >> 1;  // rows this CTA fetches: a multiple of 16
            for (int b = 0; b < 2 * low_blocks; ++b) {
              if (!open(2u * (Cfg::A_BYTES + mine * 128u))) return false;
              const uint32_t fb = full0 + stage * 8u;
              const uint32_t a_dst = ptx::smem_u32(sA) + stage * Cfg::A_BYTES;
              const uint32_t b_dst = ptx::smem_u32(sB) + stage * Cfg::B_BYTES;
              const int k0 = (b >> 1) * 64, y = (b & 1) * pp.low_rows + s0 + rank * mine;
              if (pp.up_mn_major) {
                ptx::tma_load_3d_pair(a_dst, &tmU, fb, n0, k0, g);
                ptx::tma_load_3d_pair(a_dst + 8192, &tmU, fb, n0 + 64, k0, g);
              } else {
                ptx::tma_load_3d_pair(a_dst, &tmU, fb, k0, n0, g);
              }
              if (mine == BT / 2) {
                tma_load_2d_pair(b_dst, &tmB, fb, k0, y);
              } else {
                for (int r = 0; r < mine; r += 16) tma_load_2d_pair(b_dst + r * 128, &tmR, fb, k0, y + r);
              }
              advance();
            }
            return true;
          });
        }
      }
    }
  } else if (warp == 6 && !gather) {
    // ------------------------------------------- TMA: rows that lie in plan order
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int idx = unit; ok && idx < total; idx += units) {
        const GroupedTile t = pair_tile<MODE>(p, table, idx);
        const int half = t.wide >> 1;  // rows this CTA fetches
        // one box of 128, 64 or 32 rows, the first that holds them: a load costs its
        // issuing lane more than the rows too many cost
        const int height = half > 64 ? 128 : half > 32 ? 64 : 32;
        const int y = t.r0 + rank * half;
        for (int kb = 0; kb < t.num_kb; ++kb) {
          if (!ptx::mbar_wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          if (rank == 0) ptx::mbar_arrive_expect_tx(ptx::smem_u32(&full_bar[stage]), 2u * height * 128u);
          const uint32_t fb = full0 + stage * 8u;
          const uint32_t b_dst = ptx::smem_u32(sB) + stage * Cfg::B_BYTES;
          if (height == 128) tma_load_2d_pair(b_dst, &tmB, fb, kb * 64, y);
          else if (height == 64) tma_load_2d_pair(b_dst, &tmR, fb, kb * 64, y);
          else tma_load_2d_pair(b_dst, &tmU, fb, kb * 64, y);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ---------------------------------------------------------- MMA issuer
    auto wait_all = [&](uint32_t bar, uint32_t parity) {
      return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, abort_flag)) != 0;
    };
    const bool a_mn = GRAD || p.a_mn_major;
    constexpr bool b_mn = GRAD;
    const uint32_t a_lo0 = ((a_mn ? 8192u : 16u) >> 4) << 16 | (ptx::smem_u32(sA) >> 4);
    const uint32_t b_lo0 = ((b_mn ? 8192u : 16u) >> 4) << 16 | (ptx::smem_u32(sB) >> 4);
    constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    const uint32_t a_step = (a_mn ? 2048u : 32u) >> 4, b_step = (b_mn ? 2048u : 32u) >> 4;
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    // the accumulator goes to the epilogue warps of both CTAs
    auto publish = [&]() {
      if (ptx::elect_one()) {
        ptx::umma_commit<2>(ptx::smem_u32(&tfull_bar[acc]));
        ptx::umma_commit<2>(ptx::mapa(ptx::smem_u32(&tfull_bar[acc]), 1));
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    };
    for (int idx = unit; ok && idx < total; idx += units) {
      const GroupedTile t = pair_tile<MODE>(p, table, idx);
      const uint32_t idesc = ptx::make_idesc_f16(p.bf16, a_mn, b_mn, 256, t.wide);
      // gradient: one accumulator after the other, all but the last published in between
      const int pieces = GRAD ? max(1, (t.num_kb + pp.piece_kb - 1) / pp.piece_kb) : 1;
      uint32_t d = 0u;
      for (int piece = 0; ok && piece < pieces; ++piece) {
        const int kb_end = GRAD ? min(t.num_kb, (piece + 1) * pp.piece_kb) : t.num_kb;
        if (!wait_all(ptx::smem_u32(&tempty_bar[acc]), acc_phase ^ 1u)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        d = tmem_base + static_cast<uint32_t>(acc * BT);
        const int kb_begin = GRAD ? piece * pp.piece_kb : 0;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!wait_all(ptx::smem_u32(&full_bar[stage]), phase)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            const uint32_t a_lo = a_lo0 + static_cast<uint32_t>(stage) * (Cfg::A_BYTES >> 4);
            const uint32_t b_lo = b_lo0 + static_cast<uint32_t>(stage) * (Cfg::B_BYTES >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t ad = (static_cast<uint64_t>(hi) << 32) | (a_lo + k * a_step);
              const uint64_t bd = (static_cast<uint64_t>(hi) << 32) | (b_lo + k * b_step);
              ptx::umma_k<2, 0>(d, ad, bd, idesc, kb != kb_begin || k != 0 ? 1u : 0u);
            }
            ptx::umma_commit<2>(ptx::smem_u32(&empty_bar[stage]));
            ptx::umma_commit<2>(ptx::mapa(ptx::smem_u32(&empty_bar[stage]), 1));
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if constexpr (GRAD) {
          if (ok && piece + 1 < pieces) publish();
        }
      }
      if constexpr (ADAPT) {
        if (!ok) break;
        const uint32_t u_step = (pp.up_mn_major ? 2048u : 32u) >> 4;
        const uint32_t u_lo0 = ((pp.up_mn_major ? 8192u : 16u) >> 4) << 16 | (ptx::smem_u32(sA) >> 4);
        ok = each_adapter(table, p.groups - 1, t.r0, t.r0 + t.rows, [&](int, int s0, int s1) {
          const uint32_t idesc_s = ptx::make_idesc_f16(p.bf16, pp.up_mn_major, 0, 256, s1 - s0);
          for (int b = 0; b < 2 * low_blocks; ++b) {
            if (!wait_all(ptx::smem_u32(&full_bar[stage]), phase)) return false;
            ptx::tc_fence_after();
            const int steps = (min(64, pp.rank - (b >> 1) * 64) + 15) >> 4;
            if (ptx::elect_one()) {
              const uint32_t a_lo = u_lo0 + static_cast<uint32_t>(stage) * (Cfg::A_BYTES >> 4);
              const uint32_t b_lo = b_lo0 + static_cast<uint32_t>(stage) * (Cfg::B_BYTES >> 4);
              for (int k = 0; k < steps; ++k) {
                const uint64_t ad = (static_cast<uint64_t>(hi) << 32) | (a_lo + k * u_step);
                const uint64_t bd = (static_cast<uint64_t>(hi) << 32) | (b_lo + k * 2u);
                if (b == 0 && k == 0 && pp.adapter_shift > 0)
                  ptx::umma_pair_f16_scaled(pp.adapter_shift, d + (s0 - t.r0), ad, bd, idesc_s);
                else
                  ptx::umma_k<2, 0>(d + (s0 - t.r0), ad, bd, idesc_s, 1u);
              }
              ptx::umma_commit<2>(ptx::smem_u32(&empty_bar[stage]));
              ptx::umma_commit<2>(ptx::mapa(ptx::smem_u32(&empty_bar[stage]), 1));
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          return true;
        });
      }
      if (!ok) break;
      publish();
    }
  } else if ((warp >= 2 && warp < 6) || warp >= 15) {
    // ------------------------------------------------------------ epilogue
    // Two teams of four warps, one warp to each quarter of TMEM's lanes: they take the
    // tile's chunks of 32 rows in turn.
    const int team = warp >= 15 ? 1 : 0;
    const int q = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    uint32_t swaps = 0;  // gated: exchanges so far
    bool alive = true;
    (void)swaps;
    for (int idx = unit; idx < total; idx += units) {
      const GroupedTile t = pair_tile<MODE>(p, table, idx);
      const int warp_n = GATED ? t.n0 + rank * 64 + (q & 1) * 32 : t.n0 + rank * 128 + q * 32;
      const int n = warp_n + lane;
      const bool mine = n < p.cols, both = (n | 1) < p.cols;
      float bias = 0.0f;  // gated: of this warp's side
      if (p.bias != nullptr && mine && (!ADAPT || p.bias_axis == 1)) {
        const long long at = (ADAPT ? 0ll : static_cast<long long>(t.g) * p.bias_cols) + n;
        bias = load_as_f32(p.bias, p.bias_dtype, GATED && q >= 2 ? at + p.cols : at);
      }
      const int pieces = GRAD ? max(1, (t.num_kb + pp.piece_kb - 1) / pp.piece_kb) : 1;
      for (int piece = 0; piece < pieces; piece += 2) {
        // two pieces: from this slot and the other one, which is a phase on when this is slot 1
        const bool two = GRAD && piece + 1 < pieces;
        if (!__all_sync(0xffffffffu,
                        ptx::mbar_wait(ptx::smem_u32(&tfull_bar[acc]), acc_phase, abort_flag) &&
                            (!two || ptx::mbar_wait(ptx::smem_u32(&tfull_bar[acc ^ 1]),
                                                    acc == 0 ? acc_phase : acc_phase ^ 1u, abort_flag)))) {
          alive = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t src = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * BT);
        const uint32_t tempty = leader(&tempty_bar[acc]);
        const bool warp_has = warp_n < p.cols && team * 32 < t.rows;
        char *out = static_cast<char *>(p.out) + (GRAD ? t.g * p.group_bytes : 0ll) +
                    static_cast<long long>(t.r0) * p.row_pitch + n * (p.out_dtype == KAPYB_F32 ? 4ll : 2ll);
        for (int c = team * 32; c < t.rows && warp_has; c += 64) {
          float f[32];
          if (!GRAD || t.num_kb > 0) {
            uint32_t v[32];
            ptx::tmem_ld_32x32(src + c, v);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
            if (GRAD && two) {
              ptx::tmem_ld_32x32(src + (acc == 0 ? BT : -BT) + c, v);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) f[i] += __uint_as_float(v[i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = 0.0f;
          }
          if (c + 64 >= t.rows) {  // this warp's last
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              ptx::mbar_arrive_cluster(tempty);
              if (two) ptx::mbar_arrive_cluster(leader(&tempty_bar[acc ^ 1]));
            }
          }
          if constexpr (ADAPT) {
            // rows go where the plan took them from; lane l holds row c + l's number
            int to = c + lane < t.rows ? p.order[t.r0 + c + lane] : -1;
            if (to >= p.src_rows) to = -1;
            const float alpha = t.r0 + c < table.begin[p.groups - 1] ? pp.adapter_alpha : p.alpha;
            if (p.bias != nullptr && p.bias_axis == 0) {
              const float row_bias = to >= 0 ? load_as_f32(p.bias, p.bias_dtype, to) : 0.0f;
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j] = f[j] * alpha + __shfl_sync(0xffffffffu, row_bias, j);
              grouped_activation(p.activation, f);
            } else {
              grouped_finish32(p, f, alpha, bias);
            }
            grouped_scatter32(p, static_cast<char *>(p.out) + n * (p.out_dtype == KAPYB_F32 ? 4ll : 2ll), f, to, lane,
                              mine, both);
          } else if constexpr (GATED) {
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = f[j] * p.alpha + bias;
            // the gate's warp hands over its rows 16 .. 31 and finishes 0 .. 15, the up
            // columns' warp the other way round
            const bool up_side = q >= 2;
            float *box = swap_mem + (team * 2 + (q & 1)) * 1024;
            const uint32_t written = ptx::smem_u32(&swap_bar[(team * 2 + (q & 1)) * 2]), read = written + 8u;
            float g[16], u[16];
            if (swaps > 0 && !__all_sync(0xffffffffu, ptx::mbar_wait(read, (swaps - 1) & 1, abort_flag))) {
              alive = false;
              break;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) (up_side ? box : box + 512)[j * 32 + lane] = up_side ? f[j] : f[16 + j];
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(written);
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(written, swaps & 1, abort_flag))) {
              alive = false;
              break;
            }
            ++swaps;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float other = (up_side ? box + 512 : box)[j * 32 + lane];
              g[j] = up_side ? other : f[j];
              u[j] = up_side ? f[16 + j] : other;
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(read);
            grouped_activation(p.activation, g);
#pragma unroll
            for (int j = 0; j < 16; ++j) g[j] *= u[j];
            const int first = c + (up_side ? 16 : 0);
            grouped_store(p, out + static_cast<long long>(first) * p.row_pitch, g, t.rows - first, lane, mine, both);
          } else {
            grouped_finish32(p, f, p.alpha, bias);
            char *at = out + static_cast<long long>(c) * p.row_pitch;
            if (GRAD && piece > 0) {  // f32: to what the pieces before have left there
              add_rows32(at, p.row_pitch, f, t.rows - c, lane, mine, p.wide_stores);
            } else {
              grouped_store(p, at, f, t.rows - c, lane, mine, both);
            }
          }
        }
        if (!alive) break;
        if (!warp_has) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            ptx::mbar_arrive_cluster(tempty);
            if (two) ptx::mbar_arrive_cluster(leader(&tempty_bar[acc ^ 1]));
          }
        }
        if (two) {
          acc_phase ^= 1u;  // both slots are done with: the same slot, a phase on
        } else {
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1u;
        }
      }
      if (!alive) break;
    }
  } else if (warp == 14 && gather) {
    // ------------------------- finished copies of this CTA -> the leader's barrier
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int idx = unit; ok && idx < total; idx += units) {
      const GroupedTile t = pair_tile<MODE>(p, table, idx);
      const int blocks = t.num_kb + extra(t);
      for (int kb = 0; kb < blocks; ++kb) {
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&rows_bar[stage]), phase, abort_flag))) {
          ok = false;
          break;
        }
        ptx::fence_proxy_async_smem();
        if (lane == 0) ptx::mbar_arrive_cluster(full0 + stage * 8u);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp >= 6 && warp < 14 && gather) {
    // -------------------------------------------------------------- gather
    // Two teams of four warps take stages in turn, so that one waits and reports while
    // the other keeps the copies coming: the copies alone take 460 clocks of a 512-clock
    // stage (36 bytes a clock), all eight warps on every stage 630 with the rest.
    const int tid = (threadIdx.x - 192) & 127, team = (threadIdx.x - 192) >> 7;
    const int piece = tid & 7, row0 = tid >> 3;  // 16-byte piece of rows row0, + 16, ...
    int stage = 0;
    uint32_t phase = 0, turn = 0;  // turn: stages so far
    bool ok = true;
    auto wait_slot = [&]() {
      return __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1u, abort_flag)) != 0;
    };
    auto advance = [&]() {
      ++turn;
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    };
    // source row of a plan entry, -1 for none
    auto row_of = [&](int entry) -> int {
      if (!names_row(entry)) return -1;
      return p.order ? pp.div_fan.div(entry) : entry;
    };
    if constexpr (GRAD) {
      for (int idx = unit; ok && idx < total; idx += units) {
        const GroupedTile t = pair_tile<MODE>(p, table, idx);
        const int half = t.wide >> 1;
        const int col = t.r0 + rank * half + piece * 8, n = t.n0 + rank * 128 + piece * 8;
        uint32_t bytes[2], n_bytes[2];  // of the two 64-column chunks
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          bytes[c] = static_cast<uint32_t>(max(0, min(16, (p.K - col - c * 64) * 2)));
          n_bytes[c] = static_cast<uint32_t>(max(0, min(16, (p.cols - n - c * 64) * 2)));
        }
        const bool need[2] = {piece * 8 < half, 64 + piece * 8 < half};
        const uint8_t *base = pp.lhs + (bytes[0] ? col * 2ll : 0ll);
        const uint32_t next_chunk = bytes[1] ? 128u : 0u;
        // the plan's entries of this team's next block (all 64, two a lane) are loaded as soon
        // as it has issued one, and only turned into row numbers when they are needed
        int entry[2];
        auto fetch = [&](int kb) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int q = t.p0 + kb * 64 + 32 * u + lane;
            entry[u] = q >= t.p1 ? -1 : p.order ? p.order[q] : q;
          }
        };
        fetch((turn & 1u) == static_cast<uint32_t>(team) ? 0 : 1);
        for (int kb = 0; kb < t.num_kb; ++kb, advance()) {
          if ((turn & 1u) != static_cast<uint32_t>(team)) continue;
          if (!wait_slot()) {
            ok = false;
            break;
          }
          const uint32_t off = row0 * 128 + ((piece ^ (row0 & 7)) << 4);
          const uint32_t dst = ptx::smem_u32(sB) + stage * Cfg::B_BYTES + off;
          int from[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) from[i] = row_of(__shfl_sync(0xffffffffu, entry[i >> 1], row0 + 16 * (i & 1)));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint8_t *src = base + (from[i] >= 0 ? from[i] * pp.lhs_pitch : 0ll);
            if (need[0]) cp_async16(dst + i * 2048, src, from[i] >= 0 ? bytes[0] : 0u);
            if (need[1]) cp_async16(dst + 8192 + i * 2048, src + next_chunk, from[i] >= 0 ? bytes[1] : 0u);
          }
          if (__any_sync(0xffffffffu, !names_row(entry[0]) || !names_row(entry[1]))) {  // grad's, which TMA leaves out
            const uint32_t a_dst = ptx::smem_u32(sA) + stage * Cfg::A_BYTES + off;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int q = t.p0 + kb * 64 + row0 + 16 * i;
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const uint32_t have = from[i] >= 0 ? n_bytes[c] : 0u;
                cp_async16(a_dst + c * 8192 + i * 2048,
                           pp.grad + (have ? q * pp.grad_pitch + (n + c * 64) * 2ll : 0ll), have);
              }
            }
          }
          cp_async_arrive(ptx::smem_u32(&rows_bar[stage]));
          fetch(kb + 2);
        }
      }
    } else {
      constexpr int kRows = BT / 32;
      // this thread's entries of a tile, loaded while the tile in front of it is fetched
      int entry[kRows];
      auto fetch = [&](int idx) {
        if (idx >= total) return;
        const GroupedTile t = pair_tile<MODE>(p, table, idx);
        const int half = t.wide >> 1;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int r = rank * half + row0 + 16 * i;  // row of the tile
          entry[i] = row0 + 16 * i < half && r < t.rows ? p.order ? p.order[t.r0 + r] : t.r0 + r : -1;
        }
      };
      fetch(unit);
      for (int idx = unit; ok && idx < total; idx += units) {
        const GroupedTile t = pair_tile<MODE>(p, table, idx);
        const int half = t.wide >> 1;
        const uint8_t *row[kRows];  // nullptr: zeros
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int from = row_of(entry[i]);
          row[i] = from >= 0 ? pp.lhs + from * pp.lhs_pitch : nullptr;
        }
        fetch(idx + units);
        const int blocks = t.num_kb + extra(t);
        for (int kb = 0; kb < blocks; ++kb, advance()) {
          if ((turn & 1u) != static_cast<uint32_t>(team)) continue;
          if (!wait_slot()) {
            ok = false;
            break;
          }
          const int k = kb * 64 + piece * 8;
          const uint32_t bytes = static_cast<uint32_t>(max(0, min(16, (p.K - k) * 2)));
          const uint32_t dst = ptx::smem_u32(sB) + stage * Cfg::B_BYTES + row0 * 128 + ((piece ^ (row0 & 7)) << 4);
          const long long at = bytes ? k * 2ll : 0ll;
          // (the adapters' blocks bring their rows by TMA: nothing to copy, only to arrive)
#pragma unroll
          for (int i = 0; i < kRows; ++i)
            if (row0 + 16 * i < half && kb < t.num_kb)
              cp_async16(dst + i * 2048, row[i] ? row[i] + at : pp.lhs, row[i] ? bytes : 0u);
          cp_async_arrive(ptx::smem_u32(&rows_bar[stage]));
        }
      }
    }
    cp_async_wait_all();
  }

  // ---------------------------------------------------------------- teardown
  ptx::tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0u) {
    if (threadIdx.x == 0) atomicExch(p.status, kStatusTimeout);
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 200000ull) {
    }
    __syncthreads();
  }
  // the peer may still address this CTA's barriers and shared memory
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<2>(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace kapyb
