// Matrix products over expert segments of any length: 16-bit operands (forward, gradient
// of the rows, gradient of the weights) and 8-bit integers with a scale for each token and
// channel.  Segment e is the rows ends[e-1] <= t < ends[e] of the row operand.
//
//   kFwd  y[t, n]     = sum_k x[t, k] w[e, n, k]        x, w read along k
//   kDx   dx[t, k]    = sum_n dy[t, n] w[e, n, k]       w read across its rows
//   kDw   dw[e, n, k] = sum_{t in e} dy[t, n] x[t, k]   both read across their rows
//
// The tensor core's M axis is the output's contiguous axis (weight rows n for kFwd, weight
// columns k for kDx and kDw) and its N axis is the output's rows.  So the ragged axis of
// kFwd and kDx is N, which an MMA takes in steps of 16: a segment's last tile costs what
// its rows cost, not a full 128, and one token occupies 16 columns of one 128-row weight
// tile.  Operands read across their rows are "MN-major": 64 of M or N in a 128-byte
// swizzled row, one such row for each index of the sum.
//
// Persistent CTAs, in pairs (M = 256 over both), or single ones where segments are short:
// warp 0 feeds a ring of TMA stages, warp 1 issues tcgen05.mma into one of two TMEM
// accumulators, warps 4 and following turn the other one into output rows.
// A sum is one fp32 (or exact int32) accumulator in TMEM from the first product to the
// last; where a cluster shares it, two to eight of them, added up in fp32 (int32) in the order
// of its parts.  The output is rounded once.
//
// Rows that a tile loads beyond its segment are other output rows in kFwd and kDx, computed
// and never stored.  In kDw they would enter the sum: the last warp clears them (in both operands,
// so an infinity there cannot meet a zero) in the segment's last stage before its MMA.
#include <cudaTypedefs.h>
#include <cuda_fp16.h>

#include <atomic>

#include "b2m_common.cuh"
#include "b2m_host.h"
#include "pair_ring.cuh"

namespace b2m {
namespace {

enum Mode { kFwd = 0, kDx = 1, kDw = 2 };

constexpr int kM = 128;            // output columns of a CTA's part of a tile (TMEM lanes)
constexpr int kRowBytes = 128;     // one swizzled shared-memory row
constexpr int kMaxExperts = 1024;
constexpr int kMostWarps = 13;
constexpr int kABytes = kM * kRowBytes;
constexpr int kBand = 8;           // row tiles walked together, so that they share a weight tile in L2
constexpr int kSortMost = 256;     // experts up to which segments are sorted by length
constexpr int kFeed = 4;           // tiles found ahead
constexpr int kSplitTiles = 64;    // most tiles of a launch whose CTAs share sums
constexpr int kLeastSplit = 16;    // blocks of a sum that is shared
constexpr int kStagePitch = 144;   // bytes between two staged output rows of 128: no bank is hit twice

// A tile is NT output rows by 128 output columns, or, for a pair of CTAs, by 256: each CTA
// keeps the operand rows and the accumulator of its own 128 columns and half of the row
// operand, and the leader's MMAs (cta_group::2) read both halves.
//
// Where there are too few tiles for the SMs, the CTAs of a cluster share a tile along its sum
// (kSplit): each multiplies its part of the blocks, and each adds up all parts for its share
// of the output columns.
template <int kRows, bool kTwoCtas, bool kSplitSum, int kRing, int kOnSm>
struct Shape {
  static constexpr int NT = kRows;
  static constexpr bool kPair = kTwoCtas;
  static constexpr bool kSplit = kSplitSum;
  static constexpr int kCtas = kPair ? 2 : 1;
  static constexpr int kTileM = kM * kCtas;
  static constexpr int kBRows = NT / kCtas;         // rows of the row operand in one CTA
  static constexpr int kStep = 16 * kCtas;          // granularity of N in an MMA
  static constexpr int kStageBytes = kABytes + kBRows * kRowBytes;
  static constexpr int kStages = kRing;
  static constexpr int kResident = kOnSm;  // CTAs on an SM
  static constexpr int kEpiWarps = NT > 64 ? 8 : 4;  // two sets of four, or one: 32 rows at a time each
  static constexpr uint32_t kTmemCols = 2 * NT;
};
using Wide = Shape<256, true, false, 6, 1>;
// For weight gradients of up to 128 columns, which leave one CTA of a pair without any.
using Slim = Shape<256, false, false, 4, 1>;
// Two CTAs on an SM: one streams while the other starts or ends a tile, and a few rounds of
// tiles share the memory out evenly.
using Narrow = Shape<32, false, false, 4, 2>;
// For one round of tiles or less: the whole SM's ring for one CTA.
using Single = Shape<32, false, false, 9, 1>;
using Split = Shape<32, false, true, 4, 2>;
using Split64 = Shape<64, false, true, 7, 1>;
constexpr int kMostParts = 8;

// What the CTAs of a split tile hand to each other: for every part, the accumulators of the
// columns that this CTA adds up.  A cluster has one tile at most.
template <bool kSplit, int kRows>
struct Join {};
template <int kRows>
struct Join<true, kRows> {
  uint64_t full;  // every part's accumulators are here
  alignas(16) uint32_t part[kRows * kM];
};

// Of a pair: what the CTAs need to know of each other's copies when a wait has run out.
template <bool kPair, int kStages>
struct Ends {};
template <int kStages>
struct Ends<true, kStages> {
  PairRing<kStages> ring;
};

// One output tile: rows [row0, row0 + cols) of the output (kDw: of expert e's output),
// columns from m0.  k_blocks == 0: all zero, nothing is multiplied.  e < 0: no tile is left.
struct alignas(16) Tile {
  int e;
  int m0;
  int row0;
  int cols;
  int k_blocks;
  int sum0;      // kDw: first row of the sum
  int sum_rows;  // kDw: rows of the sum
  int k0;        // first block of this CTA's part of the sum
};

template <class S>
struct Control {
  uint64_t full[S::kStages];    // operands landed; of a pair, the leader's counts both CTAs' copies
  uint64_t empty[S::kStages];   // the stage's MMAs are done
  uint64_t landed[S::kStages];  // kDw, last stage of a segment: this CTA's copies landed
  uint64_t cleared[S::kStages];  // of a pair the leader's: the rows behind the segment are cleared
  uint64_t tfull[2];            // accumulator ready
  uint64_t tempty[2];           // accumulator read; of a pair, the leader's counts both CTAs' warps
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
  int32_t warp_max[kMostWarps];
  int32_t warp_sum[kMostWarps];
  uint64_t fed[kFeed];             // a tile is there
  uint64_t taken[kFeed];           // every role has read it
  Tile feed[kFeed];
  alignas(16) int32_t start[kMaxExperts + 4];  // first row of segment e; [E] = end of the last, [E + 1] = rows
  alignas(16) int32_t tile0[kMaxExperts + 2];  // row tiles before the segment at place r of the walk
  uint16_t seg[kMaxExperts + 2];   // the segment at place r
  // 32 output rows of 64 columns, for two warps each
  alignas(16) uint8_t staging[S::kSplit ? 1 : S::kEpiWarps / 2][S::kSplit ? 16 : 32 * kStagePitch];
  Join<S::kSplit, S::NT> join;
  Ends<S::kPair, S::kStages> ends;
};

// Warps: 0 and 2 feed the ring, 1 issues MMAs, 3 finds tiles, 4 and following write outputs, the
// last one of kDw clears tails.
template <class S>
constexpr int threads_of(int mode) {
  return (4 + S::kEpiWarps + (mode == kDw ? 1 : 0)) * 32;
}

template <class S>
constexpr size_t smem_bytes() {
  return size_t(S::kStages) * S::kStageBytes + sizeof(Control<S>) + 1024;
}

// Tensor maps: the operand whose rows or columns are the output's columns, and the row operand
// with boxes of one to four quarters of the rows that a CTA can hold (kDw: rows[3] alone).
struct Maps {
  CUtensorMap cols;
  CUtensorMap rows[4];
};

// Whether tiles take boxes of i + 1 quarters: an MMA takes half of a narrow tile's rows at least.
template <class S>
__host__ __device__ constexpr bool used_map(int i) {
  return (i + 1) * (S::kBRows / 4) % (S::kStep / S::kCtas) == 0;
}

struct Params {
  const int32_t* ends;   // nullptr: one segment of all rows
  int32_t experts;
  int32_t segments;      // experts, plus one for the rows behind the last segment when they are cleared
  int64_t rows;
  int32_t m_dim;         // extent of the output's contiguous axis
  int32_t m_tiles;       // tiles along it
  int32_t tile_bits;     // log2 of a tile's most output rows
  int32_t c_dim;         // kDw: output rows of one expert
  int32_t c_tiles;       // kDw
  int32_t k_blocks;      // kFwd, kDx: blocks of the sum
  int32_t parts;         // CTAs that share a tile's sum
  uint32_t m_magic;      // for division by m_tiles, by kBand * m_tiles and (kDw) by m_tiles * c_tiles
  uint32_t band_magic;
  uint32_t expert_magic;
  uint32_t idesc;        // instruction descriptor without N
  void* out;
  int64_t ldo;
  int64_t out_expert;    // kDw: elements between two experts' outputs
  int32_t out_type;
  bool wide_out;         // 16-bit output rows are 16-byte aligned
  const float* a_scale;  // integers: scale of each row
  const float* w_scale;  // integers: scale of each weight row, [experts, m_dim]
  int32_t* status;
  uint64_t timeout_ns;
};

template <class S>
__device__ __forceinline__ int find_segment(const Control<S>* C, int segments, int slot) {
  int lo = 0, hi = segments - 1;  // the last segment whose first tile is <= slot
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (C->tile0[mid] <= slot)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Columns of a tile as an MMA takes them: N is a multiple of 16 (of 32 for a pair).
template <class S>
__device__ __forceinline__ int mma_cols(int cols) {
  return (cols + S::kStep - 1) / S::kStep * S::kStep;
}

// a / d with magic = ceil(2^32 / d), for a < 2^31: the product is the quotient or one more.
__device__ __forceinline__ int quotient(int a, int d, uint32_t magic) {
  if (d == 1) return a;
  const uint32_t q = __umulhi(static_cast<uint32_t>(a), magic);
  return static_cast<int>(q * static_cast<uint32_t>(d) > static_cast<uint32_t>(a) ? q - 1 : q);
}

template <int kMode, class S>
__device__ __forceinline__ Tile tile_at(const Params& p, const Control<S>* C, int t) {
  Tile r;
  int tiles, i;  // row tiles of the segment, and this tile's index among the segment's tiles
  if (kMode == kDw) {
    const int per = p.m_tiles * p.c_tiles;
    const int place = quotient(t, per, p.expert_magic);
    r.e = C->seg[place];
    i = t - place * per;
    tiles = p.c_tiles;
  } else {
    const int place = find_segment(C, p.segments, quotient(t, p.m_tiles, p.m_magic));
    r.e = C->seg[place];
    i = t - C->tile0[place] * p.m_tiles;
    tiles = C->tile0[place + 1] - C->tile0[place];
  }
  int m = i, c = 0;
  if (tiles > 1) {
    const int band = tiles > kBand ? quotient(i, kBand * p.m_tiles, p.band_magic) : 0;
    const int in_band = i - band * kBand * p.m_tiles;
    const int wide = min(kBand, tiles - band * kBand);
    m = in_band / wide;
    c = band * kBand + in_band - m * wide;
  }
  r.m0 = m * S::kTileM;
  if (kMode == kDw) {
    r.row0 = c << p.tile_bits;
    r.cols = min(1 << p.tile_bits, p.c_dim - r.row0);
    r.sum0 = C->start[r.e];
    r.sum_rows = C->start[r.e + 1] - C->start[r.e];
    r.k_blocks = (r.sum_rows + 63) >> 6;
  } else {
    // A segment's tiles have about the same rows: one of few rows costs four fifths of a full
    // one (258 rows: 256 and 2 take 912 cycles a block of the sum, twice 129 take 800).  Sizes
    // are whole steps of an MMA; with eight tiles and more they come to the most that a tile has,
    // and the last of fewer tiles keeps a row (256: more than 256 (n - 1) rows in n < 8 tiles of at
    // most rows / n + 31; 128: of 96 or 128; 64: of 64).
    const int rows = C->start[r.e + 1] - C->start[r.e];
    const int each = S::kPair && tiles > 1 ? mma_cols<S>((rows + tiles - 1) / tiles) : S::NT;
    r.row0 = C->start[r.e] + c * each;
    r.cols = min(each, rows - c * each);
    r.k_blocks = r.e < p.experts ? p.k_blocks : 0;
    r.sum0 = 0;
    r.sum_rows = 0;
  }
  return r;
}

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// Waits of a whole warp: true when every lane has seen the phase complete.  The slow path,
// with its clock and its limit, stays out of line: in a call of a few microseconds each line
// of code is fetched once, and fetching is part of its time.
__device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, const Params& p, int32_t code, volatile int* abort) {
  return mbar_wait(bar, parity, p.timeout_ns, p.status, code, abort);
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, const Params& p, int32_t code, int* abort) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, wait_on(bar, parity, p, code, abort));
}

// Segment starts and row-tile counts from `ends`.  An end that is below an earlier one or
// outside [0, rows] is taken as the nearest one that is in order, and noted in the status word.
//
// Narrow launches: by one warp, each lane with a run of consecutive segments.  They are the
// calls of a few tokens, and barriers between all warps would cost them more.
template <class S>
__device__ __forceinline__ void plan_narrow(const Params& p, Control<S>* C, int lane) {
  constexpr int kBatch = 4;
  const int rows = static_cast<int>(p.rows);
  const int per = (p.experts + 31) >> 5;
  const int e0 = lane * per, e1 = min(e0 + per, p.experts);
  int top = 0, lowest = rows;
  bool bad = false;
  for (int b = e0; b < e1; b += kBatch) {
    int v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) v[i] = b + i < e1 ? (p.ends ? __ldg(p.ends + b + i) : rows) : rows;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (b + i < e1) {
        lowest = min(lowest, v[i]);
        bad |= v[i] < top || v[i] > rows;  // below 0 is below `top`
        top = max(top, min(v[i], rows));
        C->start[b + i + 1] = top;
      }
  }
  int before = top;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before = max(before, o);
  }
  before = __shfl_up_sync(0xffffffffu, before, 1);
  if (lane == 0) before = 0;
  if ((bad || lowest < before) && blockIdx.x == 0) set_status(p.status, B2M_STATUS_BAD_ROUTING);
  int prev = before, sum = 0;
  for (int e = e0; e < e1; ++e) {
    const int end = max(C->start[e + 1], before);
    C->start[e + 1] = end;
    C->tile0[e] = sum;
    C->seg[e] = static_cast<uint16_t>(e);
    sum += (end - prev + S::NT - 1) / S::NT;
    prev = end;
  }
  int at = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, at, off);
    if (lane >= off) at += o;
  }
  const int total = __shfl_sync(0xffffffffu, at, 31);
  at -= sum;
  for (int e = e0; e < e1; ++e) C->tile0[e] += at;
  const int last = __shfl_sync(0xffffffffu, max(prev, before), 31);
  if (lane == 0) {
    C->start[0] = 0;
    C->start[p.experts + 1] = rows;
    C->tile0[p.experts] = total;
    C->seg[p.experts] = static_cast<uint16_t>(p.experts);
    // the rows behind the last segment, as one more segment
    C->tile0[p.experts + 1] = total + (rows - last + S::NT - 1) / S::NT;
  }
}

// Wide launches: by all threads, long segments before short ones in the walk.
template <int kMode, class S>
__device__ __forceinline__ void plan_wide(const Params& p, Control<S>* C) {
  const int nt = 1 << p.tile_bits;
  constexpr int kThreads = threads_of<S>(kMode);
  static_assert(kThreads >= kSortMost && kSortMost % 32 == 0 && kSortMost <= kMaxExperts, "one segment a thread");
  constexpr int kPer = (kMaxExperts + kThreads - 1) / kThreads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = static_cast<int>(p.rows);
  int v[kPer], top = 0, lowest = rows;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = tid * kPer + i;
    v[i] = e < p.experts ? (p.ends ? __ldg(p.ends + e) : rows) : rows;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    lowest = min(lowest, v[i]);
    bad |= v[i] < top || v[i] > rows;  // below 0 is below `top`
    if (tid * kPer + i < p.experts) top = max(top, min(v[i], rows));
    v[i] = top;
  }
  int scan = top;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, scan, off);
    if (lane >= off) scan = max(scan, o);
  }
  if (lane == 31) C->warp_max[warp] = scan;
  __syncthreads();
  int prev = __shfl_up_sync(0xffffffffu, scan, 1);
  if (lane == 0) prev = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w)
    if (w < warp) prev = max(prev, C->warp_max[w]);
  if ((bad || lowest < prev) && blockIdx.x == 0) set_status(p.status, B2M_STATUS_BAD_ROUTING);
  int n[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = tid * kPer + i;
    const int end = max(v[i], prev);
    if (e < p.experts) C->start[e] = prev;
    if (e == p.experts - 1) C->start[p.experts] = end;
    n[i] = e < p.experts ? (end - prev + nt - 1) >> p.tile_bits : 0;
    prev = end;
  }
  if (tid == 0) C->start[p.experts + 1] = rows;
  if (p.experts > 1 && p.experts <= kSortMost) {
    // Counted into 32 classes of length, four to an octave from 32 to 4096 rows, where tiles
    // differ in cost; within a class segments stay in order.  (Exact ranks, each segment compared with
    // all others, took 4.1 us more at 256 segments: 24 rows each, 256 x 128, 13.8 us a call, 9.7.)
    __syncthreads();
    int32_t(*count)[32] = reinterpret_cast<int32_t(*)[32]>(C->tile0);  // [warp][class, longest first]
    int cls = 31, rank = 0;
    if (warp < kSortMost / 32) {
      count[warp][lane] = 0;
      if (tid < p.experts) {
        const int len = C->start[tid + 1] - C->start[tid];
        const int octave = 31 - __clz(max(len, 1));
        if (len >= 32) cls = max(0, 30 - 4 * (octave - 5) - (len >> (octave - 2) & 3));
      }
      const bool real = tid < p.experts;
      __syncwarp();
      const uint32_t same = __match_any_sync(0xffffffffu, real ? cls : 32);
      rank = __popc(same & ((1u << lane) - 1));
      if (real && rank == 0) count[warp][cls] = __popc(same);
    }
    __syncthreads();
    if (warp == 0) {  // lane: class
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kSortMost / 32; ++w) {
        const int n = count[w][lane];
        count[w][lane] = sum;
        sum += n;
      }
      int before = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += o;
      }
      before -= sum;
#pragma unroll
      for (int w = 0; w < kSortMost / 32; ++w) count[w][lane] += before;
    }
    __syncthreads();
    if (tid < p.experts) C->seg[count[warp][cls] + rank] = static_cast<uint16_t>(tid);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = tid * kPer + i;
      const int e = r < p.experts ? C->seg[r] : 0;
      n[i] = r < p.experts ? (C->start[e + 1] - C->start[e] + nt - 1) >> p.tile_bits : 0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (tid * kPer + i < p.experts) C->seg[tid * kPer + i] = static_cast<uint16_t>(tid * kPer + i);
  }
  if (tid == 0) C->seg[p.experts] = static_cast<uint16_t>(p.experts);
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += n[i];
  int acc = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, acc, off);
    if (lane >= off) acc += o;
  }
  if (lane == 31) C->warp_sum[warp] = acc;
  __syncthreads();
  int at = acc - sum, total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) at += C->warp_sum[w];
    total += C->warp_sum[w];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = tid * kPer + i;
    if (r < p.experts) C->tile0[r] = at;
    at += n[i];
  }
  if (tid == 0) {
    C->tile0[p.experts] = total;
    // the rows behind the last segment, as one more segment
    C->tile0[p.experts + 1] = total + ((rows - C->start[p.experts] + nt - 1) >> p.tile_bits);
  }
}

// Place of this CTA in its pair, and of the pair in the grid.
struct Where {
  uint32_t rank;
  int first;   // first tile
  int stride;  // pairs (or CTAs, or clusters that share tiles) in the grid
  int part;    // of a tile's sum
};

// Warp 3, one lane: this CTA's tiles, on their way to its other roles.  Finding a tile takes
// some hundred cycles of divisions and searches, longer than a short sum.  (The CTAs of a pair
// find the same tiles each for itself: handing them over needs releases at cluster scope, which
// wait for the epilogue's output stores, 3000 cycles a tile.)
//
// A wide launch of up to 256 segments walks them from long classes of length to short ones (all
// below 32 rows are one class, all from 6144 on another), with more segments as they come; all
// pairs go side by side on the same segment, and every second round of tiles is dealt out
// backwards, which evens the shares out.  Long segments are limited by the tensor cores and short ones by memory, but doing both
// at once lost more than it gave: pairs that share weights or rows drift apart and read them
// again (16384 rows over 32 experts of 4096 x 7168, lengths by Zipf 1.2: 3.6 GB instead of
// 2.1 GB, 862 us instead of 800), and stores wait behind the others' loads (weight gradient:
// 1305 us instead of 935 with pairs of their own for the short segments).
template <int kMode, class S>
__device__ __forceinline__ void feed_tiles(const Params& p, Control<S>* C, int num_tiles, const Where& at) {
  uint32_t s = 0, phase = 0;
  for (int i = 0;; ++i) {
    const int t = i * at.stride + (S::kPair && (i & 1) ? at.stride - 1 - at.first : at.first);
    Tile r{};
    r.e = -1;
    if (t < num_tiles) r = tile_at<kMode, S>(p, C, t);
    if (S::kSplit) {
      const int blocks = r.k_blocks;
      r.k0 = blocks * at.part / p.parts;
      r.k_blocks = blocks * (at.part + 1) / p.parts - r.k0;
      if (kMode == kDw) {
        r.sum0 += r.k0 * 64;
        r.sum_rows = min(r.sum_rows - r.k0 * 64, r.k_blocks * 64);
      }
    }
    const bool last = i * at.stride >= num_tiles;  // every CTA has had its last tile
    if (r.e >= 0 || last) {
      if (!mbar_try_wait(&C->taken[s], phase ^ 1) &&
          !wait_on(&C->taken[s], phase ^ 1, p, B2M_STATUS_TIMEOUT_PRODUCER, &C->abort))
        return;
      C->feed[s] = r;
      mbar_arrive(&C->fed[s]);
      if (++s == kFeed) s = 0, phase ^= 1;
    }
    if (last) return;
  }
}

// The receiving end, for a whole warp.
template <class S>
struct TileFeed {
  Control<S>* C;
  const Params& p;
  uint32_t s = 0, phase = 0;

  __device__ __forceinline__ TileFeed(const Params& p_, Control<S>* c) : C(c), p(p_) {}

  // False after a timeout, else the next tile (e < 0: none is left).
  __device__ __forceinline__ bool next(Tile& r) {
    if (!wait_warp(&C->fed[s], phase, p, B2M_STATUS_TIMEOUT_MMA, &C->abort)) return false;
    const Tile v = C->feed[s];
    // equal in all lanes, which the compiler then knows
    r.e = __shfl_sync(0xffffffffu, v.e, 0);
    r.m0 = __shfl_sync(0xffffffffu, v.m0, 0);
    r.row0 = __shfl_sync(0xffffffffu, v.row0, 0);
    r.cols = __shfl_sync(0xffffffffu, v.cols, 0);
    r.k_blocks = __shfl_sync(0xffffffffu, v.k_blocks, 0);
    r.sum0 = __shfl_sync(0xffffffffu, v.sum0, 0);
    r.sum_rows = __shfl_sync(0xffffffffu, v.sum_rows, 0);
    r.k0 = S::kSplit ? __shfl_sync(0xffffffffu, v.k0, 0) : 0;
    if ((threadIdx.x & 31) == 0) mbar_arrive(&C->taken[s]);
    if (++s == kFeed) s = 0, phase ^= 1;
    return true;
  }
};

// Shared-memory descriptor of an operand whose 128-byte swizzled rows run along M or N:
// 64 elements of M (N) in a row, eight rows (indices of the sum) in a group, groups 1024
// bytes apart, the next 64 of M (N) `chunk_bytes` further on.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr, uint32_t chunk_bytes) {
  uint64_t d = smem_desc_sw128(saddr) & ~(static_cast<uint64_t>(0x3FFF) << 16);
  return d | static_cast<uint64_t>(chunk_bytes >> 4) << 16;
}

// D = A B (first) or D += A B.
template <bool kI8, bool kPair>
__device__ __forceinline__ void mma_first(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
#define B2M_MMA(group, kind)                                                                      \
  asm volatile(                                                                                   \
      "{\n\t.reg .pred p;\n\t"                                                                    \
      "setp.ne.b32 p, %4, 0;\n\t"                                                                 \
      "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),  \
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)                                         \
      : "memory")
  if (kI8 && kPair)
    B2M_MMA("2", "i8");
  else if (kI8)
    B2M_MMA("1", "i8");
  else if (kPair)
    B2M_MMA("2", "f16");
  else
    B2M_MMA("1", "f16");
#undef B2M_MMA
}
template <bool kI8, bool kPair>
__device__ __forceinline__ void mma_more(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
#define B2M_MMA(group, kind)                                                                           \
  asm volatile("tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, 1;" ::"r"(d_tmem),     \
               "l"(adesc), "l"(bdesc), "r"(idesc)                                                       \
               : "memory")
  if (kI8 && kPair)
    B2M_MMA("2", "i8");
  else if (kI8)
    B2M_MMA("1", "i8");
  else if (kPair)
    B2M_MMA("2", "f16");
  else
    B2M_MMA("1", "f16");
#undef B2M_MMA
}

// Tiled loads whose bytes are counted on the barrier at `bar`, an address in the cluster's
// shared memory (of a pair: the leader's barrier).  No multicast.
template <bool kPair>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y) {
  if (kPair)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
template <bool kPair>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y,
                                        int32_t z) {
  if (kPair)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Warps 0 and 2, every second stage each: this CTA's operands.  Like the MMA warp, all lanes
// run the loop and one is elected for the copies, so that addresses and coordinates are
// uniform across the warp.  One such warp took 330 cycles to issue a stage (380 for kDx, which
// has three copies in it), about what a short segment's MMAs take.
template <int kMode, bool kI8, class S>
__device__ __forceinline__ void producer(const Maps& maps, const Params& p, uint8_t* smem, Control<S>* C,
                                         uint32_t rank, int which) {
  constexpr int kElems = kI8 ? 128 : 64;  // elements in a 128-byte row
  const uint32_t smem0 = smem_u32(smem);
  const uint32_t full0 = smem_u32(&C->full[0]), landed0 = smem_u32(&C->landed[0]);
  const uint32_t full0_leader = S::kPair ? mapa_shared(full0, 0) : full0;
  const uint32_t landed0_own = S::kPair ? mapa_shared(landed0, rank) : landed0;
  uint32_t kg = 0;      // stages of the tiles before this one
  uint32_t issued = 0;  // one more than the last stage that this warp issued
  uint32_t tails = 0, last_tail = 0;  // bit s: parity of the next use of landed[s]; the last use of stage s was one
  bool alive = true;
  TileFeed<S> feed(p, C);
  Tile r;
  while (alive) {
    alive = feed.next(r);
    if (!alive || r.e < 0) break;
    const int half = mma_cols<S>(r.cols) / S::kCtas;  // rows of the row operand in this CTA
    // One box of the row operand for each stage, of the smallest size that holds the tile's rows:
    // as many 32-row boxes as it needs took longer to issue than the rows that they leave out
    // (E=32, 224 rows each: 419 us, 385 with single boxes).  kDw: boxes of 64 columns.
    constexpr int kQuarter = S::kBRows / 4;
    const int size = (half + kQuarter - 1) / kQuarter;
    const int boxes = (half + 63) / 64;
    const uint32_t bytes = kABytes + (kMode == kDw ? boxes * 64 : size * kQuarter) * kRowBytes;
    const CUtensorMap* const map_cols = &maps.cols;
    const CUtensorMap* const map_rows = &maps.rows[kMode == kDw ? 3 : size - 1];
    const int row = r.row0 + static_cast<int>(rank) * half;
    const int m0 = r.m0 + static_cast<int>(rank) * kM;
    int kb = (kg + which) & 1;
    uint32_t s = (kg + kb) % S::kStages, phase = ((kg + kb) / S::kStages) & 1;
    for (; kb < r.k_blocks; kb += 2) {
      if (!wait_warp(&C->empty[s], phase ^ 1, p, B2M_STATUS_TIMEOUT_PRODUCER, &C->abort)) {
        alive = false;
        break;
      }
      const uint32_t a = smem0 + s * S::kStageBytes, b = a + kABytes;
      const bool tail = kMode == kDw && r.sum_rows - kb * 64 < 64;  // the last warp comes between the copies and the MMA
      const uint32_t bar = (tail ? landed0_own : full0_leader) + s * 8;
      if (elect_one()) {
        if constexpr (S::kPair) C->ends.ring.bytes[s] = tail ? 0 : bytes;
        if (tail) {
          if (rank == 0) mbar_arrive(&C->full[s]);
          mbar_arrive_expect_tx(&C->landed[s], bytes);
        } else if (rank == 0) {
          mbar_arrive_expect_tx(&C->full[s], S::kCtas * bytes);
        }
        if (kMode == kFwd) {
          load_3d<S::kPair>(a, map_cols, bar, (r.k0 + kb) * kElems, m0, r.e);
          load_2d<S::kPair>(b, map_rows, bar, (r.k0 + kb) * kElems, row);
        } else if (kMode == kDx) {
          load_3d<S::kPair>(a, map_cols, bar, m0, (r.k0 + kb) * 64, r.e);
          load_3d<S::kPair>(a + kABytes / 2, map_cols, bar, m0 + 64, (r.k0 + kb) * 64, r.e);
          load_2d<S::kPair>(b, map_rows, bar, (r.k0 + kb) * kElems, row);
        } else {
          const int sum = r.sum0 + kb * 64;
          load_2d<S::kPair>(a, map_cols, bar, m0, sum);
          load_2d<S::kPair>(a + kABytes / 2, map_cols, bar, m0 + 64, sum);
          load_2d<S::kPair>(b, map_rows, bar, row, sum);
          if (boxes > 1) load_2d<S::kPair>(b + 64 * kRowBytes, map_rows, bar, row + 64, sum);
          if (S::kBRows > 128)
            for (int i = 2; i < boxes; ++i) load_2d<S::kPair>(b + i * 64 * kRowBytes, map_rows, bar, row + i * 64, sum);
        }
      }
      __syncwarp();
      issued = kg + kb + 1;
      if (kMode == kDw) {
        last_tail = tail ? last_tail | 1u << s : last_tail & ~(1u << s);
        if (tail) tails ^= 1u << s;
      }
      if ((s += 2) >= S::kStages) s -= S::kStages, phase ^= 1;
    }
    kg += r.k_blocks;
  }
  // Before the CTA exits, the copies of the stages still in use have landed: they are when the
  // stage is released.  After a timeout nothing may release it; then this warp waits, again
  // within the limit, for its last copies themselves.  Those that a pair's leader counts are
  // settled when both CTAs have stopped (leave_pair).
  const uint32_t first = issued > S::kStages ? issued - S::kStages : 0;
  for (uint32_t i = first; i < issued && alive; ++i)
    if (((i ^ which) & 1) == 0)
      alive = wait_warp(&C->empty[i % S::kStages], (i / S::kStages) & 1, p, B2M_STATUS_TIMEOUT_DRAIN, &C->abort);
  for (uint32_t i = first; i < issued && !alive; ++i) {
    const uint32_t s = i % S::kStages;
    if (((i ^ which) & 1) != 0) continue;
    if (kMode == kDw && (last_tail >> s & 1))
      wait_on(&C->landed[s], (tails >> s & 1) ^ 1, p, B2M_STATUS_TIMEOUT_DRAIN, nullptr);
    else if (!S::kPair)
      wait_on(&C->full[s], (i / S::kStages) & 1, p, B2M_STATUS_TIMEOUT_DRAIN, nullptr);
  }
  if constexpr (S::kPair)
    if ((threadIdx.x & 31) == 0) C->ends.ring.issued[which] = issued;
  __syncwarp();
}

// The last warp of kDw: when this CTA's copies of a segment's last, partly filled stage have landed,
// clears the rows behind the segment, up to the next step of the MMA, and tells the (leader's)
// MMA warp.
template <class S>
__device__ __forceinline__ void clear_tails(const Params& p, uint8_t* smem, Control<S>* C, int lane) {
  uint32_t kg = 0, phases = 0;  // bit s: parity of the next use of landed[s]
  TileFeed<S> feed(p, C);
  Tile r;
  while (true) {
    if (!feed.next(r) || r.e < 0) return;
    const int left = r.sum_rows & 63;
    kg += r.k_blocks;
    if (left == 0) continue;
    const int chunks = 2 + (mma_cols<S>(r.cols) / S::kCtas + 63) / 64;  // 64 columns each, of both operands
    const int s = (kg - 1) % S::kStages;
    if (!wait_warp(&C->landed[s], (phases >> s) & 1, p, B2M_STATUS_TIMEOUT_MMA, &C->abort)) return;
    phases ^= 1u << s;
    const int vecs = ((left + 15) / 16 * 16 - left) * (kRowBytes / 16);  // 16-byte pieces of a chunk
    uint8_t* rows = smem + s * S::kStageBytes + left * kRowBytes;
    for (int i = lane; i < vecs * chunks; i += 32) {
      const int chunk = i / vecs;
      *reinterpret_cast<uint4*>(rows + chunk * 64 * kRowBytes + (i - chunk * vecs) * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (S::kPair)
        mbar_arrive_cluster(mapa_shared(smem_u32(&C->cleared[s]), 0));
      else
        mbar_arrive(&C->cleared[s]);
    }
  }
}

// Warp 1 (of a pair: the leader's).  Short segments make this loop's own instructions count:
// the tensor cores need 157 cycles for a block of the sum (four MMAs) with N = 32, 256 with
// N = 128 and 512 with N = 256.  All lanes run the loop and one is elected to issue, so that
// descriptors live in uniform registers; only the low word of a descriptor changes, and only
// a block's first MMA carries a predicate.  Measured alone, with operands in place: 208, 256
// and 512 cycles; with 64-bit descriptor sums and a predicate each it was 371, 371 and 512,
// and a loop run by one lane took 510 whatever N.
template <int kMode, bool kI8, class S>
__device__ __forceinline__ void mma_warp(const Params& p, uint8_t* smem, Control<S>* C, uint32_t tmem_base) {
  // 32 bytes of the sum in each step: within the row, or 16 rows further on
  constexpr uint32_t a_step = kMode == kFwd ? 2 : 128, b_step = kMode == kDw ? 128 : 2;
  const uint32_t as = smem_u32(smem), bs = as + kABytes;
  const uint64_t adesc = kMode == kFwd ? smem_desc_sw128(as) : smem_desc_mn(as, kABytes / 2);
  const uint64_t bdesc = kMode == kDw ? smem_desc_mn(bs, 64 * kRowBytes) : smem_desc_sw128(bs);
  const uint32_t a_lo = static_cast<uint32_t>(adesc), b_lo = static_cast<uint32_t>(bdesc);
  const uint64_t a_hi = adesc >> 32 << 32, b_hi = bdesc >> 32 << 32;
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
  uint32_t s = 0, phase = 0, used = 0, tails = 0;  // tails, bit s: parity of the next use of cleared[s]
  bool alive = true, any = false;
  TileFeed<S> feed(p, C);
  Tile r;
  while (alive) {
    if (!feed.next(r) || r.e < 0) break;
    if (r.k_blocks == 0) continue;
    const uint32_t buf = used & 1;
    if (!wait_warp(&C->tempty[buf], ((used >> 1) & 1) ^ 1, p, B2M_STATUS_TIMEOUT_MMA, &C->abort)) break;
    const uint32_t d = tmem + buf * S::NT;
    const uint32_t idesc = p.idesc | (static_cast<uint32_t>(mma_cols<S>(r.cols)) >> 3 << 17);
    for (int kb = 0; kb < r.k_blocks; ++kb) {
      bool ok = wait_warp(&C->full[s], phase, p, B2M_STATUS_TIMEOUT_MMA, &C->abort);
      const int left = kMode == kDw ? r.sum_rows - kb * 64 : 64;
      if (kMode == kDw && left < 64) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait_cluster(&C->cleared[s], (tails >> s) & 1, p.timeout_ns, p.status,
                                                             B2M_STATUS_TIMEOUT_MMA, &C->abort));
        tails ^= 1u << s;
      }
      if (!ok) {
        alive = false;
        break;
      }
      tc_fence_after();
      const uint32_t a_s = a_lo + s * (S::kStageBytes >> 4), b_s = b_lo + s * (S::kStageBytes >> 4);
      if (elect_one()) {
        mma_first<kI8, S::kPair>(d, a_hi | a_s, b_hi | b_s, idesc, kb > 0);
#pragma unroll
        for (int k = 1; k < 4; ++k)
          if (kMode != kDw || k * 16 < left)
            mma_more<kI8, S::kPair>(d, a_hi | (a_s + a_step * k), b_hi | (b_s + b_step * k), idesc);
        if (S::kPair)
          mma_commit_pair(&C->empty[s], 0x3);
        else
          mma_commit(&C->empty[s]);
        if (kb == r.k_blocks - 1) {
          if (S::kPair)
            mma_commit_pair(&C->tfull[buf], 0x3);
          else
            mma_commit(&C->tfull[buf]);
        }
      }
      __syncwarp();
      any = true;
      if (++s == S::kStages) s = 0, phase ^= 1;
    }
    ++used;
  }
  // every MMA issued here has completed before TMEM is freed
  if (any) {
    if (elect_one()) {
      if (S::kPair)
        mma_commit_pair(&C->mma_done, 0x1);
      else
        mma_commit(&C->mma_done);
    }
    __syncwarp();
    wait_on(&C->mma_done, 0, p, B2M_STATUS_TIMEOUT_DRAIN, nullptr);
  }
  __syncwarp();
}

// 16 TMEM lanes x 32 columns.  Thread l gets, for each group g of eight columns, lane l/4
// (v[4g], v[4g+1]) and lane l/4 + 8 (v[4g+2], v[4g+3]) of columns 8g + 2(l%4) and the next.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Four 8x8 matrices of 16-bit values, each stored transposed: thread l gives the address of
// row l%8 of matrix l/8.
__device__ __forceinline__ void store_matrices_t(uint32_t saddr, const uint32_t (&m)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(saddr), "r"(m[0]),
               "r"(m[1]), "r"(m[2]), "r"(m[3])
               : "memory");
}

__device__ __forceinline__ uint32_t pack_16bit(float a, float b, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Two epilogue warps that share a staging block.
struct Duo {
  int bar;   // named barrier
  int half;  // which 32 of the 64 output columns this warp holds
  __device__ __forceinline__ void sync() const { named_bar_sync(bar, 64); }
  // Whether both warps say yes: the warps leave the kernel's loop together or not at all.
  __device__ __forceinline__ bool both(bool yes) const {
    int r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, %2, 64, p;\n\t"
        "selp.b32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(static_cast<int>(yes)), "r"(bar)
        : "memory");
    return r != 0;
  }
};

// 64 output columns (TMEM lanes of two warps) of 32 output rows (TMEM columns), rounded to 16
// bits.  An output row is contiguous along the lanes, so the block is transposed on its way
// out: pairs of rows in a register, 8x8 matrices through stmatrix into the staging block, and
// from there whole 128-byte lines, four in a warp's store.  (The weight gradient of E=32,
// 4096 x 7168 took 1.08 ms with two-byte stores straight from the registers and 0.66 ms with
// half lines, both bound by the L1's stores.)  Lines that do not start on 16 bytes, or end
// inside 16, go out as pairs of elements, a line in a warp's store, four lines read before the
// first is written: bf16, 3855 x 4745, a sum of 240, 32 us, 58 line by line and 90 with 16 bytes
// by single elements in each thread; 20 at 4744.
// `v` holds the block's accumulators, or will when the loads in flight are done, and then takes
// the next block's from `next` (0: there is none) while this one is written: the weight gradient
// above takes 600 us, 635 with the loads at the start of the block.
// `o`: the block's first element; n rows and m columns of it exist.  kLong: code of its own for each type
// and for whole blocks (integers, 8192 x 8192, k = 256, to bf16 49 us, 54 without); where a CTA has a tile
// or two, fetching more code costs more than it saves (integers, one row, 28672 x 4096: 23.7 us, 24.5).
template <bool kI8, bool kLong>
__device__ __forceinline__ void emit_16bit(uint16_t* o, int64_t ldo, int n, int m, bool wide, bool bf16, bool zero,
                                           uint32_t next, uint8_t* staging, const Duo& duo, float a_scale,
                                           const float (&w_scale)[4], int lane, float (&v)[32]) {
  if (!zero) tmem_ld_wait();
  uint32_t packed[4][4];
  const uint32_t to = smem_u32(staging) + (lane & 7) * kStagePitch + duo.half * 64 + (lane >> 3) * 16;
  const auto pack = [&](bool to_bf16) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float s0 = kI8 ? __shfl_sync(0xffffffffu, a_scale, 8 * g + 2 * (lane & 3)) : 1.0f;
      const float s1 = kI8 ? __shfl_sync(0xffffffffu, a_scale, 8 * g + 2 * (lane & 3) + 1) : 1.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // lanes 8i .. 8i + 7
        float x = v[(i >> 1) * 16 + 4 * g + 2 * (i & 1)], y = v[(i >> 1) * 16 + 4 * g + 2 * (i & 1) + 1];
        if (kI8) {
          x = __int2float_rn(__float_as_int(x)) * s0 * w_scale[i];
          y = __int2float_rn(__float_as_int(y)) * s1 * w_scale[i];
        }
        packed[g][i] = pack_16bit(x, y, to_bf16);
      }
    }
  };
  if (zero) {
#pragma unroll
    for (int i = 0; i < 16; ++i) packed[i >> 2][i & 3] = 0;
  } else if (!kLong) {
    pack(bf16);
  } else if (bf16) {
    pack(true);
  } else {
    pack(false);
  }
  if (next) {
    tmem_ld_16x32(next, v);
    tmem_ld_16x32(next + (16u << 16), v + 16);
  }
#pragma unroll
  for (int g = 0; g < 4; ++g) store_matrices_t(to + 8 * g * kStagePitch, packed[g]);
  duo.sync();
  constexpr int kAtOnce = 4;  // rows
  if (wide && (m & 7) == 0) {
    const int at = (lane & 7) * 8;  // this thread's eight columns
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = 16 * duo.half + 4 * i + (lane >> 3);
      if (j < n && at < m)
        *reinterpret_cast<uint4*>(o + j * ldo + at) = *reinterpret_cast<const uint4*>(staging + j * kStagePitch + at * 2);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; i += kAtOnce) {
      // a row that starts between two words: its first element alone, then pairs from the second on
      const int j0 = 16 * duo.half + i;
      uint32_t pair[kAtOnce], first[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const uint16_t* from = reinterpret_cast<const uint16_t*>(staging + (j0 + k) * kStagePitch);
        const int at = 2 * lane + (static_cast<int>(reinterpret_cast<uintptr_t>(o + (j0 + k) * ldo) >> 1) & 1);
        first[k] = from[0];
        pair[k] = from[at] | static_cast<uint32_t>(from[at + 1]) << 16;
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        uint16_t* d = o + (j0 + k) * ldo;
        const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(d) >> 1) & 1, at = 2 * lane + odd;
        const bool exists = j0 + k < n;
        if (exists && at + 1 < m) *reinterpret_cast<uint32_t*>(d + at) = pair[k];
        if (exists && at + 1 == m) d[at] = static_cast<uint16_t>(pair[k]);
        if (exists && odd && lane == 0) d[0] = static_cast<uint16_t>(first[k]);
      }
    }
  }
  duo.sync();
}

// The same in fp32: a row's 32 columns are 128 contiguous bytes across the warp.
template <bool kI8, bool kLong>
__device__ __forceinline__ void emit_fp32(float* o, int64_t ldo, int n, int m, bool zero, uint32_t taddr,
                                          float a_scale, float w_scale, int lane) {
  float v[32];
  if (!zero) {
    tmem_ld32(taddr, v);
    tmem_ld_wait();
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float s = kI8 ? __shfl_sync(0xffffffffu, a_scale, j) : 0.0f;
    if (kI8) v[j] = __int2float_rn(__float_as_int(v[j])) * s * w_scale;
    if (zero) v[j] = 0.0f;
  }
  if (lane < m) {
    float* d = o + lane;
    if (kLong && n == 32) {
#pragma unroll
      for (int j = 0; j < 32; ++j, d += ldo) *d = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j, d += ldo)
        if (j < n) *d = v[j];
    }
  }
  __syncwarp();
}

template <int kMode, bool kI8, class S>
__device__ __forceinline__ void epilogue(const Params& p, Control<S>* C, uint32_t tmem_base, uint32_t rank, int warp,
                                         int lane) {
  const int q = warp & 3;  // TMEM lane quarter of this warp
  const int h = (warp - 4) >> 2;
  const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
  const Duo duo{1 + h * 2 + (q >> 1), q & 1};
  uint8_t* staging = C->staging[duo.bar - 1];
  uint32_t used = 0;
  TileFeed<S> feed(p, C);
  Tile r;
  while (true) {
    if (!duo.both(feed.next(r)) || r.e < 0) return;
    const int buf = used & 1;
    const int m0 = r.m0 + static_cast<int>(rank) * kM + q * 32;
    const int m = min(32, p.m_dim - m0);  // columns of this warp that exist, and of both
    const int m_duo = min(64, p.m_dim - m0 + duo.half * 32);
    const bool zero = r.k_blocks == 0;
    float w_lane = 0.0f, w_scale[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of column m0 + lane; of the columns 8i + lane / 4
    if (kI8 && !zero) {
      if (lane < m) w_lane = __ldg(p.w_scale + static_cast<int64_t>(r.e) * p.m_dim + m0 + lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) w_scale[i] = __shfl_sync(0xffffffffu, w_lane, 8 * i + (lane >> 2));
    }
    // the scales of a block's rows are on their way while the block before them is written
    float a_next = 0.0f;
    if (kI8 && !zero && h * 32 + lane < r.cols) a_next = __ldg(p.a_scale + r.row0 + h * 32 + lane);
    if (!zero) {
      const bool ok = wait_warp(&C->tfull[buf], (used >> 1) & 1, p, B2M_STATUS_TIMEOUT_EPILOGUE, &C->abort);
      if (!duo.both(ok)) return;
      tc_fence_after();
    }
    const int64_t base = (kMode == kDw ? r.e * p.out_expert : 0) + static_cast<int64_t>(r.row0) * p.ldo + m0;
    constexpr int kEvery = S::kEpiWarps / 4 * 32;
    constexpr bool kLong = S::NT > 64;
    float v[32];
    if (!zero && p.out_type != B2M_FP32 && h * 32 < r.cols && m_duo > 0) {
      const uint32_t taddr = tmem_base + lane_off + static_cast<uint32_t>(buf * S::NT + h * 32);
      tmem_ld_16x32(taddr, v);
      tmem_ld_16x32(taddr + (16u << 16), v + 16);
    }
    for (int c = h * 32; c < r.cols && m_duo > 0; c += kEvery) {
      const int n = min(32, r.cols - c);
      const uint32_t taddr = tmem_base + lane_off + static_cast<uint32_t>(buf * S::NT + c);
      const float a_scale = a_next;
      if (kLong && kI8 && !zero && c + kEvery + lane < r.cols) a_next = __ldg(p.a_scale + r.row0 + c + kEvery + lane);
      const int64_t o = base + c * p.ldo;
      if (p.out_type == B2M_FP32)
        emit_fp32<kI8, kLong>(static_cast<float*>(p.out) + o, p.ldo, n, m, zero, taddr, a_scale, w_lane, lane);
      else
        emit_16bit<kI8, kLong>(static_cast<uint16_t*>(p.out) + o - duo.half * 32, p.ldo, n, m_duo, p.wide_out,
                               p.out_type == B2M_BF16, zero,
                               kLong && !zero && c + kEvery < r.cols ? taddr + kEvery : 0u, staging, duo, a_scale,
                               w_scale, lane, v);
      if (!kLong) break;  // a tile is one block
    }
    if (!zero) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (S::kPair)
          mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&C->tempty[buf]), 0));
        else
          mbar_arrive(&C->tempty[buf]);
      }
      ++used;
    }
  }
}

// One output element.
__device__ __forceinline__ void put(void* out, int64_t at, int32_t type, float v) {
  if (type == B2M_FP32)
    static_cast<float*>(out)[at] = v;
  else
    static_cast<uint16_t*>(out)[at] = static_cast<uint16_t>(pack_16bit(v, 0.0f, type == B2M_BF16));
}

// Epilogue of a split sum, warps 4-7.  Of the tile's 128 columns (TMEM lanes), CTA d of the
// cluster adds up columns d * 128 / parts and following: every CTA sends each of them the
// accumulators of its part, [part][row][column], and the owner adds them in the order of the
// parts, so the result does not depend on who comes first.
template <int kMode, bool kI8, class S>
__device__ __forceinline__ void epilogue_split(const Params& p, Control<S>* C, uint32_t tmem_base, const Where& at,
                                               int warp, int lane) {
  const int q = warp & 3;
  const int share = kM / p.parts;  // columns of one CTA: 16, 32 or 64
  const int bits = 31 - __clz(share);
  const int column = q * 32 + lane, owner = column >> bits, in_share = column & (share - 1);
  TileFeed<S> feed(p, C);
  Tile r;
  if (!feed.next(r) || r.e < 0) return;
  const int64_t out = (kMode == kDw ? r.e * p.out_expert : 0) + static_cast<int64_t>(r.row0) * p.ldo + r.m0;
  if (kMode != kDw && r.e >= p.experts) {  // rows of no expert
    if (at.part == 0 && r.m0 + column < p.m_dim)
      for (int j = 0; j < r.cols; ++j) put(p.out, out + j * p.ldo + column, p.out_type, 0.0f);
    return;
  }
  // A thread adds up one column of every 128 / share rows.
  const int mine = at.part * share + in_share;
  constexpr int kBlocks = S::NT / 32;  // of 32 rows
  float a_lane[kBlocks] = {}, w_scale = 0.0f;  // a_lane[h]: of row 32 h + lane
#pragma unroll
  for (int h = 0; h < kBlocks; ++h)
    if (kI8 && 32 * h + lane < r.cols) a_lane[h] = __ldg(p.a_scale + r.row0 + 32 * h + lane);
  if (kI8 && r.m0 + mine < p.m_dim) w_scale = __ldg(p.w_scale + static_cast<int64_t>(r.e) * p.m_dim + r.m0 + mine);
  const bool some = kMode != kDw || r.k_blocks > 0;  // a short segment leaves parts without a block
  if (some && !wait_warp(&C->tfull[0], 0, p, B2M_STATUS_TIMEOUT_EPILOGUE, &C->abort)) return;
  tc_fence_after();
  const uint32_t to =
      mapa_shared(smem_u32(&C->join.part[at.part * S::NT * share + in_share]), static_cast<uint32_t>(owner));
#pragma unroll
  for (int h = 0; h < kBlocks; ++h) {
    float v[32] = {};
    if (some) {
      tmem_ld32(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + 32 * h, v);
      tmem_ld_wait();
    }
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (32 * h + j < r.cols)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + static_cast<uint32_t>((32 * h + j) * share * 4)),
                     "f"(v[j])
                     : "memory");
  }
  tc_fence_before();
  __syncwarp();
  if ((lane & (share - 1)) == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&C->join.full), owner));

  const bool ok = mbar_wait_cluster(&C->join.full, 0, p.timeout_ns, p.status, B2M_STATUS_TIMEOUT_EPILOGUE, &C->abort);
  if (!ok) return;
  __syncwarp();
  // four rows at a time: one by one, a thread's 16 rows of two parts took 3 us
  constexpr int kAtOnce = 4;
  for (int i0 = column; i0 - lane < r.cols << bits; i0 += kAtOnce * kM) {
    uint32_t sum[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) sum[u] = (i0 + u * kM) >> bits < r.cols ? C->join.part[i0 + u * kM] : 0;
    for (int k = 1; k < p.parts; ++k)
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if ((i0 + u * kM) >> bits >= r.cols) continue;
        const uint32_t add = C->join.part[k * S::NT * share + i0 + u * kM];
        sum[u] = kI8 ? sum[u] + add : __float_as_uint(__uint_as_float(sum[u]) + __uint_as_float(add));
      }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int j = (i0 + u * kM) >> bits;
      float y = __uint_as_float(sum[u]);
      if (kI8) {
        const float a_scale = __shfl_sync(0xffffffffu, kBlocks > 1 && j >= 32 ? a_lane[kBlocks - 1] : a_lane[0], j & 31);
        y = __int2float_rn(static_cast<int>(sum[u])) * a_scale * w_scale;
      }
      if (j < r.cols && r.m0 + mine < p.m_dim) put(p.out, out + j * p.ldo + mine, p.out_type, y);
    }
  }
}

template <int kMode, bool kI8, class S>
__global__ void __launch_bounds__(threads_of<S>(kMode), S::kResident)
    grouped_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Control<S>* C = reinterpret_cast<Control<S>*>(smem + S::kStages * S::kStageBytes);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0);
  const int lane = threadIdx.x & 31;
  const int ctas = S::kSplit ? p.parts : S::kCtas;  // of a cluster
  const Where at{S::kPair ? cluster_ctarank() : 0u, static_cast<int>(blockIdx.x) / ctas,
                 static_cast<int>(gridDim.x) / ctas, S::kSplit ? static_cast<int>(cluster_ctarank()) : 0};
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&C->full[s], 1);
      mbar_init(&C->empty[s], 1);
      mbar_init(&C->landed[s], 1);
      mbar_init(&C->cleared[s], S::kCtas);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&C->tfull[b], 1);
      mbar_init(&C->tempty[b], S::kCtas * S::kEpiWarps);
    }
    if constexpr (S::kSplit)  // from every part, one arrival for each run of a warp's lanes
      mbar_init(&C->join.full, p.parts * max(1, S::kEpiWarps / p.parts));
    // readers of a tile: producers, epilogue warps, (kDw) the last warp, and the MMA warp of the leader
    for (int s = 0; s < kFeed; ++s) {
      mbar_init(&C->fed[s], 1);
      mbar_init(&C->taken[s], 2 + S::kEpiWarps + (kMode == kDw ? 1 : 0) + (at.rank == 0 ? 1 : 0));
    }
    mbar_init(&C->mma_done, 1);
    C->abort = 0;
    if constexpr (S::kPair) C->ends.ring.peer_abort = 0;
    fence_mbar_init();
    if (p.rows > 0) {  // without rows nothing is loaded, and kDw has no maps
      tma_prefetch_desc(&maps.cols);
      for (int i = 0; i < 4; ++i)
        if (used_map<S>(i) && (kMode == kDw ? i == 3 : S::kBRows / 4 * i * S::kCtas < 1 << p.tile_bits))
          tma_prefetch_desc(&maps.rows[i]);
    }
  }
  if (warp == 1) {
    if (S::kPair)
      tmem_alloc_pair(&C->tmem_base, S::kTmemCols);
    else
      tmem_alloc(&C->tmem_base, S::kTmemCols);
  }
  if (S::kPair)
    plan_wide<kMode, S>(p, C);
  else if (warp == 2)
    plan_narrow<S>(p, C, lane);
  tc_fence_before();
  if (S::kPair || S::kSplit)
    cluster_sync();  // all barriers exist before one CTA signals another's
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = C->tmem_base;
  if (warp == 0 || warp == 2) {
    producer<kMode, kI8, S>(maps, p, smem, C, at.rank, warp >> 1);
  } else if (warp == 1) {
    if (at.rank == 0) mma_warp<kMode, kI8, S>(p, smem, C, tmem_base);
  } else if (warp == 3) {
    const int num_tiles = kMode == kDw ? p.experts * p.m_tiles * p.c_tiles : C->tile0[p.segments] * p.m_tiles;
    if (lane == 0) feed_tiles<kMode, S>(p, C, num_tiles, at);
    __syncwarp();
  } else if (kMode == kDw && warp == 4 + S::kEpiWarps) {
    clear_tails<S>(p, smem, C, lane);
  } else if constexpr (S::kSplit) {
    epilogue_split<kMode, kI8, S>(p, C, tmem_base, at, warp, lane);
  } else {
    epilogue<kMode, kI8, S>(p, C, tmem_base, at.rank, warp, lane);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (S::kPair)
    leave_pair(C->full, &C->ends.ring, C->abort, at.rank, p.timeout_ns, p.status);
  else if (S::kSplit)
    cluster_sync();  // the other parts are done with this CTA's memory
  if (warp == 1) {
    tc_fence_after();
    if (S::kPair)
      tmem_dealloc_pair(tmem_base, S::kTmemCols);
    else
      tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// ------------------------------------------------------------------ host side
// The SM count of the current device, whose context is made this thread's current one: the
// tensor maps are made by a driver call, and a thread that has made no runtime call that
// needs a context (torch's backward threads) has none.
int device_ready(int* num_sms) {
  int dev = 0;
  B2M_TRY(require_sm100(num_sms));
  B2M_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
  return check_cuda(cudaSetDevice(dev), "cudaSetDevice");
}

int encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
               const cuuint64_t* strides, const cuuint32_t* box, const char* what) {
  void* fn = nullptr;
  B2M_TRY(driver_entry("cuTensorMapEncodeTiled", &fn));
  const auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUresult r = encode(map, type, rank, const_cast<void*>(base), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B2M_ERR_ARG, "%s: cuTensorMapEncodeTiled failed (%d)", what, static_cast<int>(r));
  return B2M_OK;
}

struct Matrix {  // rows of `cols` elements, ld elements apart
  const void* ptr;
  int64_t rows, cols, ld;
};

struct Weights {  // [experts, n, k], strides in elements
  const void* ptr;
  int64_t experts, n, k, ld, expert_stride;
};

template <int kMode, bool kI8, class S>
int launch(const Maps& maps, const Params& p, int64_t tiles_bound, int num_sms, cudaStream_t s) {
  static_assert(S::kResident * (smem_bytes<S>() + 1024) <= 228 * 1024, "shared memory budget");
  static std::atomic<bool> attr_done[64];
  int dev = 0;
  B2M_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
  auto kernel = grouped_kernel<kMode, kI8, S>;
  if (dev >= 64 || !attr_done[dev].load(std::memory_order_acquire)) {
    B2M_TRY(check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            static_cast<int>(smem_bytes<S>())),
                       "grouped: cudaFuncSetAttribute"));
    if (dev < 64) attr_done[dev].store(true, std::memory_order_release);
  }
  const int ctas = S::kSplit ? p.parts : S::kCtas;
  // a cluster that shares a sum has one tile
  const int64_t most = S::kSplit ? tiles_bound : S::kResident * num_sms / ctas;
  cudaLaunchAttribute cluster[1];
  cluster[0].id = cudaLaunchAttributeClusterDimension;
  cluster[0].val.clusterDim = {static_cast<unsigned>(ctas), 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas * (tiles_bound < most ? tiles_bound : most)));
  cfg.blockDim = dim3(threads_of<S>(kMode));
  cfg.dynamicSmemBytes = smem_bytes<S>();
  cfg.stream = s;
  cfg.attrs = cluster;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, maps, p), "grouped launch");
}

constexpr int64_t kMaxDim = int64_t(1) << 30;
constexpr int64_t kMaxStride = int64_t(1) << 38;  // elements: more than any memory holds
constexpr int64_t kMaxTiles = int64_t(1) << 30;

uint32_t magic(int64_t d) { return static_cast<uint32_t>(((uint64_t(1) << 32) + d - 1) / d); }

// Output rows of a wide tile at most: 256, and half or a quarter of it while the tiles, of which
// there are tiles_of(rows) or fewer, still are no more than the pairs.  A tile of fewer rows
// reads the other operand as often and takes more than its share of the time, but pairs
// without a tile take it all: bf16, 1024 x 1024 x 1024, 12.6 us by 256, 9.2 by 64; 4096 x 256, a sum of
// 7168, 39 and 25; its weight gradient, a sum of 4096, 26 and 21.  (Tiles of 32 gave no more
// than 0.1 us.)
template <class S, class F>
int64_t rows_of_tile(int num_sms, const F& tiles_of) {
  int64_t n = S::NT;
  while (n > S::NT / 4 && tiles_of(n / 2) <= num_sms / S::kCtas) n /= 2;
  return n;
}

int32_t bits_of(int64_t n) {
  int32_t b = 0;
  while (n >> (b + 1)) ++b;
  return b;
}

// CTAs that share a tile of a sum of `blocks` blocks: as many as are resident together (33 clusters
// of eight were, of two CTAs on an SM), so that a cluster has one tile.  The exchange costs 1 us,
// which 16 blocks of a sum are worth (integers, 200 rows, 512 x 1024, eight blocks: 6.3 us
// unshared, 6.8 by fours; bf16, 16 blocks: 8.2 and 7.5), and CTAs that share an SM need more of
// them.  Integers, one row: 2048 x 7168 (16 tiles) 15.8 us unshared, 7.5 by eights; 8192 x 8192
// (64) 19.3, 16.8 by fours, 18.2 by twos; eight rows, 4096 x 4096 (32, four blocks each by
// eights) 11.0, 7.5 by fours, 8.2 by eights.  From 65 tiles on sharing costs more than it gives
// (14336 x 4096, 112 tiles: 14.7 unshared, 16.0 by twos).
int parts_of(int64_t tiles, int64_t blocks, int on_sm) {
  int parts = 1;
  while (parts < kMostParts && tiles <= kSplitTiles && blocks >= kLeastSplit &&
         tiles * parts * 2 <= 2 * on_sm * kSplitTiles &&
         blocks >= (tiles * parts * 2 <= 2 * kSplitTiles ? 2 : 8) * parts * 2)
    parts *= 2;
  return parts;
}

// Limit of a wait inside a CTA's pipeline, where nothing but the CTA's own work is waited for: a
// sum of `blocks` blocks takes a third of a microsecond for each, and a role may wait for
// several tiles.
uint64_t wait_limit(int64_t blocks) { return 2 * timeout_ns() + 8000ull * static_cast<uint64_t>(blocks); }

int check_matrix(const char* what, const char* name, const Matrix& m, int elem) {
  if (m.rows < 0 || m.rows > kMaxDim || m.cols < 1 || m.cols > kMaxDim)
    return fail(B2M_ERR_ARG, "%s: %s is [%lld, %lld]; each extent is at most 2^30 and it has columns", what, name,
                (long long)m.rows, (long long)m.cols);
  if (m.ld < m.cols || m.ld > kMaxStride || m.ld * elem % 16)
    return fail(B2M_ERR_ARG, "%s: rows of %s must be at least %lld elements and a multiple of 16 bytes apart (%lld)",
                what, name, (long long)m.cols, (long long)m.ld);
  if (m.rows > 0 && (!m.ptr || !aligned16(m.ptr)))
    return fail(B2M_ERR_ARG, "%s: %s must not be null and must be 16-byte aligned", what, name);
  return B2M_OK;
}

int check_weights(const char* what, const Weights& w, int elem) {
  if (w.experts < 1 || w.experts > kMaxExperts)
    return fail(B2M_ERR_ARG, "%s: need 1 <= experts <= %d (%lld)", what, kMaxExperts, (long long)w.experts);
  B2M_TRY(check_matrix(what, "w", Matrix{w.ptr, w.n, w.k, w.ld}, elem));
  if (w.n < 1) return fail(B2M_ERR_ARG, "%s: w has no rows", what);
  if (w.expert_stride < 1 || w.expert_stride > kMaxStride || w.expert_stride * elem % 16)
    return fail(B2M_ERR_ARG, "%s: experts of w must be a multiple of 16 bytes apart (%lld elements)", what,
                (long long)w.expert_stride);
  return B2M_OK;
}

int check_out(const char* what, const void* out, int64_t cols, int64_t ldo, int32_t out_type, int32_t in_type) {
  if (!out) return fail(B2M_ERR_ARG, "%s: null output", what);
  if (ldo < cols) return fail(B2M_ERR_ARG, "%s: output rows are %lld elements apart, need %lld", what, (long long)ldo,
                              (long long)cols);
  if (ldo > kMaxStride) return fail(B2M_ERR_ARG, "%s: output rows are more than 2^38 elements apart", what);
  if (out_type != B2M_FP32 && out_type != in_type)
    return fail(B2M_ERR_ARG, "%s: output type %d must be the input type or fp32", what, out_type);
  if (reinterpret_cast<uintptr_t>(out) % (out_type == B2M_FP32 ? 4 : 2))
    return fail(B2M_ERR_ARG, "%s: misaligned output", what);
  return B2M_OK;
}

// What the kernels read or write as 32-bit words; any of them may be null here.
int check_words(const char* what, const int32_t* ends, const int32_t* status, const float* a_scale = nullptr,
                const float* w_scale = nullptr) {
  if (!aligned4(ends) || !aligned4(status) || !aligned4(a_scale) || !aligned4(w_scale))
    return fail(B2M_ERR_ARG, "%s: ends, scales and status must be 4-byte aligned", what);
  return B2M_OK;
}

// kFwd and kDx: `rows` (x, dy or integer codes) times each segment's weights.
template <int kMode, bool kI8>
int rows_times_weights(const char* what, const Matrix& x, const Weights& w, const int32_t* ends, int32_t in_type,
                       void* out, int64_t ldo, int32_t out_type, int32_t clear_rest, const float* a_scale,
                       const float* w_scale, int32_t* status, void* stream) {
  const int elem = kI8 ? 1 : 2;
  const CUtensorMapDataType type = kI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                       : (in_type == B2M_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                              : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
  const cuuint32_t in_row = kRowBytes / elem;  // elements in a shared-memory row
  const int64_t m_dim = kMode == kFwd ? w.n : w.k;
  const int64_t sum = kMode == kFwd ? w.k : w.n;
  Params p{};
  p.ends = ends;
  p.experts = static_cast<int32_t>(w.experts);
  p.segments = p.experts + (clear_rest && ends ? 1 : 0);
  p.rows = x.rows;
  p.m_dim = static_cast<int32_t>(m_dim);
  p.k_blocks = static_cast<int32_t>((sum + in_row - 1) / in_row);
  p.out = out;
  p.ldo = ldo;
  p.out_type = out_type;
  p.wide_out = aligned16(out) && ldo % 8 == 0;
  p.a_scale = a_scale;
  p.w_scale = w_scale;
  p.status = status;
  p.timeout_ns = wait_limit(p.k_blocks);

  // Most row tiles of n that x.rows rows in so many segments can take: one not full for each that has rows.
  const auto row_tiles = [&](int64_t n, int64_t segments) {
    return (x.rows + (n - 1) * (x.rows < segments ? x.rows : segments)) / n;
  };
  const auto m_tiles = [&](int64_t m) { return (m_dim + m - 1) / m; };
  // Row tiles of 32, one CTA each, while segments are short: weights alone bound these calls,
  // and four times as many CTAs share them out (E=32, 4096 x 7168, forward: 280 us narrow, 288
  // wide at 8 rows each).  The mean is all that the host knows of the lengths.  Under Zipf 1.2 the
  // longest segments cost a narrow launch more than it saves from 16 rows on average (299
  // narrow, 292 wide; 377 and 311 at 32), and not yet at 12 (278, 292).  Nor does one segment that has a
  // quarter of 12 rows an expert (E=256, 1536 x 2048: 243 narrow, 250 wide; E=1024, 768 x 2048: 496, 491);
  // half of them on one cost 249 and 250 (508, 491), all of them 41 and 31 (85, 34).  One segment alone
  // has the length that the host sees: up to one narrow tile.
  //
  // Few tiles for the SMs: clusters of two to eight CTAs share each one along its sum.  So a
  // launch is narrow whenever that makes no more than 64 tiles (bf16, one segment of 96 rows, 2048 x
  // 7168: 26.8 us wide, 16.7 narrow), and takes tiles of 64 rows when those are so few and their
  // sums long: 256 rows 26.8 wide, 21.2; 64 rows, 4096 x 4096, 18.8 and 15.7; integers, 64 rows, 7168 x
  // 2048 (16 blocks), 9.9 and 11.3.
  const int64_t narrow_tiles = row_tiles(Split::NT, w.experts) * m_tiles(Split::kTileM);
  const int64_t middle_tiles = row_tiles(Split64::NT, w.experts) * m_tiles(Split64::kTileM);
  const bool narrow = x.rows <= (w.experts == 1 ? Narrow::NT : 12 * w.experts) || narrow_tiles <= kSplitTiles;
  const bool middle = !narrow && middle_tiles <= kSplitTiles && p.k_blocks >= 2 * kLeastSplit;
  const int64_t most = narrow   ? row_tiles(Narrow::NT, p.segments) * m_tiles(Narrow::kTileM)
                       : middle ? row_tiles(Split64::NT, p.segments) * m_tiles(Split64::kTileM)
                                : row_tiles(Wide::NT, p.segments) * m_tiles(Wide::kTileM);
  if (most > kMaxTiles) return fail(B2M_ERR_ARG, "%s: more than 2^30 tiles", what);
  int num_sms = 0;
  B2M_TRY(device_ready(&num_sms));
  if (x.rows == 0) return B2M_OK;

  // `shape` is the launch's, `n` the rows of its tiles.
  const auto run = [&](auto shape, int64_t n, int parts) -> int {
    using S = decltype(shape);
    p.parts = parts;
    p.tile_bits = bits_of(n);
    p.m_tiles = static_cast<int32_t>(m_tiles(S::kTileM));
    p.m_magic = magic(p.m_tiles);
    p.band_magic = magic(int64_t(kBand) * p.m_tiles);
    p.idesc = (kI8 ? (2u << 4) | (1u << 7) | (1u << 10)                                  // S32, both signed
                   : (1u << 4) | (in_type == B2M_BF16 ? (1u << 7) | (1u << 10) : 0u)) |  // F32
              (kMode == kDx ? 1u << 15 : 0u) | (static_cast<uint32_t>(S::kTileM >> 4) << 24);
    const cuuint64_t w_dims[3] = {static_cast<cuuint64_t>(w.k), static_cast<cuuint64_t>(w.n),
                                  static_cast<cuuint64_t>(w.experts)};
    const cuuint64_t w_strides[2] = {static_cast<cuuint64_t>(w.ld * elem),
                                     static_cast<cuuint64_t>(w.expert_stride * elem)};
    const cuuint32_t w_box[3] = {in_row, kMode == kFwd ? static_cast<cuuint32_t>(kM) : 64u, 1};
    const cuuint64_t x_dims[2] = {static_cast<cuuint64_t>(x.cols), static_cast<cuuint64_t>(x.rows)};
    const cuuint64_t x_strides[1] = {static_cast<cuuint64_t>(x.ld * elem)};
    Maps maps{};
    B2M_TRY(encode_map(&maps.cols, type, 3, w.ptr, w_dims, w_strides, w_box, what));
    for (int i = 0; i < 4 && S::kBRows / 4 * i < n / S::kCtas; ++i) {  // a tile of n rows takes no larger box
      if (!used_map<S>(i)) continue;
      const cuuint32_t box[2] = {in_row, static_cast<cuuint32_t>(S::kBRows / 4 * (i + 1))};
      B2M_TRY(encode_map(&maps.rows[i], type, 2, x.ptr, x_dims, x_strides, box, what));
    }
    return launch<kMode, kI8, S>(maps, p, row_tiles(n, p.segments) * p.m_tiles, num_sms,
                                 static_cast<cudaStream_t>(stream));
  };
  if (middle) return run(Split64{}, Split64::NT, parts_of(middle_tiles, p.k_blocks, Split64::kResident));
  if (narrow) {
    const int parts = parts_of(narrow_tiles, p.k_blocks, Split::kResident);
    if (parts > 1) return run(Split{}, Split::NT, parts);
    // E=128, eight rows, 1536 x 2048 (96 tiles): 14.2 us single, 15.7 two on an SM; integers,
    // 28672 x 4096 (224): 24.9 and 23.3; E=8, two rows, 28672 x 4096 (448): 84 and 77.5.
    if (most <= num_sms) return run(Single{}, Single::NT, 1);
    return run(Narrow{}, Narrow::NT, 1);
  }
  const auto tiles = [&](int64_t n) { return row_tiles(n, p.segments) * m_tiles(Wide::kTileM); };
  return run(Wide{}, rows_of_tile<Wide>(num_sms, tiles), 1);
}

int check_16bit(const char* what, int32_t in_type) {
  if (in_type != B2M_BF16 && in_type != B2M_FP16)
    return fail(B2M_ERR_ARG, "%s: input type %d is neither bf16 nor fp16", what, in_type);
  return B2M_OK;
}

}  // namespace
}  // namespace b2m

extern "C" int b2m_grouped_mm(const void* x, int64_t rows, int64_t ldx, const void* w, int32_t experts, int64_t n,
                              int64_t k, int64_t ldw, int64_t w_stride, const int32_t* ends, int32_t in_type, void* out,
                              int64_t ldo, int32_t out_type, int32_t clear_rest, int32_t* dev_status, void* stream) {
  using namespace b2m;
  const Matrix mx{x, rows, k, ldx};
  const Weights mw{w, experts, n, k, ldw, w_stride};
  B2M_TRY(check_16bit("grouped_mm", in_type));
  B2M_TRY(check_weights("grouped_mm", mw, 2));
  B2M_TRY(check_matrix("grouped_mm", "x", mx, 2));
  if (!ends) return fail(B2M_ERR_ARG, "grouped_mm: null ends");
  B2M_TRY(check_words("grouped_mm", ends, dev_status));
  if (rows > 0) B2M_TRY(check_out("grouped_mm", out, n, ldo, out_type, in_type));
  return rows_times_weights<kFwd, false>("grouped_mm", mx, mw, ends, in_type, out, ldo, out_type, clear_rest, nullptr,
                                         nullptr, dev_status, stream);
}

extern "C" int b2m_grouped_mm_dx(const void* dy, int64_t rows, int64_t lddy, const void* w, int32_t experts, int64_t n,
                                 int64_t k, int64_t ldw, int64_t w_stride, const int32_t* ends, int32_t in_type,
                                 void* out, int64_t ldo, int32_t out_type, int32_t clear_rest, int32_t* dev_status, void* stream) {
  using namespace b2m;
  const Matrix mdy{dy, rows, n, lddy};
  const Weights mw{w, experts, n, k, ldw, w_stride};
  B2M_TRY(check_16bit("grouped_mm_dx", in_type));
  B2M_TRY(check_weights("grouped_mm_dx", mw, 2));
  B2M_TRY(check_matrix("grouped_mm_dx", "dy", mdy, 2));
  if (!ends) return fail(B2M_ERR_ARG, "grouped_mm_dx: null ends");
  B2M_TRY(check_words("grouped_mm_dx", ends, dev_status));
  if (rows > 0) B2M_TRY(check_out("grouped_mm_dx", out, k, ldo, out_type, in_type));
  return rows_times_weights<kDx, false>("grouped_mm_dx", mdy, mw, ends, in_type, out, ldo, out_type, clear_rest,
                                        nullptr, nullptr, dev_status, stream);
}

extern "C" int b2m_grouped_mm_dw(const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t rows, int64_t n,
                                 int64_t k, const int32_t* ends, int32_t experts, int32_t in_type, void* out,
                                 int64_t ldo, int64_t out_stride, int32_t out_type, int32_t* dev_status, void* stream) {
  using namespace b2m;
  const char* what = "grouped_mm_dw";
  const Matrix mdy{dy, rows, n, lddy}, mx{x, rows, k, ldx};
  B2M_TRY(check_16bit(what, in_type));
  B2M_TRY(check_matrix(what, "dy", mdy, 2));
  B2M_TRY(check_matrix(what, "x", mx, 2));
  if (experts < 1 || experts > kMaxExperts)
    return fail(B2M_ERR_ARG, "%s: need 1 <= experts <= %d (%d)", what, kMaxExperts, experts);
  if (!ends) return fail(B2M_ERR_ARG, "%s: null ends", what);
  B2M_TRY(check_words(what, ends, dev_status));
  B2M_TRY(check_out(what, out, k, ldo, out_type, in_type));
  // One expert behind the other, or row by row between the others'.  (Up to 2^30 rows, up to 2^38 elements apart: the
  // products need 128 bits.)
  const bool apart = out_stride >= static_cast<__int128>(n - 1) * ldo + k;
  const bool between = out_stride >= k && ldo >= static_cast<__int128>(experts - 1) * out_stride + k;
  if (out_stride > kMaxStride || (!apart && !between))
    return fail(B2M_ERR_ARG, "%s: experts of the output overlap, or are more than 2^38 elements apart", what);
  Params p{};
  p.ends = ends;
  p.experts = experts;
  p.segments = experts;
  p.rows = rows;
  p.m_dim = static_cast<int32_t>(k);
  p.c_dim = static_cast<int32_t>(n);
  p.out = out;
  p.ldo = ldo;
  p.out_expert = out_stride;
  p.out_type = out_type;
  p.wide_out = aligned16(out) && ldo % 8 == 0 && out_stride % 8 == 0;
  p.status = dev_status;
  p.timeout_ns = wait_limit(rows / 64);
  const auto tiles_of = [&](int64_t c, int64_t m) { return (n + c - 1) / c * ((k + m - 1) / m) * experts; };
  if (tiles_of(Wide::NT, Wide::kTileM) > kMaxTiles) return fail(B2M_ERR_ARG, "%s: more than 2^30 tiles", what);
  int num_sms = 0;
  B2M_TRY(device_ready(&num_sms));
  const CUtensorMapDataType type =
      in_type == B2M_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  // Without rows every segment is empty: nothing is loaded, and a map of no rows cannot be made.
  const cuuint64_t x_dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t dy_dims[2] = {static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(rows)};
  const cuuint64_t x_strides[1] = {static_cast<cuuint64_t>(ldx * 2)};
  const cuuint64_t dy_strides[1] = {static_cast<cuuint64_t>(lddy * 2)};
  const cuuint32_t box[2] = {64, 64};
  Maps maps{};
  if (rows > 0) {
    B2M_TRY(encode_map(&maps.cols, type, 2, x, x_dims, x_strides, box, what));
    B2M_TRY(encode_map(&maps.rows[3], type, 2, dy, dy_dims, dy_strides, box, what));
  }
  const auto run = [&](auto shape, int64_t c, int parts) -> int {
    using S = decltype(shape);
    p.parts = parts;
    p.tile_bits = bits_of(c);
    p.m_tiles = static_cast<int32_t>((k + S::kTileM - 1) / S::kTileM);
    p.c_tiles = static_cast<int32_t>((n + c - 1) / c);
    p.band_magic = magic(int64_t(kBand) * p.m_tiles);
    p.expert_magic = magic(int64_t(p.m_tiles) * p.c_tiles);
    p.idesc = (1u << 4) | (in_type == B2M_BF16 ? (1u << 7) | (1u << 10) : 0u) | (1u << 15) | (1u << 16) |
              (static_cast<uint32_t>(S::kTileM >> 4) << 24);
    return launch<kDw, false, S>(maps, p, tiles_of(c, S::kTileM), num_sms, static_cast<cudaStream_t>(stream));
  };
  // Long sums of few tiles are shared like those of the other directions, by the segments' mean
  // length.  bf16, 272 x 128 (five tiles): 8192 rows 32 us wide, 11 by eights; 1024 rows 9.6, 7.4;
  // 512 x 1024 (64 tiles): 32.5, 25.6 by twos; 2048 rows 13.1, 12.9; 1024 rows 9.6, 10.6.
  const int64_t mean = rows / 64 / experts;  // blocks
  const int parts = parts_of(tiles_of(Split64::NT, Split64::kTileM), mean, Split64::kResident);
  if (parts > 2 || (parts == 2 && mean >= 2 * kLeastSplit)) return run(Split64{}, Split64::NT, parts);
  const auto tiles = [&](int64_t c) { return tiles_of(c, Wide::kTileM); };
  // Gradients of up to 128 columns: 64 experts of 4096 x 64, 100 rows each, 43 us by pairs, 24; 32 of 4096 x
  // 128, 1024 rows, 59 and 53.  (The other directions at such widths: 32768 rows, k = 4096, 57 by
  // pairs, 52; but eight segments of 512 rows 17.7 and 19.4, sixteen of 230, k = 12352, 46 and 59.)
  if (k <= Slim::kTileM) return run(Slim{}, rows_of_tile<Slim>(num_sms, tiles), 1);
  return run(Wide{}, rows_of_tile<Wide>(num_sms, tiles), 1);
}

extern "C" int b2m_int8_mm(const void* a, const float* a_scale, int64_t rows, int64_t lda, const void* w,
                           const float* w_scale, int32_t experts, int64_t n, int64_t k, int64_t ldw, int64_t w_stride,
                           const int32_t* ends, void* out, int64_t ldo, int32_t out_type, int32_t clear_rest,
                           int32_t* dev_status, void* stream) {
  using namespace b2m;
  const Matrix ma{a, rows, k, lda};
  const Weights mw{w, experts, n, k, ldw, w_stride};
  B2M_TRY(check_weights("int8_mm", mw, 1));
  B2M_TRY(check_matrix("int8_mm", "a", ma, 1));
  if (k > 131071) return fail(B2M_ERR_ARG, "int8_mm: k=%lld; sums of more than 131071 products can pass 32 bits", (long long)k);
  if (!w_scale || (rows > 0 && !a_scale)) return fail(B2M_ERR_ARG, "int8_mm: null scales");
  B2M_TRY(check_words("int8_mm", ends, dev_status, a_scale, w_scale));
  if (!ends && experts != 1) return fail(B2M_ERR_ARG, "int8_mm: ends may be null for one expert only");
  if (out_type != B2M_BF16 && out_type != B2M_FP16 && out_type != B2M_FP32)
    return fail(B2M_ERR_ARG, "int8_mm: unknown output type %d", out_type);
  if (rows > 0) B2M_TRY(check_out("int8_mm", out, n, ldo, out_type, out_type));
  return rows_times_weights<kFwd, true>("int8_mm", ma, mw, ends, B2M_BF16, out, ldo, out_type, clear_rest, a_scale,
                                        w_scale, dev_status, stream);
}
