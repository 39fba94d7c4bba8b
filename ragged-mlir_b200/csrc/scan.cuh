// Gated linear recurrence over ragged segments, forward and backward.
//
//   forward   h[t] = a[t] h[t-1] + x[t]            (h before a segment: its
//             initial state; without one, h = x on the first row)
//   backward  g[t] = dh[t] + u[t+1],  u[t] = a[t] g[t]   (u past a segment's
//             last row: the gradient of its final state)
//             dx[t] = g[t],  da[t] = g[t] h[t-1],  dinitial = u[first row]
//
// Both are first-order recurrences, one forward and one backward in t, whose
// steps compose: rows r..s act on the state before them as H + A * state with
// A the product of the gates.  Work is cut into slabs of rows by tiles of
// columns, and every task belongs to one warp: 8 or 4 bytes of a row a lane
// (narrow rows: several row groups side by side), down the rows in batches of
// 8.  No block barrier, no exchange between lanes; warps hide each other's
// latency.
//
//   fold   (A, H) of each slab.  Only the rows past its last segment start
//          count, and none where its last row ends a segment.
//   join   column by column over the slabs: the state before each of them.
//   walk   the recurrence over a slab's rows from the state before them.
//
// Three launches in stream order: nothing waits on anything inside a kernel,
// the order of all sums is fixed, and equal inputs give equal bits.  Device
// memory is the bound: walk reads every input once and writes every output
// once; fold reads again what of the inputs belongs to segments that cross
// slabs, and walk goes through the slabs from the last one back (forward ones
// in a backward pass), so that it meets first what fold left in L2.  The
// arithmetic is one FMA an element, about 10 instructions an element in all.
// bf16 65536 x 1024 in 16 segments: 132 us forward, 176 backward, 5.1 TB/s of 5
// and 7 passes over a tensor where 3 and 5 are the least; f32 262144 x 100 in 1024
// segments 98 us and 142.  What is left is the second reading, the join and each
// launch's first loads; rows read once in a single launch, with waits for the slab
// before, took 173 to 231 us where this form took 140.  Two halves of a batch in
// turn, one on its way, spill: 172.  (Times of this form: a graph of calls, inputs
// larger than L2.  Times of the others, here and beside the rules in scan.cu, are of
// single launches between events, which come in steps of 2 us.)
//
// For few rows walk is the only launch: a lane whose rows go on from earlier ones
// runs the recurrence over those itself.  Bound there: latency.  200 rows of 200
// segments, bf16 x 1024, are 104 warps in 13 CTAs, each a chain of dependent reads
// (the search in the offsets, rows, initial states, segments without rows): 8 us in
// a graph of calls, 11 with cold inputs.
//
// The backward pass needs the states again.  It recomputes 8 rows at a time from
// values and gates, from the state before them that forward records in f32 (4
// bytes for 8 elements; reading `out` would cost as much as reading values
// does): no rounded state enters a gradient.  16 rows at a time halve those
// bytes, but their states leave registers for 4 bytes a lane and not 8: 219
// instead of 184 us backward, 137 instead of 139 forward (bf16 65536 x 1024).
//
// States, products and sums are f32; results are rounded to the tensor's type
// once, when they are written.  Segment starts cut the fold by a flag, never
// by a multiplication with zero, so nothing crosses from one segment to
// another.  Where a state is zero its product with A counts as zero, also if A
// has overflowed.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "common.cuh"

namespace rgb {

constexpr int kScanThreads = 256;
constexpr int kScanWarps = kScanThreads / 32;
constexpr int kScanBatch = 8;     // rows of a lane in flight; rows per recorded state
constexpr int kJoinCols = 4;      // columns of a join's block
constexpr int kJoinParts = 128;   // parts that it cuts the slabs into, a thread each
constexpr int kJoinBatch = 8;     // pairs of a thread in flight

struct ScanArgs {
  const void *values, *gates, *offsets;
  const float *initial;  // [B, D] or null
  int64_t n, d;
  int64_t b;
  int shift;           // log2 of the lanes across a tile's columns
  int lane_rows;       // rows of a lane: 16, 32 or 64
  int row_shift;       // log2 of a slab's rows: lane_rows * (32 >> shift)
  int tiles;           // column tiles
  int64_t slabs;       // slabs that hold rows
  int64_t blocks;      // slabs launched (more than `slabs` where many segments are empty)
  int64_t per_block;   // segments whose emptiness a slab looks at
  bool clear_rest;     // rows of the results behind the last segment: set to zero, else left alone
  float *carries;      // [N / 8, D] state before every 8th row (written by forward, read by backward)
  // forward
  void *out;
  float *final_state;  // [B, D] or null
  // backward
  const void *grad_out;
  const float *grad_final;  // [B, D] or null
  void *grad_values, *grad_gates;
  float *grad_initial;  // [B, D] or null
  // workspace (null where walk is the only launch)
  float2 *pairs;    // (A, H) of each slab: [slabs][D]; A is NaN-boxed where the pair starts at a segment
  float *states;    // state before each slab: [slabs][D]
};

__device__ __forceinline__ float scan_apply(float a, float h, float state) {
  return state == 0.0f ? h : fmaf(a, state, h);
}

// In place of A: the pair starts at a segment, and no state before it counts.
// (A NaN that arithmetic does not make; other NaNs become the usual one.)
constexpr unsigned kScanReset = 0x7fc05e70u;

template <int VEC>
struct ScanPair {
  float a[VEC], h[VEC];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      a[v] = 1.0f;
      h[v] = 0.0f;
    }
  }
  // This pair after `first`.
  __device__ __forceinline__ void after(const ScanPair &first) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      h[v] = scan_apply(a[v], h[v], first.h[v]);
      a[v] *= first.a[v];
    }
  }
  __device__ __forceinline__ void store(float2 *at, bool reset) const {
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      at[v] = make_float2(__uint_as_float(reset ? kScanReset : a[v] != a[v] ? 0x7fffffffu : __float_as_uint(a[v])), h[v]);
  }
};

// Composition over a warp's row groups (lanes of one group hold one group's
// columns), in lane order or, REV, from the last group down.  On return `own`
// describes the groups before the lane's own, `total` all of them.
template <int VEC, bool REV>
__device__ __forceinline__ void scan_groups(ScanPair<VEC> &own, int &own_reset, ScanPair<VEC> &total, int &total_reset,
                                            int shift) {
  total = own;
  total_reset = own_reset;
  if (shift == 5) {  // one group
    own.clear();
    own_reset = 0;
    return;
  }
  const int lane = threadIdx.x & 31;
  const int lanes = 1 << shift;
  auto from = [&](float x, int off) { return REV ? __shfl_down_sync(~0u, x, off) : __shfl_up_sync(~0u, x, off); };
  for (int off = lanes; off < 32; off <<= 1) {
    const bool live = REV ? lane + off < 32 : lane >= off;
    const int r = REV ? __shfl_down_sync(~0u, total_reset, off) : __shfl_up_sync(~0u, total_reset, off);
    ScanPair<VEC> first;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      first.a[v] = from(total.a[v], off);
      first.h[v] = from(total.h[v], off);
    }
    if (live && !total_reset) {
      total.after(first);
      total_reset = r;
    }
  }
  const bool edge = REV ? lane >= 32 - lanes : lane < lanes;
  own_reset = REV ? __shfl_down_sync(~0u, total_reset, lanes) : __shfl_up_sync(~0u, total_reset, lanes);
  if (edge) own_reset = 0;
  const int last = (REV ? 0 : 32 - lanes) + (lane & (lanes - 1));
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const float a = from(total.a[v], lanes), h = from(total.h[v], lanes);
    own.a[v] = edge ? 1.0f : a;
    own.h[v] = edge ? 0.0f : h;
    total.a[v] = __shfl_sync(~0u, total.a[v], last);
    total.h[v] = __shfl_sync(~0u, total.h[v], last);
  }
  total_reset = __shfl_sync(~0u, total_reset, last);
}

// Segment of row `row` (the last one that starts at or before it), by a warp:
// a 32-way search.
template <typename OffT>
__device__ __forceinline__ int64_t scan_find(const OffT *__restrict__ offsets, int64_t b, int64_t row) {
  const int lane = threadIdx.x & 31;
  int64_t lo = 0, hi = b;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 31) >> 5;
    const int64_t at = lo + lane * step;
    const unsigned below = __ballot_sync(~0u, lane == 0 || (at < hi && static_cast<int64_t>(offsets[at]) <= row));
    const int count = __popc(below);
    const int64_t next = lo + count * step;
    lo += (count - 1) * step;
    if (next < hi) hi = next;
  }
  return lo;
}

// Where segments with rows start and end among a slab's rows: a bit per first
// row in start_mask and per last row in end_mask, and the segment in start_seg
// and end_seg (a warp's own shared memory).  Offsets that are out of order set
// nothing outside the arrays.
struct ScanMarks {
  unsigned *start_mask, *end_mask;  // max(rows, 64) / 32 words each
  int *start_seg, *end_seg;         // rows each
};

// Returns the segment of row `row0`.
template <typename OffT>
__device__ __forceinline__ int64_t scan_mark(const OffT *__restrict__ offsets, int64_t b, int64_t row0, int rows,
                                             const ScanMarks &m) {
  const int lane = threadIdx.x & 31;
  const int words = (rows < 64 ? 64 : rows) / 32;
  for (int i = lane; i < 2 * words; i += 32) m.start_mask[i] = 0;
  __syncwarp();
  int64_t first = -1, next = 0, row = row0;
  bool search = true;
  for (;;) {
    if (search) next = max(next, scan_find(offsets, b, row));
    if (first < 0) first = next;
    const int64_t s = next + lane;
    const bool there = s < b;
    const int64_t begin = there ? static_cast<int64_t>(offsets[s]) - row0 : rows;
    const int64_t end = there ? static_cast<int64_t>(offsets[s + 1]) - 1 - row0 : rows;
    if (begin < rows && begin <= end) {
      if (begin >= 0) {
        m.start_seg[begin] = static_cast<int>(s);
        atomicOr(&m.start_mask[begin >> 5], 1u << (begin & 31));
      }
      if (end >= 0 && end < rows) {
        m.end_seg[end] = static_cast<int>(s);
        atomicOr(&m.end_mask[end >> 5], 1u << (end & 31));
      }
    }
    if (__any_sync(~0u, begin >= rows)) break;
    next += 32;
    search = !__any_sync(~0u, begin <= end);  // 32 segments without rows: on to the last one that starts there
    row = row0 + __shfl_sync(~0u, begin, 31);
  }
  __syncwarp();
  return first;
}

// Words of shared memory of a warp's marks.
__host__ __device__ constexpr int scan_marks_words(int rows) { return 2 * ((rows < 64 ? 64 : rows) / 32) + 2 * rows; }

// A batch of rows of a lane, `d` elements apart; of `count` rows (at least
// one), the last stands in for those that are missing.
template <typename T, int VEC>
__device__ __forceinline__ void scan_rows(const T *__restrict__ at, int64_t d, int count,
                                          typename VecIO<T, VEC>::Raw (&raw)[kScanBatch]) {
#pragma unroll
  for (int i = 0; i < kScanBatch; ++i) {
    raw[i] = VecIO<T, VEC>::load_raw(at);
    at += i + 1 < count ? d : 0;
  }
}

// What fold and walk share: a warp's place, and its slab's marks.
template <typename T, typename OffT, int VEC, bool BACKWARD>
struct ScanWarp {
  using IO = VecIO<T, VEC>;
  using Raw = typename IO::Raw;
  using State = VecIO<float, VEC>;
  using Pair = ScanPair<VEC>;
  static constexpr int BATCH = kScanBatch;
  const ScanArgs &p;
  const OffT *__restrict__ offsets;
  int lanes, rows, words, base;  // base: this lane's first row of a slab
  int limit;                     // rows of the slab before the last segment's end; those behind it are left alone
  int64_t pos, row0, col, seg0;  // slab in the order of the recurrence, its first row, this lane's column
  bool col_ok;
  ScanMarks m;

  __device__ __forceinline__ ScanWarp(const ScanArgs &args, unsigned *smem) : p(args) {
    offsets = static_cast<const OffT *>(p.offsets);
    const int lane = threadIdx.x & 31;
    lanes = 1 << p.shift;
    rows = 1 << p.row_shift;
    words = (rows < 64 ? 64 : rows) / 32;
    base = (lane >> p.shift) * p.lane_rows;
    m.start_mask = smem + (threadIdx.x >> 5) * scan_marks_words(rows);
    m.end_mask = m.start_mask + words;
    m.start_seg = reinterpret_cast<int *>(m.end_mask + words);
    m.end_seg = m.start_seg + rows;
  }
  __device__ __forceinline__ void go(int64_t slab, int tile) {
    pos = slab;
    row0 = (BACKWARD ? p.slabs - 1 - pos : pos) << p.row_shift;
    limit = static_cast<int>(min(max(min(static_cast<int64_t>(offsets[p.b]), p.n) - row0, int64_t{0}), int64_t{rows}));
    col = (static_cast<int64_t>(tile) * lanes + (threadIdx.x & (lanes - 1))) * VEC;
    col_ok = col < p.d;
  }
  __device__ __forceinline__ void mark() {
    __syncwarp();
    seg0 = scan_mark(offsets, p.b, row0, rows, m);
  }
  __device__ __forceinline__ uint64_t lane_bits(const unsigned *mask) const {  // of this lane's rows
    if (p.lane_rows == 64) return mask[base >> 5] | (static_cast<uint64_t>(mask[(base >> 5) + 1]) << 32);
    const unsigned word = mask[base >> 5];
    return p.lane_rows == 32 ? word : (word >> (base & 31)) & 0xffffu;
  }
  __device__ __forceinline__ bool starts_at_first() const { return m.start_mask[0] & 1; }
  __device__ __forceinline__ bool ends_at_last() const {
    const int last = limit - 1;
    return last >= 0 && (m.end_mask[last >> 5] >> (last & 31)) & 1;
  }
  __device__ __forceinline__ int row_count(int batch) const {  // rows of this lane's batch
    return min(max(limit - base - batch * BATCH, 0), BATCH);
  }
  __device__ __forceinline__ void state_of(const float *states, int64_t seg, float (&x)[VEC]) const {
    if (states) {
      State::load(states + seg * p.d + col, x);
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[v] = 0.0f;
    }
  }

  // Folds this lane's rows from the last segment start on (first end,
  // BACKWARD).  Returns whether there is one.
  __device__ __forceinline__ bool fold(Pair &f) const {
    f.clear();
    const uint64_t marks = lane_bits(BACKWARD ? m.end_mask : m.start_mask);
    if (!col_ok) return marks != 0;
    const T *__restrict__ gates = static_cast<const T *>(p.gates);
    const T *__restrict__ second = static_cast<const T *>(BACKWARD ? p.grad_out : p.values);
    const int batches = p.lane_rows / BATCH;
    const int enter = !marks ? (BACKWARD ? batches - 1 : 0)
                             : (BACKWARD ? __ffsll(marks) - 1 : 63 - __clzll(marks)) / BATCH;
#pragma unroll 1
    for (int batch = enter; BACKWARD ? batch >= 0 : batch < batches; batch += BACKWARD ? -1 : 1) {
      const int64_t row = row0 + base + batch * BATCH;
      const int count = row_count(batch);
      if (count <= 0) continue;
      Raw ra[BATCH], rx[BATCH];
      scan_rows<T, VEC>(gates + row * p.d + col, p.d, count, ra);
      scan_rows<T, VEC>(second + row * p.d + col, p.d, count, rx);
      const unsigned mark = static_cast<unsigned>(marks >> (batch * BATCH)) & ((1u << BATCH) - 1);
      const int *seg = (BACKWARD ? m.end_seg : m.start_seg) + base + batch * BATCH;
      const bool plain = mark == 0 && count == BATCH;
      auto step = [&](int i, bool alone) {
        float a[VEC], x[VEC];
        IO::unpack(ra[i], a);
        IO::unpack(rx[i], x);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          if constexpr (BACKWARD)
            f.h[v] = a[v] * (x[v] + f.h[v]);
          else
            f.h[v] = alone ? x[v] : fmaf(a[v], f.h[v], x[v]);
          f.a[v] *= a[v];
        }
      };
      if (plain) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) step(BACKWARD ? BATCH - 1 - j : j, false);
      } else {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const int i = BACKWARD ? BATCH - 1 - j : j;
          if (i < count) {
            const bool enters = (mark >> i) & 1;
            if (enters) state_of(BACKWARD ? p.grad_final : p.initial, seg[i], f.h);
            step(i, enters && !p.initial);
          }
        }
      }
    }
    return marks != 0;
  }

  // Without a workspace: the state before this lane's rows, by running the
  // recurrence over the rows of their segment before (after, BACKWARD) them.
  __device__ __forceinline__ void catch_up(float (&h)[VEC]) const {
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = 0.0f;
    const int64_t mine = row0 + base;
    if (base >= limit || !col_ok) return;
    const T *__restrict__ gates = static_cast<const T *>(p.gates);
    const T *__restrict__ second = static_cast<const T *>(BACKWARD ? p.grad_out : p.values);
    int64_t seg = seg0;  // the segment of this lane's first (last, BACKWARD) row
    const int64_t here = BACKWARD ? row0 + min(base + p.lane_rows, limit) - 1 : mine;
    const int at = static_cast<int>(here - row0);
    for (int i = at >> 5; i >= 0; --i) {
      const unsigned bits = m.start_mask[i] & (i == at >> 5 ? (2u << (at & 31)) - 1 : ~0u);
      if (bits) {
        seg = m.start_seg[i * 32 + 31 - __clz(bits)];
        break;
      }
    }
    const int64_t begin = max(static_cast<int64_t>(offsets[seg]), int64_t{0});
    const int64_t end = min(static_cast<int64_t>(offsets[seg + 1]), p.n);
    if (BACKWARD ? end - 1 <= here : begin >= mine) return;
    state_of(BACKWARD ? p.grad_final : p.initial, seg, h);
    const int64_t count = BACKWARD ? end - 1 - here : mine - begin;
#pragma unroll 4
    for (int64_t i = 0; i < count; ++i) {
      const int64_t at = (BACKWARD ? end - 1 - i : begin + i) * p.d + col;
      float a[VEC], x[VEC];
      IO::load(gates + at, a);
      IO::load(second + at, x);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if constexpr (BACKWARD)
          h[v] = a[v] * (x[v] + h[v]);
        else
          h[v] = i == 0 && !p.initial ? x[v] : fmaf(a[v], h[v], x[v]);
      }
    }
  }
};

template <typename T, typename OffT, int VEC, bool BACKWARD>
__global__ void __launch_bounds__(kScanThreads, 4) scan_fold_kernel(const ScanArgs p) {
  extern __shared__ unsigned scan_smem[];
  grid_dependents_launch();
  ScanWarp<T, OffT, VEC, BACKWARD> w(p, scan_smem);
  const unsigned tasks = static_cast<unsigned>(p.slabs * p.tiles);
  for (unsigned t = blockIdx.x * kScanWarps + (threadIdx.x >> 5); t < tasks; t += gridDim.x * kScanWarps) {
    const unsigned slab = t / p.tiles;
    w.go(slab, static_cast<int>(t - slab * p.tiles));
    w.mark();
    // A slab that ends a segment is a start for those after it.
    const bool closed = BACKWARD ? w.starts_at_first() : w.ends_at_last();
    ScanPair<VEC> f, total;
    int reset = 1, total_reset = 1;
    f.clear();
    total.clear();
    if (!closed) {
      reset = w.fold(f);
      scan_groups<VEC, BACKWARD>(f, reset, total, total_reset, p.shift);
    }
    if ((threadIdx.x & 31) < w.lanes && w.col_ok) total.store(p.pairs + slab * p.d + w.col, total_reset);
  }
}

// (a, h) of rows, and whether a segment starts in them (a does not count then).
struct ScanSpan {
  float a, h;
  bool reset;
  // This span after `first`.
  __device__ __forceinline__ void after(const ScanSpan &first) {
    if (reset) return;
    h = scan_apply(a, h, first.h);
    a *= first.a;
    reset = first.reset;
  }
};

__device__ __forceinline__ ScanSpan scan_span(const float2 &pair) {
  return ScanSpan{pair.x, pair.y, __float_as_uint(pair.x) == kScanReset};
}

// (Pairs and states are read past L1: the launch that writes them may still
// run when the one that reads them starts.)
//
// 4 columns (a sector of pairs) by 128 parts of the slabs a block: each thread
// composes its part, a doubling scan over the parts gives the state before each,
// and each thread goes through its part again (from registers up to 8 slabs a
// part).  Bound by latency.  A whole forward scan of f32 262001 x 100 takes 105
// us, 108 with 8 columns; 256 parts cost 6 us at bf16 65536 x 1024, where blocks
// of half the threads start beside more of fold's; 32 parts of 8 columns, with
// their pairs in registers, 7 us at 262001 x 100.
__global__ void __launch_bounds__(kJoinCols * kJoinParts) scan_join_kernel(const ScanArgs p) {
  __shared__ ScanSpan spans[2][kJoinParts][kJoinCols];
  const int c = threadIdx.x % kJoinCols, part = threadIdx.x / kJoinCols;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kJoinCols + c;
  const bool live = col < p.d;
  const int64_t per = (p.slabs + kJoinParts - 1) / kJoinParts;
  const int64_t begin = min(part * per, p.slabs), end = live ? min(begin + per, p.slabs) : begin;
  const float2 *pairs = p.pairs + col;
  float *states = p.states + col;
  float2 pair[kJoinBatch];
  auto load = [&](int64_t s) {
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i)
      if (s + i < end) pair[i] = __ldcg(pairs + (s + i) * p.d);
  };
  grid_dependents_launch();
  grid_dependency_wait();
  ScanSpan all{1.0f, 0.0f, false};
#pragma unroll 1
  for (int64_t s = begin; s < end; s += kJoinBatch) {
    load(s);
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) {
      if (s + i < end) {
        ScanSpan next = scan_span(pair[i]);
        next.after(all);
        all = next;
      }
    }
  }
  int from = 0;
  spans[0][part][c] = all;
  __syncthreads();
#pragma unroll 1
  for (int off = 1; off < kJoinParts; off <<= 1) {
    if (part >= off) all.after(spans[from][part - off][c]);
    spans[from ^ 1][part][c] = all;
    from ^= 1;
    __syncthreads();
  }
  float state = part ? spans[from][part - 1][c].h : 0.0f;
#pragma unroll 1
  for (int64_t s = begin; s < end; s += kJoinBatch) {
    if (per > kJoinBatch) load(s);
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) {
      if (s + i < end) {
        states[(s + i) * p.d] = state;
        const ScanSpan x = scan_span(pair[i]);
        state = x.reset ? x.h : scan_apply(x.a, x.h, state);
      }
    }
  }
}

template <typename T, typename OffT, int VEC, bool BACKWARD>
__global__ void __launch_bounds__(kScanThreads, BACKWARD ? 2 : 3) scan_walk_kernel(const ScanArgs p) {
  constexpr int BATCH = kScanBatch;
  using IO = VecIO<T, VEC>;
  using Raw = typename IO::Raw;
  using State = VecIO<float, VEC>;
  extern __shared__ unsigned scan_smem[];
  const T *__restrict__ values = static_cast<const T *>(p.values);
  const T *__restrict__ gates = static_cast<const T *>(p.gates);
  const T *__restrict__ grads = static_cast<const T *>(p.grad_out);
  ScanWarp<T, OffT, VEC, BACKWARD> w(p, scan_smem);
  const unsigned tasks = static_cast<unsigned>(p.blocks * p.tiles);
  for (unsigned t = blockIdx.x * kScanWarps + (threadIdx.x >> 5); t < tasks; t += gridDim.x * kScanWarps) {
    const int64_t block = p.blocks - 1 - t / p.tiles;
    const int tile = static_cast<int>(t % p.tiles);
    if (block < p.slabs) {
      w.go(block, tile);
      w.mark();
      const uint64_t starts = w.lane_bits(w.m.start_mask), ends = w.lane_bits(w.m.end_mask);
      float h[VEC];
      if (!p.pairs) {
        w.catch_up(h);
      } else {
        grid_dependency_wait();
        ScanPair<VEC> f, total;
        int reset = 0, total_reset;
        f.clear();
        if (p.shift < 5) {  // rows of other lanes come before this lane's
          reset = w.fold(f);
          scan_groups<VEC, BACKWARD>(f, reset, total, total_reset, p.shift);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = 0.0f;
        if (w.col_ok && !(BACKWARD ? w.ends_at_last() : w.starts_at_first())) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) h[v] = __ldcg(p.states + w.pos * p.d + w.col + v);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = reset ? f.h[v] : scan_apply(f.a[v], f.h[v], h[v]);
      }
      const int batches = p.lane_rows / BATCH;
#pragma unroll 1
      for (int k = 0; k < batches; ++k) {
        const int batch = BACKWARD ? batches - 1 - k : k;
        const int64_t row = w.row0 + w.base + batch * BATCH;
        const int count = w.row_count(batch);
        if (count <= 0 || !w.col_ok) continue;
        const int64_t at = row * p.d + w.col;
        const unsigned start = static_cast<unsigned>(starts >> (batch * BATCH)) & ((1u << BATCH) - 1);
        const unsigned end = static_cast<unsigned>(ends >> (batch * BATCH)) & ((1u << BATCH) - 1);
        const int *start_seg = w.m.start_seg + w.base + batch * BATCH;
        const int *end_seg = w.m.end_seg + w.base + batch * BATCH;
        const bool plain = (start | end) == 0 && count == BATCH;
        Raw ra[BATCH], rx[BATCH];
        scan_rows<T, VEC>(gates + at, p.d, count, ra);
        scan_rows<T, VEC>(values + at, p.d, count, rx);
        // A row that starts a segment goes on from the initial state, or is its value.
        auto advance = [&](int i, float (&s)[VEC], bool alone) {
          float a[VEC], x[VEC];
          IO::unpack(ra[i], a);
          IO::unpack(rx[i], x);
#pragma unroll
          for (int v = 0; v < VEC; ++v) s[v] = alone ? x[v] : fmaf(a[v], s[v], x[v]);
        };
        if constexpr (!BACKWARD) {
          if (p.carries) State::store(p.carries + row / BATCH * p.d + w.col, h);
          T *to = static_cast<T *>(p.out) + at;
          if (plain) {
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
              advance(i, h, false);
              IO::store(to, h);
              to += p.d;
            }
          } else {
            // Four rows at a time, their initial states asked for together.
#pragma unroll
            for (int q = 0; q < BATCH; q += 4) {
              float first[4][VEC];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (q + i < count && ((start >> (q + i)) & 1)) w.state_of(p.initial, start_seg[q + i], first[i]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (q + i < count) {
                  const bool is_first = (start >> (q + i)) & 1;
#pragma unroll
                  for (int v = 0; v < VEC; ++v) h[v] = is_first ? first[i][v] : h[v];
                  advance(q + i, h, is_first && !p.initial);
                  IO::store(to, h);
                  to += p.d;
                  if (p.final_state && ((end >> (q + i)) & 1))
                    State::store(p.final_state + static_cast<int64_t>(end_seg[q + i]) * p.d + w.col, h);
                }
              }
            }
          }
        } else {
          Raw rg[BATCH];
          scan_rows<T, VEC>(grads + at, p.d, count, rg);
          float previous[BATCH][VEC], s[VEC];  // state before each row
          State::load(p.carries + row / BATCH * p.d + w.col, s);
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const bool is_first = (start >> i) & 1;
            if (is_first) w.state_of(p.initial, start_seg[i], s);
#pragma unroll
            for (int v = 0; v < VEC; ++v) previous[i][v] = s[v];
            advance(i, s, is_first && !p.initial);
          }
          const int64_t last = at + (count - 1) * p.d;
          T *to_values = p.grad_values ? static_cast<T *>(p.grad_values) + last : nullptr;
          T *to_gates = p.grad_gates ? static_cast<T *>(p.grad_gates) + last : nullptr;
#pragma unroll
          for (int i = BATCH - 1; i >= 0; --i) {
            if (i < count) {
              float a[VEC], g[VEC];
              IO::unpack(ra[i], a);
              IO::unpack(rg[i], g);
              if ((end >> i) & 1) w.state_of(p.grad_final, end_seg[i], h);
              const bool is_first = (start >> i) & 1, unused = is_first && !p.initial;
#pragma unroll
              for (int v = 0; v < VEC; ++v) g[v] += h[v];
              if (to_values) {
                IO::store(to_values, g);
                to_values -= p.d;
              }
#pragma unroll
              for (int v = 0; v < VEC; ++v) {
                h[v] = a[v] * g[v];
                g[v] = unused ? 0.0f : g[v] * previous[i][v];
              }
              if (to_gates) {
                IO::store(to_gates, g);
                to_gates -= p.d;
              }
              if (p.grad_initial && is_first)
                State::store(p.grad_initial + static_cast<int64_t>(start_seg[i]) * p.d + w.col, h);
            }
          }
        }
      }
    }
    // Segments without rows: the state passes through (as does its gradient).
    float *to = BACKWARD ? p.grad_initial : p.final_state;
    w.go(block, tile);
    if (block < p.slabs && p.clear_rest && w.col_ok) {
      const int stop = static_cast<int>(min(p.n - w.row0, static_cast<int64_t>(w.base + p.lane_rows)));
      const float zero[VEC] = {};
      for (int i = max(w.base, w.limit); i < stop; ++i) {
        const int64_t at = (w.row0 + i) * p.d + w.col;
        if constexpr (BACKWARD) {
          if (p.grad_values) IO::store(static_cast<T *>(p.grad_values) + at, zero);
          if (p.grad_gates) IO::store(static_cast<T *>(p.grad_gates) + at, zero);
        } else {
          IO::store(static_cast<T *>(p.out) + at, zero);
        }
      }
    }
    if (to && w.col_ok) {
      const int64_t stop = min(p.b, (block + 1) * p.per_block);
      for (int64_t s = block * p.per_block + ((threadIdx.x & 31) >> p.shift); s < stop; s += 32 >> p.shift) {
        if (static_cast<int64_t>(w.offsets[s]) < static_cast<int64_t>(w.offsets[s + 1])) continue;
        float x[VEC];
        w.state_of(BACKWARD ? p.grad_final : p.initial, s, x);
        State::store(to + s * p.d + w.col, x);
      }
    }
  }
}

}  // namespace rgb
