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
// A the product of the gates.  A CTA takes a chunk of rows by a tile of at
// most 128 bytes of columns, keeps its inputs in registers, and
//   1. folds (A, H) per thread, warp and chunk and publishes the chunk's pair;
//   2. gets the state before the chunk from the chunks its segment started
//      in (the start row is known from the offsets, so no flag is read past it);
//   3. runs the recurrence over its rows from that state and writes them.
// Every input is read once and every output written once, which is the bound:
// the recurrence itself is one FMA an element.
//
// Step 2 folds a fixed tree (chunks of its group of 16, groups of its
// supergroup of 16, then the state at the last supergroup's end), so the
// result does not depend on which CTA came first, and the serial chain is one
// hop per 256 chunks.  Chunks are handed out by a ticket in dependence order:
// whoever waits waits on CTAs that already run.  Waits are bounded; one that
// gives up sets the call's status word and goes on.
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
constexpr int kScanCols = 64;     // columns of a tile at most
constexpr int kScanFan = 16;      // chunks per group, groups per supergroup
constexpr int kScanWaitLimit = 1 << 22;

// Rows a thread keeps in registers: 4 with the full 16-byte vectors, 8 of the
// narrower ones.
__host__ __device__ constexpr int scan_rows(int elem_bytes, int vec) { return vec * elem_bytes == 16 ? 4 : 8; }

struct ScanArgs {
  const void *values, *gates, *offsets;
  const float *initial;  // [B, D] or null
  int64_t n, d;
  int64_t b;
  int shift;        // log2 of the lanes across a tile's columns
  int vec_cols;     // D / VEC
  int tiles;        // column tiles
  int64_t chunks;   // chunks that hold rows
  int64_t blocks;   // chunks launched (more than `chunks` where many segments are empty)
  float *carries;   // [chunks, D] state before each chunk (written by forward, read by backward)
  // forward
  void *out;
  float *final_state;  // [B, D] or null
  // backward
  const void *grad_out;
  const float *grad_final;  // [B, D] or null
  void *grad_values, *grad_gates;
  float *grad_initial;  // [B, D] or null
  // workspace (null with a single chunk)
  unsigned *ticket;
  unsigned long long *status;
  unsigned *flags;        // chunk, group and supergroup flags
  float2 *pairs;          // (A, H) of chunks, then of groups
  float *supers;          // state at each supergroup's end
};

__device__ __forceinline__ float scan_apply(float a, float h, float state) {
  return state == 0.0f ? h : fmaf(a, state, h);
}

__device__ __forceinline__ void st_release_gpu(unsigned *p, unsigned v) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// Waits until *flag is set (bounded).
__device__ __forceinline__ void scan_wait(const unsigned *flag, unsigned long long *status) {
  for (int i = 0; i < kScanWaitLimit; ++i) {
    if (ld_acquire_gpu(flag)) return;
    if (i > 16) __nanosleep(32);
  }
  atomicMax(status, 1ull);
}

// Segment starts of a chunk's rows, in shared memory.  start[i]: the segment
// whose rows begin at row row0 + i (-1: none; of empty segments and the one
// with rows that share an offset, the last, which has the rows).  ended[i]:
// one past the segment whose rows end before row row0 + i (INT_MAX: none).
struct ScanMarks {
  int *start;
  int *ended;
  int last;  // segment of the chunk's last row
};

constexpr int kNoEnd = 0x7fffffff;

// Segment of row `row` (the last one that starts at or before it), by all
// threads of the CTA: a 256-way search, one round for up to 256 segments.
template <typename OffT>
__device__ __forceinline__ int64_t scan_find(const OffT *__restrict__ offsets, int64_t b, int64_t row) {
  int64_t lo = 0, hi = b;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + kScanThreads - 1) / kScanThreads;
    const int64_t at = lo + threadIdx.x * step;
    const int count = __syncthreads_count(threadIdx.x == 0 || (at < hi && static_cast<int64_t>(offsets[at]) <= row));
    const int64_t next = lo + count * step;
    lo += (count - 1) * step;
    if (next < hi) hi = next;
  }
  return lo;
}

// Fills the marks of rows [row0, row0 + rows]; `first` is the segment of row0.
// Offsets outside the chunk write nothing, whatever they hold.
template <typename OffT>
__device__ __forceinline__ void scan_mark(const OffT *__restrict__ offsets, int64_t b, int64_t first, int64_t row0,
                                          int rows, int64_t end_row, int *start, int *ended, int *last) {
  for (int64_t s = first + threadIdx.x; s <= b; s += kScanThreads) {
    const int64_t at = static_cast<int64_t>(offsets[s]) - row0;
    if (at > rows) break;
    if (s == first) {
      if (at == 0) atomicMax(&start[0], static_cast<int>(s));
      continue;
    }
    if (at < 0) continue;
    atomicMin(&ended[at], static_cast<int>(s));
    if (s == b) continue;  // the end of the last segment starts none
    atomicMax(&start[at], static_cast<int>(s));
    if (at < end_row - row0) atomicMax(last, static_cast<int>(s));
  }
}

// Inclusive-to-exclusive composition over a warp's row groups (lanes of one
// group hold one group's columns).  REV composes from the last group down.
// On return a, h, reset describe the groups before this one (after it, REV);
// the warp's total goes to `total` / `total_reset`.
template <int VEC, bool REV>
__device__ __forceinline__ void scan_warp(float (&a)[VEC], float (&h)[VEC], int &reset, int shift, float2 *total,
                                          int *total_reset) {
  const int lane = threadIdx.x & 31;
  const int lanes = 1 << shift;
  for (int off = lanes; off < 32; off <<= 1) {
    const bool live = REV ? lane + off < 32 : lane >= off;
    const int r = REV ? __shfl_down_sync(~0u, reset, off) : __shfl_up_sync(~0u, reset, off);
    const bool take = live && !reset;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float pa = REV ? __shfl_down_sync(~0u, a[v], off) : __shfl_up_sync(~0u, a[v], off);
      const float ph = REV ? __shfl_down_sync(~0u, h[v], off) : __shfl_up_sync(~0u, h[v], off);
      if (take) {
        h[v] = scan_apply(a[v], h[v], ph);
        a[v] *= pa;
      }
    }
    if (take) reset = r;
  }
  const bool is_total = REV ? lane < lanes : lane >= 32 - lanes;
  if (is_total) {
    const int col = (lane & (lanes - 1)) * VEC;
#pragma unroll
    for (int v = 0; v < VEC; ++v) total[col + v] = make_float2(a[v], h[v]);
    *total_reset = reset;
  }
  const bool edge = REV ? lane >= 32 - lanes : lane < lanes;
  reset = REV ? __shfl_down_sync(~0u, reset, lanes & 31) : __shfl_up_sync(~0u, reset, lanes & 31);
  if (edge) reset = 0;
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const float pa = REV ? __shfl_down_sync(~0u, a[v], lanes & 31) : __shfl_up_sync(~0u, a[v], lanes & 31);
    const float ph = REV ? __shfl_down_sync(~0u, h[v], lanes & 31) : __shfl_up_sync(~0u, h[v], lanes & 31);
    a[v] = edge ? 1.0f : pa;
    h[v] = edge ? 0.0f : ph;
  }
}

// State before chunk `pos` of this thread's column (threads of the tile's
// columns only; whole warps).  (a, h, reset) is the chunk's own pair and
// `first` the chunk in which the segment of the chunk's first row starts
// (`pos`: the chunk starts with a segment).  Positions count in the order of
// the recurrence.  Each warp publishes and polls for its own 32 columns.
__device__ __forceinline__ float scan_lookback(const ScanArgs &p, int tile, int64_t pos, int64_t first, int width,
                                               float a, float h, bool reset) {
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int col = threadIdx.x;
  const int64_t groups = (p.chunks + kScanFan - 1) / kScanFan;
  const int64_t slots = static_cast<int64_t>(p.tiles) * 2;
  unsigned *chunk_flags = p.flags + tile * 2 + warp;
  unsigned *group_flags = chunk_flags + p.chunks * slots;
  unsigned *super_flags = group_flags + groups * slots;
  const int64_t pitch = static_cast<int64_t>(p.tiles) * kScanCols;
  float2 *chunk_pairs = p.pairs + tile * kScanCols + col;
  float2 *group_pairs = chunk_pairs + p.chunks * pitch;
  float *supers = p.supers + tile * kScanCols + col;
  const bool live = col < width;

  auto publish = [&](unsigned *flag) {
    __threadfence();
    __syncwarp();
    if (lane == 0) st_release_gpu(flag, 1u);
  };

  if (live) chunk_pairs[pos * pitch] = make_float2(a, h);
  publish(chunk_flags + pos * slots);

  const int64_t group = pos / kScanFan;
  float fa = 1.0f, fh = 0.0f;     // the group's chunks before this one
  bool fixed = first == pos;      // (fa, fh) starts at a segment: no state before it counts
  if (!fixed) {
    const int64_t c0 = max(first, group * kScanFan);
    const int count = static_cast<int>(pos - c0);
    if (lane < count) scan_wait(chunk_flags + (c0 + lane) * slots, p.status);
    __syncwarp();
    float2 part[kScanFan - 1];
#pragma unroll
    for (int i = 0; i < kScanFan - 1; ++i)
      part[i] = i < count && live ? __ldcg(chunk_pairs + (c0 + i) * pitch) : make_float2(1.0f, 0.0f);
    fixed = c0 == first;
#pragma unroll
    for (int i = 0; i < kScanFan - 1; ++i) {
      if (i < count) {
        fh = i == 0 ? part[0].y : scan_apply(part[i].x, part[i].y, fh);
        fa *= part[i].x;
      }
    }
  }
  if (pos % kScanFan == kScanFan - 1) {
    // A pair that starts at a segment is read only as the first of a fold or
    // under a state that a later pair replaces: its A does not matter.
    if (live) group_pairs[group * pitch] = reset ? make_float2(a, h) : make_float2(fa * a, scan_apply(a, h, fh));
    publish(group_flags + group * slots);
  }
  float state = fh;
  if (!fixed) {
    const int64_t super = group / kScanFan, first_group = first / kScanFan;
    const bool before = first_group < super * kScanFan;  // the segment started before this supergroup
    const int64_t g0 = max(first_group, super * kScanFan);
    const int count = static_cast<int>(group - g0);
    if (lane < count) scan_wait(group_flags + (g0 + lane) * slots, p.status);
    if (before && lane == 31) scan_wait(super_flags + (super - 1) * slots, p.status);
    __syncwarp();
    float2 part[kScanFan - 1];
#pragma unroll
    for (int i = 0; i < kScanFan - 1; ++i)
      part[i] = i < count && live ? __ldcg(group_pairs + (g0 + i) * pitch) : make_float2(1.0f, 0.0f);
    float s = before && live ? __ldcg(supers + (super - 1) * pitch) : 0.0f;
#pragma unroll
    for (int i = 0; i < kScanFan - 1; ++i)
      if (i < count) s = i == 0 && !before ? part[0].y : scan_apply(part[i].x, part[i].y, s);
    state = scan_apply(fa, fh, s);
  }
  if (pos % (kScanFan * kScanFan) == kScanFan * kScanFan - 1) {
    if (live) supers[pos / (kScanFan * kScanFan) * pitch] = reset ? h : scan_apply(a, h, state);
    publish(super_flags + pos / (kScanFan * kScanFan) * slots);
  }
  return state;
}

struct ScanShared {
  float2 total[kScanWarps][kScanCols];
  float carry[kScanWarps][kScanCols];  // state before each warp's rows
  float before[kScanCols];             // backward: the recorded state before the chunk
  int total_reset[kScanWarps];
  int last;
  unsigned ticket;
};

// From the warps' totals: the chunk's pair, the state before it (lookback
// unless `first` is this chunk) and the state before each warp's rows.  All
// threads; ends with a barrier.
template <bool REV>
__device__ __forceinline__ void scan_chunk(const ScanArgs &p, ScanShared &sh, int tile, int64_t pos, int64_t first,
                                           int width) {
  __syncthreads();
  const int col = threadIdx.x;
  if (threadIdx.x < ((width + 31) & ~31)) {
    const bool live = col < width;
    float state = 0.0f;
    if (p.ticket) {
      float a = 1.0f, h = 0.0f;
      bool reset = false;
#pragma unroll
      for (int i = 0; i < kScanWarps; ++i) {
        const int w = REV ? kScanWarps - 1 - i : i;
        const float2 t = live ? sh.total[w][col] : make_float2(1.0f, 0.0f);
        if (sh.total_reset[w]) {
          h = t.y;
          reset = true;
        } else {
          h = scan_apply(t.x, t.y, h);
          a *= t.x;
        }
      }
      state = scan_lookback(p, tile, pos, first, width, a, h, reset);
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < kScanWarps; ++i) {
        const int w = REV ? kScanWarps - 1 - i : i;
        sh.carry[w][col] = state;
        const float2 t = sh.total[w][col];
        state = sh.total_reset[w] ? t.y : scan_apply(t.x, t.y, state);
      }
    }
  }
  __syncthreads();
}

// Shared memory after ScanShared: start[rows + 1], ended[rows + 1].
template <typename T, typename OffT, int VEC, bool BACKWARD>
__global__ void __launch_bounds__(kScanThreads, 2) scan_kernel(const ScanArgs p) {
  constexpr int ROWS = scan_rows(Elem<T>::kBytes, VEC);
  using IO = VecIO<T, VEC>;
  using Raw = typename IO::Raw;
  using State = VecIO<float, VEC < 4 ? VEC : 4>;  // f32 states move in pieces of up to 16 bytes
  constexpr int kPiece = VEC < 4 ? VEC : 4;
  __shared__ ScanShared sh;
  extern __shared__ int scan_smem[];
  const OffT *__restrict__ offsets = static_cast<const OffT *>(p.offsets);
  const T *__restrict__ values = static_cast<const T *>(p.values);
  const T *__restrict__ gates = static_cast<const T *>(p.gates);

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lanes = 1 << p.shift;
  const int rows = (kScanThreads >> p.shift) * ROWS;
  int *start = scan_smem, *ended = scan_smem + rows + 1;

  unsigned task = blockIdx.x;
  if (p.ticket) {
    if (threadIdx.x == 0) sh.ticket = atomicAdd(p.ticket, 1u);
    __syncthreads();
    task = sh.ticket;
  }
  const int tile = static_cast<int>(task % p.tiles);
  const int64_t block = task / p.tiles;
  // Chunk of this CTA, in the order of the recurrence; the extra blocks come last.
  const int64_t pos = block;
  const int64_t chunk = BACKWARD ? p.chunks - 1 - block : block;
  const int vc = tile * lanes + (threadIdx.x & (lanes - 1));
  const bool col_ok = vc < p.vec_cols;
  const int64_t col = static_cast<int64_t>(vc) * VEC;
  const int local_col = (threadIdx.x & (lanes - 1)) * VEC;
  const int width = min(lanes, p.vec_cols - tile * lanes) * VEC;

  auto load_state = [&](const float *at, float (&x)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC / kPiece; ++i) {
      float y[kPiece];
      State::load(at + i * kPiece, y);
#pragma unroll
      for (int v = 0; v < kPiece; ++v) x[i * kPiece + v] = y[v];
    }
  };
  auto store_state = [&](float *at, const float (&x)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC / kPiece; ++i) {
      float y[kPiece];
#pragma unroll
      for (int v = 0; v < kPiece; ++v) y[v] = x[i * kPiece + v];
      State::store(at + i * kPiece, y);
    }
  };

  if (block < p.chunks) {
    const int64_t row0 = chunk * rows;
    const int64_t end_row = min(row0 + rows, p.n);
    const int group = threadIdx.x >> p.shift;
    const int64_t my_row = row0 + static_cast<int64_t>(group) * ROWS;
    const int base = group * ROWS;

    Raw ra[ROWS], rx[ROWS], rg[BACKWARD ? ROWS : 1];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const bool ok = col_ok && my_row + i < p.n;
      const int64_t at = (my_row + i) * p.d + col;
      ra[i] = ok ? IO::load_raw(gates + at) : Raw{};
      rx[i] = ok ? IO::load_raw(values + at) : Raw{};
      if constexpr (BACKWARD) rg[i] = ok ? IO::load_raw(static_cast<const T *>(p.grad_out) + at) : Raw{};
    }

    for (int i = threadIdx.x; i <= rows; i += kScanThreads) {
      start[i] = -1;
      ended[i] = kNoEnd;
    }
    if (threadIdx.x == 0) sh.last = -1;
    const int64_t seg0 = scan_find(offsets, p.b, row0);
    __syncthreads();
    scan_mark(offsets, p.b, seg0, row0, rows, end_row, start, ended, &sh.last);
    if (BACKWARD && threadIdx.x < width) {
      const int64_t begin = static_cast<int64_t>(offsets[seg0]);
      sh.before[threadIdx.x] = begin < row0 ? p.carries[chunk * p.d + static_cast<int64_t>(tile) * lanes * VEC +
                                                        threadIdx.x]
                                            : 0.0f;
    }
    __syncthreads();

    float previous[BACKWARD ? ROWS : 1][VEC];  // h before each row
    // ---------------------------------------------------- forward fold --
    // A row with a start replaces what came before by its initial state.
    {
      float a[VEC], h[VEC];
      int reset = 0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        a[v] = 1.0f;
        h[v] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        if (my_row + i < p.n) {
          float ga[VEC], x[VEC];
          IO::unpack(ra[i], ga);
          IO::unpack(rx[i], x);
          const int s = start[base + i];
          if (s >= 0) {
            reset = 1;
            if (p.initial && col_ok) {
              load_state(p.initial + s * p.d + col, h);
            } else {
#pragma unroll
              for (int v = 0; v < VEC; ++v) h[v] = 0.0f;
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = p.initial ? fmaf(ga[v], h[v], x[v]) : x[v];
          } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
              h[v] = fmaf(ga[v], h[v], x[v]);
              a[v] *= ga[v];
            }
          }
        }
      }
      scan_warp<VEC, false>(a, h, reset, p.shift, sh.total[warp], &sh.total_reset[warp]);
      if constexpr (!BACKWARD) {
        const int64_t begin = static_cast<int64_t>(offsets[seg0]);
        const int64_t first = begin >= row0 ? pos : (begin > 0 ? begin / rows : 0);
        scan_chunk<false>(p, sh, tile, pos, first, width);
        if (p.carries && threadIdx.x < width)
          p.carries[chunk * p.d + static_cast<int64_t>(tile) * lanes * VEC + threadIdx.x] = sh.carry[0][threadIdx.x];
        float state[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          state[v] = reset ? h[v] : scan_apply(a[v], h[v], col_ok ? sh.carry[warp][local_col + v] : 0.0f);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          if (col_ok && my_row + i < p.n) {
            float ga[VEC], x[VEC];
            IO::unpack(ra[i], ga);
            IO::unpack(rx[i], x);
            const int s = start[base + i];
            if (s >= 0 && !p.initial) {
#pragma unroll
              for (int v = 0; v < VEC; ++v) state[v] = x[v];
            } else {
              if (s >= 0) load_state(p.initial + s * p.d + col, state);
#pragma unroll
              for (int v = 0; v < VEC; ++v) state[v] = fmaf(ga[v], state[v], x[v]);
            }
            IO::store(static_cast<T *>(p.out) + (my_row + i) * p.d + col, state);
            const int e = ended[base + i + 1];
            if (p.final_state && e != kNoEnd) store_state(p.final_state + (static_cast<int64_t>(e) - 1) * p.d + col, state);
          }
        }
      } else {
        __syncthreads();
        if (threadIdx.x < width) {
          float state = sh.before[threadIdx.x];
#pragma unroll
          for (int w = 0; w < kScanWarps; ++w) {
            sh.carry[w][threadIdx.x] = state;
            const float2 t = sh.total[w][threadIdx.x];
            state = sh.total_reset[w] ? t.y : scan_apply(t.x, t.y, state);
          }
        }
        __syncthreads();
        float state[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          state[v] = reset ? h[v] : scan_apply(a[v], h[v], col_ok ? sh.carry[warp][local_col + v] : 0.0f);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          float ga[VEC], x[VEC];
          IO::unpack(ra[i], ga);
          IO::unpack(rx[i], x);
          const bool ok = col_ok && my_row + i < p.n;
          const int s = ok ? start[base + i] : -1;
          if (s >= 0) {
            if (p.initial) {
              load_state(p.initial + s * p.d + col, state);
            } else {
#pragma unroll
              for (int v = 0; v < VEC; ++v) state[v] = 0.0f;
            }
          }
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            previous[i][v] = state[v];
            state[v] = s >= 0 && !p.initial ? x[v] : fmaf(ga[v], state[v], x[v]);
          }
        }
        __syncthreads();
      }
    }

    // --------------------------------------------------- backward fold --
    if constexpr (BACKWARD) {
      float a[VEC], u[VEC];
      int reset = 0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        a[v] = 1.0f;
        u[v] = 0.0f;
      }
      auto at_end = [&](int i, float (&x)[VEC]) {  // u past row i where a segment ends there
        const int e = ended[base + i + 1];
        if (e == kNoEnd) return false;
        if (p.grad_final && col_ok) {
          load_state(p.grad_final + (static_cast<int64_t>(e) - 1) * p.d + col, x);
        } else {
#pragma unroll
          for (int v = 0; v < VEC; ++v) x[v] = 0.0f;
        }
        return true;
      };
#pragma unroll
      for (int i = ROWS - 1; i >= 0; --i) {
        if (my_row + i < p.n) {
          float ga[VEC], g[VEC];
          IO::unpack(ra[i], ga);
          IO::unpack(rg[i], g);
          if (at_end(i, u)) {
            reset = 1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) u[v] = ga[v] * (g[v] + u[v]);
          } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
              u[v] = ga[v] * (g[v] + u[v]);
              a[v] *= ga[v];
            }
          }
        }
      }
      scan_warp<VEC, true>(a, u, reset, p.shift, sh.total[warp], &sh.total_reset[warp]);
      const int64_t last = max(seg0, static_cast<int64_t>(sh.last));
      const int64_t stop = min(static_cast<int64_t>(offsets[last + 1]), p.n);
      const int64_t first = stop <= end_row ? pos : p.chunks - 1 - (stop - 1) / rows;
      scan_chunk<true>(p, sh, tile, pos, first, width);
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        u[v] = reset ? u[v] : scan_apply(a[v], u[v], col_ok ? sh.carry[warp][local_col + v] : 0.0f);
#pragma unroll
      for (int i = ROWS - 1; i >= 0; --i) {
        if (col_ok && my_row + i < p.n) {
          float ga[VEC], g[VEC];
          IO::unpack(ra[i], ga);
          IO::unpack(rg[i], g);
          at_end(i, u);
          const int s = start[base + i];
          const int64_t at = (my_row + i) * p.d + col;
#pragma unroll
          for (int v = 0; v < VEC; ++v) g[v] += u[v];
          if (p.grad_values) IO::store(static_cast<T *>(p.grad_values) + at, g);
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            u[v] = ga[v] * g[v];
            g[v] = s >= 0 && !p.initial ? 0.0f : g[v] * previous[i][v];
          }
          if (p.grad_gates) IO::store(static_cast<T *>(p.grad_gates) + at, g);
          if (p.grad_initial && s >= 0) store_state(p.grad_initial + s * p.d + col, u);
        }
      }
    }
  }

  // Segments without rows: the state passes through (as does its gradient).
  float *state_out = BACKWARD ? p.grad_initial : p.final_state;
  const float *state_in = BACKWARD ? p.grad_final : p.initial;
  if (state_out && col_ok) {
    const int64_t per = (p.b + p.blocks - 1) / p.blocks;
    const int64_t stop = min(p.b, (block + 1) * per);
    for (int64_t s = block * per + (threadIdx.x >> p.shift); s < stop; s += kScanThreads >> p.shift) {
      if (static_cast<int64_t>(offsets[s]) < static_cast<int64_t>(offsets[s + 1])) continue;
      float x[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[v] = 0.0f;
      if (state_in) load_state(state_in + s * p.d + col, x);
      store_state(state_out + s * p.d + col, x);
    }
  }
}

}  // namespace rgb
