// Segmented matrix products: out[t] = left[t] @ right[s] for the rows t of
// segment s, and the two products of its backward pass.
//
//   kind     out                  left (rows x contraction)   right
//   forward  [N, M]               values [N, K]               weights[s] [K, M]
//   values   [N, K] (gradient)    grad_out [N, M]             weights[s] transposed
//   weights  [s] [K, M] (grad.)   values_s transposed         grad_out_s
//
// This file has what both kernels share: the list of output tiles, which the
// device derives from the offsets.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "common.cuh"

namespace rgb {

enum MatmulKind : int { MATMUL_FORWARD = 0, MATMUL_GRAD_VALUES = 1, MATMUL_GRAD_WEIGHTS = 2 };

struct MatmulArgs {
  const void *left, *right, *offsets;
  void *out;
  int64_t n, b;
  int64_t k, m;              // widths of values and of out (forward)
  int64_t rows, cols, depth; // of a product; for the kinds whose rows (depth) are a segment's: unused
  int64_t left_pitch, right_pitch, out_pitch;  // elements between rows
  int col_tiles;
  int row_tiles;             // weights kind: row tiles of a segment
  // Weights kind, where there are few tiles and long segments: each segment's
  // rows in `splits` parts, with a sum each in `parts` (f32 [splits][B][K][M]).
  int splits;
  float *parts;
  unsigned long long *status;
  bool packed;               // a pack launch comes right before
  bool clear_rest;           // rows of the output behind the last segment: set to zero, else left alone
};

// One output tile: rows [row, row_end) of the output (of segment `seg` for the
// weights kind), and the segment's rows [begin, end).
struct MatmulTile {
  int64_t seg, row, row_end, begin, end;
  int col_tile, split;
};

// Walks a CTA's tiles, in ascending order.  Forward and values: the tiles of a
// segment are its rows in steps of TILE, so the segment of a tile is found by
// counting them, 32 segments at a time and on from the last one found.  All
// lanes of a warp take part and get the same answer.
template <typename OffT, int KIND, int TILE>
struct MatmulWalk {
  const OffT *__restrict__ offsets;
  int64_t b, first, before;  // tiles before segment `first`
  __device__ __forceinline__ MatmulWalk(const void *o, int64_t segments)
      : offsets(static_cast<const OffT *>(o)), b(segments), first(0), before(0) {}

  // False past the last tile.  `n` clamps offsets that are out of order.
  __device__ __forceinline__ bool find(const MatmulArgs &p, int64_t index, MatmulTile &t) {
    t.col_tile = static_cast<int>(index % p.col_tiles);
    const int64_t tile = index / p.col_tiles;
    if constexpr (KIND == MATMUL_GRAD_WEIGHTS) {
      const int64_t part = tile / p.row_tiles;
      t.split = static_cast<int>(part / b);
      if (t.split >= p.splits) return false;
      t.seg = part - t.split * b;
      t.row = (tile - part * p.row_tiles) * TILE;
      t.row_end = min(t.row + TILE, p.rows);
      t.begin = min(max(static_cast<int64_t>(offsets[t.seg]), int64_t{0}), p.n);
      t.end = max(min(static_cast<int64_t>(offsets[t.seg + 1]), p.n), t.begin);
      if (p.splits > 1) {  // (parts of whole slices of 64)
        const int64_t per = ((t.end - t.begin + p.splits - 1) / p.splits + 63) / 64 * 64;
        t.begin = min(t.begin + t.split * per, t.end);
        t.end = min(t.begin + per, t.end);
      }
      return true;
    } else {
      const int lane = threadIdx.x & 31;
      for (;;) {
        if (first >= b) return false;
        const int64_t s = first + lane;
        int64_t lo = 0, hi = 0;
        if (s < b) {
          lo = min(max(static_cast<int64_t>(offsets[s]), int64_t{0}), p.n);
          hi = max(min(static_cast<int64_t>(offsets[s + 1]), p.n), lo);
        }
        int64_t sum = (hi - lo + TILE - 1) / TILE;  // tiles up to this lane's segment
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int64_t up = __shfl_up_sync(~0u, sum, off);
          if (lane >= off) sum += up;
        }
        const unsigned past = __ballot_sync(~0u, before + sum > tile);
        if (past) {
          const int src = __ffs(past) - 1;
          const int64_t up = __shfl_up_sync(~0u, sum, 1);
          const int64_t start = __shfl_sync(~0u, lane ? up : int64_t{0}, src) + before;
          t.begin = __shfl_sync(~0u, lo, src);
          t.end = __shfl_sync(~0u, hi, src);
          t.seg = first + src;
          t.row = t.begin + (tile - start) * TILE;
          t.row_end = min(t.row + TILE, t.end);
          return true;
        }
        before += __shfl_sync(~0u, sum, 31);
        first += 32;
      }
    }
  }
};

// Rows of the output behind the last segment: zeros, by `count` threads of which
// this is number `at`.  They are one range of memory, written in 16-byte pieces.
template <typename T, typename OffT>
__device__ __forceinline__ void matmul_clear_rest(const MatmulArgs &p, int64_t at, int64_t count) {
  if (!p.clear_rest) return;
  const int64_t used = min(max(static_cast<int64_t>(static_cast<const OffT *>(p.offsets)[p.b]), int64_t{0}), p.n);
  T *from = static_cast<T *>(p.out) + used * p.out_pitch, *to = static_cast<T *>(p.out) + p.n * p.out_pitch;
  const int64_t elements = to - from;
  constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
  const int64_t head = min(static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(from) & 15)) & 15) / int64_t{sizeof(T)},
                           elements);
  const int64_t pieces = (elements - head) / kPiece;
  uint4 *body = reinterpret_cast<uint4 *>(from + head);
  for (int64_t i = at; i < pieces; i += count) body[i] = uint4{0, 0, 0, 0};
  const T zero = static_cast<T>(0.0f);
  if (at < head) from[at] = zero;
  if (at < elements - head - pieces * kPiece) to[-1 - at] = zero;
}

// The parts' sums, in order, rounded once.
template <typename T>
__global__ void __launch_bounds__(256) matmul_parts_kernel(const float *__restrict__ parts, T *__restrict__ out,
                                                           int64_t count, int splits) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += int64_t{gridDim.x} * 256) {
    float sum[1] = {0.0f};
#pragma unroll 4
    for (int z = 0; z < splits; ++z) sum[0] += parts[z * count + i];
    VecIO<T, 1>::store(out + i, sum);
  }
}

}  // namespace rgb
