// Segmented matrix products in f32 arithmetic on the FP32 pipes.
//
// f32 tensors take this kernel: the tensor cores round f32 operands to 10-bit
// (tf32) or fewer bits of mantissa.  A CTA of 256 threads computes a TILE x
// TILE block of the output, 8 x 8 (4 x 4) values a thread held in registers, from
// slices of 16 of the contraction in a ring of shared-memory stages that
// asynchronous copies fill three slices ahead; two CTAs an SM fill each other's
// waits.  Bound: 128 FMAs a clock and SM; a thread loads 16 values from shared
// memory for 64 FMAs, so the pipes and not the loads set the pace.  Packed FMAs
// (two columns at once) leave issue slots to the loads.
//
// 8192 rows x 512 x 512 in 8 segments: 98 us forward, 105 and 119 to 134 for the
// gradients of values and weights: 32 to 44 TFLOP/s of the pipes' 74.  288 tiles on
// 296 places are one wave, partly of rows past the segments' ends; within a tile the
// FMA pipe is busy 38 % in packed FMAs (two each), the issue slots half.
#pragma once

#include "matmul.cuh"

namespace rgb {

constexpr int kSimtThreads = 256;
constexpr int kSimtDepth = 16;
constexpr int kSimtStages = 4;

constexpr int simt_pitch(int tile) { return tile + 4; }
constexpr int simt_smem_bytes(int tile) { return kSimtStages * 2 * kSimtDepth * simt_pitch(tile) * 4; }

// Copies BYTES (4 or 16) or, not `ok`, writes zeros.
template <int BYTES>
__device__ __forceinline__ void copy_or_zero(uint32_t to, const float *from, bool ok) {
  const int count = ok ? BYTES : 0;
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from), "r"(count) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(to), "l"(from), "r"(count) : "memory");
}

// A thread's share of a slice of one operand, [contraction][tile] in shared
// memory.  ALONG: the tile's rows (columns) are contiguous in memory, and SIZE
// of them go at once; else the contraction is, and elements go one by one.
template <int TILE, int SIZE, bool ALONG>
struct SimtOperand {
  static constexpr int kSize = ALONG ? SIZE : 1;
  static constexpr int kPieces = TILE * kSimtDepth / (kSimtThreads * kSize);
  static constexpr int kAcross = (ALONG ? TILE : kSimtDepth) / kSize;  // pieces of a line
  static constexpr int kLines = kSimtThreads / kAcross;                // lines between a thread's pieces
  const float *base, *at;
  int64_t pitch;
  int line, place;  // of the first piece
  int64_t limit;    // lines (elements of a line) of the tile that exist

  __device__ __forceinline__ void begin(const float *from, int64_t row_pitch, int64_t first, int64_t end) {
    line = threadIdx.x / kAcross;
    place = threadIdx.x % kAcross * kSize;
    pitch = row_pitch;
    limit = end - first;
    base = from;
    at = ALONG ? base + line * pitch + first + place : base + (first + line) * pitch + place;
  }
  // Starts the copies of the slice with `left` of the contraction to go (none:
  // zeros); moves on to the next.
  __device__ __forceinline__ void copy(uint32_t stage, int64_t left) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int l = line + i * kLines;
      const bool ok = ALONG ? l < left && place < limit : l < limit && place < left;
      const uint32_t to = stage + (ALONG ? l * simt_pitch(TILE) + place : place * simt_pitch(TILE) + l) * 4;
      copy_or_zero<kSize * 4>(to, ok ? at + i * kLines * pitch : base, ok);
    }
    at += ALONG ? kSimtDepth * pitch : int64_t{kSimtDepth};
  }
};

template <typename OffT, int KIND, int TILE, int SIZE>
__global__ void __launch_bounds__(kSimtThreads, TILE == 128 ? 2 : 3) matmul_simt_kernel(const MatmulArgs p) {
  constexpr int DEPTH = kSimtDepth;
  constexpr int PER = TILE / 16;  // outputs of a thread in each direction
  constexpr int PITCH = simt_pitch(TILE);
  constexpr int kOperand = DEPTH * PITCH;  // floats of an operand's stage
  extern __shared__ __align__(16) float simt_smem[];
  float *__restrict__ out = static_cast<float *>(p.out);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  MatmulWalk<OffT, KIND, TILE> walk(p.offsets, p.b);
  MatmulTile t;
  SimtOperand<TILE, SIZE, KIND == MATMUL_GRAD_WEIGHTS> left;
  SimtOperand<TILE, SIZE, KIND != MATMUL_GRAD_VALUES> right;
  for (int64_t index = blockIdx.x; walk.find(p, index, t); index += gridDim.x) {
    const int64_t col0 = static_cast<int64_t>(t.col_tile) * TILE;
    const int64_t depth = KIND == MATMUL_GRAD_WEIGHTS ? t.end - t.begin : p.depth;
    left.begin(static_cast<const float *>(p.left) + (KIND == MATMUL_GRAD_WEIGHTS ? t.begin * p.left_pitch : int64_t{0}),
               p.left_pitch, t.row, t.row_end);
    right.begin(static_cast<const float *>(p.right) +
                    (KIND == MATMUL_GRAD_WEIGHTS ? t.begin * p.right_pitch : t.seg * p.k * p.m),
                p.right_pitch, col0, p.cols);
    // Columns in pairs, for the packed FMA.
    unsigned long long acc[PER][PER / 2];
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < PER / 2; ++j) acc[i][j] = 0;
    int64_t ahead = depth;  // of the contraction, not asked for yet
    auto copy = [&](int stage) {
      if (ahead > 0) {
        const uint32_t to = smem_u32(simt_smem + stage * 2 * kOperand);
        left.copy(to, ahead);
        right.copy(to + kOperand * 4, ahead);
      }
      ahead -= DEPTH;
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kSimtStages - 1; ++i) copy(i);
    int stage = 0;
#pragma unroll 1
    for (int64_t to_go = depth; to_go > 0; to_go -= DEPTH) {
      cp_async_wait<kSimtStages - 2>();
      __syncthreads();  // all copies of the slice are there, and the last slice's readers done
      copy((stage + kSimtStages - 1) % kSimtStages);
      const float *left_s = simt_smem + stage * 2 * kOperand, *right_s = left_s + kOperand;
      stage = (stage + 1) % kSimtStages;
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        float l[PER];
        unsigned long long r[PER / 2];
        // A thread's rows and columns lie in groups of 4, 64 apart: its vector
        // loads then meet no other thread's banks.
#pragma unroll
        for (int g = 0; g < PER / 4; ++g) {
          const float4 v = *reinterpret_cast<const float4 *>(left_s + d * PITCH + g * 64 + ty * 4);
          l[g * 4] = v.x; l[g * 4 + 1] = v.y; l[g * 4 + 2] = v.z; l[g * 4 + 3] = v.w;
          const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(right_s + d * PITCH + g * 64 + tx * 4);
          r[g * 2] = w.x;
          r[g * 2 + 1] = w.y;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const unsigned long long both = pack2(l[i], l[i]);
#pragma unroll
          for (int j = 0; j < PER / 2; ++j)
            asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[i][j]) : "l"(both), "l"(r[j]));
        }
      }
    }
    float *to = out;
    if constexpr (KIND == MATMUL_GRAD_WEIGHTS) to = (p.parts ? p.parts + t.split * p.b * p.k * p.m : out) + t.seg * p.k * p.m;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t row = t.row + (i / 4) * 64 + ty * 4 + i % 4;
      if (row >= t.row_end) continue;
#pragma unroll
      for (int g = 0; g < PER / 4; ++g) {
        const int64_t col = col0 + g * 64 + tx * 4;
        float *at = to + row * p.out_pitch + col;
        float x[4];
        unpack2(acc[i][g * 2], x[0], x[1]);
        unpack2(acc[i][g * 2 + 1], x[2], x[3]);
        if constexpr (SIZE == 4) {
          if (col < p.cols) *reinterpret_cast<float4 *>(at) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < p.cols) at[e] = x[e];
        }
      }
    }
    cp_async_wait<0>();
    __syncthreads();  // the last slice has been read
  }
  if constexpr (KIND != MATMUL_GRAD_WEIGHTS)
    matmul_clear_rest<float, OffT>(p, int64_t{blockIdx.x} * kSimtThreads + threadIdx.x, int64_t{gridDim.x} * kSimtThreads);
}

}  // namespace rgb
