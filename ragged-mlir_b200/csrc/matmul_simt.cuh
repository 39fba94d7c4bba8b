// Segmented matrix products in f32 arithmetic on the FP32 pipes.
//
// f32 tensors take this kernel: the tensor cores round f32 operands to 10-bit
// (tf32) or fewer bits of mantissa.  A CTA of 256 threads computes a TILE x
// TILE block of the output, 8 x 8 (4 x 4) values a thread held in registers, from
// slices of 16 of the contraction in shared memory, the next slice on its way
// in registers.  Bound: 128 FMAs a clock and SM; a thread loads 16 values from
// shared memory for 64 FMAs, so the pipes and not the loads set the pace.
#pragma once

#include "matmul.cuh"

namespace rgb {

constexpr int kSimtThreads = 256;
constexpr int kSimtDepth = 16;

// LEFT_T / RIGHT_T: how the operand lies in memory.  Left: rows x depth, or
// (transposed) depth x rows; right: depth x cols, or (transposed) cols x depth.
template <typename OffT, int KIND, int TILE>
__global__ void __launch_bounds__(kSimtThreads) matmul_simt_kernel(const MatmulArgs p) {
  constexpr bool LEFT_T = KIND == MATMUL_GRAD_WEIGHTS, RIGHT_T = KIND == MATMUL_GRAD_VALUES;
  constexpr int DEPTH = kSimtDepth;
  constexpr int PER = TILE / 16;                      // outputs of a thread in each direction
  constexpr int LOADS = TILE * DEPTH / kSimtThreads;  // elements of an operand's slice a thread loads
  constexpr int PITCH = TILE + 4;
  __shared__ __align__(16) float left_s[2][DEPTH][PITCH], right_s[2][DEPTH][PITCH];
  const float *__restrict__ left = static_cast<const float *>(p.left);
  const float *__restrict__ right = static_cast<const float *>(p.right);
  float *__restrict__ out = static_cast<float *>(p.out);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  MatmulWalk<OffT, KIND, TILE> walk(p.offsets, p.b);
  MatmulTile t;
  for (int64_t index = blockIdx.x; walk.find(p, index, t); index += gridDim.x) {
    const int64_t col0 = static_cast<int64_t>(t.col_tile) * TILE;
    const int64_t depth = KIND == MATMUL_GRAD_WEIGHTS ? t.end - t.begin : p.depth;
    const float *lbase = left + (LEFT_T ? t.begin * p.left_pitch : int64_t{0});
    const float *rbase = right + (KIND == MATMUL_GRAD_WEIGHTS ? t.begin * p.right_pitch : t.seg * p.k * p.m);
    const int64_t row_limit = t.row_end, col_limit = p.cols;
    float lreg[LOADS], rreg[LOADS];
    auto load = [&](int64_t d0) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * kSimtThreads + threadIdx.x;
        {
          const int d = LEFT_T ? e / TILE : e % DEPTH, r = LEFT_T ? e % TILE : e / DEPTH;
          const int64_t row = t.row + r, at = LEFT_T ? (d0 + d) * p.left_pitch + row : row * p.left_pitch + d0 + d;
          lreg[i] = row < row_limit && d0 + d < depth ? __ldg(lbase + at) : 0.0f;
        }
        {
          const int d = RIGHT_T ? e % DEPTH : e / TILE, c = RIGHT_T ? e / DEPTH : e % TILE;
          const int64_t col = col0 + c, at = RIGHT_T ? col * p.right_pitch + d0 + d : (d0 + d) * p.right_pitch + col;
          rreg[i] = col < col_limit && d0 + d < depth ? __ldg(rbase + at) : 0.0f;
        }
      }
    };
    auto stage = [&](int buffer) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * kSimtThreads + threadIdx.x;
        if (LEFT_T)
          left_s[buffer][e / TILE][e % TILE] = lreg[i];
        else
          left_s[buffer][e % DEPTH][e / DEPTH] = lreg[i];
        if (RIGHT_T)
          right_s[buffer][e % DEPTH][e / DEPTH] = rreg[i];
        else
          right_s[buffer][e / TILE][e % TILE] = rreg[i];
      }
    };
    // Columns in pairs, for the packed FMA.
    unsigned long long acc[PER][PER / 2];
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < PER / 2; ++j) acc[i][j] = 0;
    if (depth > 0) load(0);
    int buffer = 0;
    for (int64_t d0 = 0; d0 < depth; d0 += DEPTH, buffer ^= 1) {
      stage(buffer);
      __syncthreads();  // the slice is there; the other buffer's readers are done
      if (d0 + DEPTH < depth) load(d0 + DEPTH);
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        float l[PER];
        unsigned long long r[PER / 2];
        // A thread's rows and columns lie in groups of 4, 64 apart: its vector
        // loads then meet no other thread's banks.
#pragma unroll
        for (int g = 0; g < PER / 4; ++g) {
          const float4 v = *reinterpret_cast<const float4 *>(&left_s[buffer][d][g * 64 + ty * 4]);
          l[g * 4] = v.x; l[g * 4 + 1] = v.y; l[g * 4 + 2] = v.z; l[g * 4 + 3] = v.w;
          const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(&right_s[buffer][d][g * 64 + tx * 4]);
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
    float *to = out + (KIND == MATMUL_GRAD_WEIGHTS ? t.seg * p.k * p.m : int64_t{0});
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t row = t.row + (i / 4) * 64 + ty * 4 + i % 4;
      if (row >= row_limit) continue;
#pragma unroll
      for (int j = 0; j < PER / 2; ++j) {
        const int64_t col = col0 + (j / 2) * 64 + tx * 4 + (j % 2) * 2;
        float lo, hi;
        unpack2(acc[i][j], lo, hi);
        if (col < col_limit) to[row * p.out_pitch + col] = lo;
        if (col + 1 < col_limit) to[row * p.out_pitch + col + 1] = hi;
      }
    }
    __syncthreads();  // the last slice has been read
  }
}

}  // namespace rgb
