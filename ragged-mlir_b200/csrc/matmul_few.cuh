// The segmented product of few rows a segment (single tokens): out[t] =
// values[t] @ weights[s], where reading the weights once is the work.
//
// A tile is up to 8 rows of a segment by 16 lanes of 16-byte column vectors.
// The 16 half-warps of a CTA split the contraction, each taking every 16th row
// of the weights, 16 of them on their way into shared memory at a time (a
// thread reads what it copied: no barrier), and keep f32 sums of all rows of
// the tile; the sums meet in shared memory, in the order of the half-warps.
// 32 rows in 16 segments, 1024 x 2048: bf16 21 us for the 50 MB of the 12 segments
// with rows, f32 24 for 101 MB, from L2 as from device memory.  Bound: 192 tiles of
// 256 KB on 148 SMs, so that a third of the SMs carries two (bf16), and the first
// loads' way.  For bf16 tensor-core tiles read the
// same bytes and start later, but take more rows at no cost; for f32 the other
// kernel's tiles compute 64 rows where few are there.
#pragma once

#include "matmul.cuh"

namespace rgb {

constexpr int kFewThreads = 256;
constexpr int kFewParts = kFewThreads / 16;
constexpr int kFewRows = 8;
constexpr int kFewDepth = 1024;  // of the values in shared memory at a time
constexpr int kFewAhead = 16;    // weight rows of a half-warp on their way, in groups
constexpr int kFewGroup = 4;

template <typename T>
constexpr int few_cols() {
  return 16 * (16 / Elem<T>::kBytes);
}
constexpr int kFewRing = kFewAhead * kFewThreads * 16;  // bytes; the parts' sums take its place
constexpr int kFewSmem = kFewRing + kFewRows * kFewDepth * 4;
static_assert(kFewRing >= kFewParts * kFewRows * few_cols<__nv_bfloat16>() * 4, "the sums fit the ring");

template <typename T, int ROWS>
__device__ __forceinline__ void few_tile(const MatmulArgs &p, const MatmulTile &t, float *smem) {
  constexpr int VEC = 16 / Elem<T>::kBytes, COLS = few_cols<T>();
  using IO = VecIO<T, VEC>;
  const int part = threadIdx.x / 16, lane = threadIdx.x % 16;
  const int64_t col = static_cast<int64_t>(t.col_tile) * COLS + lane * VEC;
  const bool live = col < p.cols;
  const int rows = static_cast<int>(t.row_end - t.row);
  const T *values = static_cast<const T *>(p.left) + t.row * p.left_pitch;
  const T *weights = static_cast<const T *>(p.right) + t.seg * p.k * p.m + (live ? col : 0);
  float sum[ROWS][VEC];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int v = 0; v < VEC; ++v) sum[r][v] = 0.0f;
  float *x_smem = smem + kFewRing / 4;
  unsigned char *ring = reinterpret_cast<unsigned char *>(smem) + threadIdx.x * 16;
  for (int64_t k0 = 0; k0 < p.k; k0 += kFewDepth) {
    const int depth = static_cast<int>(min(p.k - k0, int64_t{kFewDepth}));
    const int mine = (depth - part + kFewParts - 1) / kFewParts;  // weight rows of this half-warp
    const T *w = weights + (k0 + part) * p.m;
    auto copy = [&](int group) {  // starts the copies of a group of its rows
#pragma unroll
      for (int i = 0; i < kFewGroup; ++i) {
        const int row = group * kFewGroup + i;
        if (row < mine) cp_async<16>(smem_u32(ring + row % kFewAhead * (kFewThreads * 16)), w + int64_t{kFewParts} * row * p.m);
      }
      cp_async_commit();
    };
    __syncthreads();  // the last slice (or sums) have been read
#pragma unroll
    for (int g = 0; g < kFewAhead / kFewGroup - 1; ++g) copy(g);
#pragma unroll 4
    for (int k = threadIdx.x; k < depth; k += kFewThreads) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        float x[1] = {0.0f};
        if (r < rows) VecIO<T, 1>::load(values + r * p.left_pitch + k0 + k, x);
        x_smem[k * ROWS + r] = x[0];
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int g = 0; g * kFewGroup < mine; ++g) {
      copy(g + kFewAhead / kFewGroup - 1);
      cp_async_wait<kFewAhead / kFewGroup - 1>();
#pragma unroll
      for (int i = 0; i < kFewGroup; ++i) {
        const int row = g * kFewGroup + i;
        if (row < mine) {
          float y[VEC];
          IO::unpack(*reinterpret_cast<const typename IO::Raw *>(ring + row % kFewAhead * (kFewThreads * 16)), y);
          const float *x = x_smem + (row * kFewParts + part) * ROWS;
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const float xr = x[r];
#pragma unroll
            for (int v = 0; v < VEC; ++v) sum[r][v] = fmaf(xr, y[v], sum[r][v]);
          }
        }
      }
    }
    cp_async_wait<0>();
  }
  __syncthreads();  // the ring has been read
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int v = 0; v < VEC; ++v) smem[(part * ROWS + r) * COLS + lane * VEC + v] = sum[r][v];
  __syncthreads();
  T *out = static_cast<T *>(p.out);
  for (int i = threadIdx.x; i < rows * COLS; i += kFewThreads) {
    const int r = i / COLS, c = i % COLS;
    const int64_t at = static_cast<int64_t>(t.col_tile) * COLS + c;
    if (at >= p.cols) continue;
    float x[1] = {0.0f};
#pragma unroll
    for (int q = 0; q < kFewParts; ++q) x[0] += smem[(q * ROWS + r) * COLS + c];
    VecIO<T, 1>::store(out + (t.row + r) * p.m + at, x);
  }
}

template <typename T, typename OffT>
__global__ void __launch_bounds__(kFewThreads, 2) matmul_few_kernel(const MatmulArgs p) {
  extern __shared__ __align__(16) float few_smem[];
  MatmulWalk<OffT, MATMUL_FORWARD, kFewRows> walk(p.offsets, p.b);
  MatmulTile t;
  for (int64_t index = blockIdx.x; walk.find(p, index, t); index += gridDim.x) {
    const int rows = static_cast<int>(t.row_end - t.row);
    if (rows == 1)
      few_tile<T, 1>(p, t, few_smem);
    else if (rows == 2)
      few_tile<T, 2>(p, t, few_smem);
    else if (rows <= 4)
      few_tile<T, 4>(p, t, few_smem);
    else
      few_tile<T, 8>(p, t, few_smem);
  }
  matmul_clear_rest<T, OffT>(p, int64_t{blockIdx.x} * kFewThreads + threadIdx.x, int64_t{gridDim.x} * kFewThreads);
}

}  // namespace rgb
