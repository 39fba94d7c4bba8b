// Launch code of the segmented matrix products (kernels: matmul_tensor.cuh for
// bf16, matmul_simt.cuh for f32, matmul_few.cuh for few rows a segment).
#include <algorithm>
#include <cstring>

#include "internal.h"
#include "matmul_few.cuh"
#include "matmul_pair.cuh"
#include "matmul_simt.cuh"
#include "matmul_tensor.cuh"

namespace rgb {

namespace {

// (The times beside the rules are of single launches between events, inputs cold:
// they come in steps of 2 us, and a difference of one step decides nothing.)
constexpr int64_t kMaxWidth = 65536;

struct MatmulShape {
  int64_t rows, cols, depth;         // rows (depth) of a segment's product in the weights kind (else): N
  int64_t left_rows, left_cols;      // operands as matrices
  int64_t right_rows, right_cols;
  int64_t left_pitch, right_pitch;   // after packing
  bool few;                          // the few-rows kernel computes it
  bool pack_left, pack_right;
  int splits;                        // of the segments' rows, in the weights kind
  int64_t left_at, right_at, parts_at, bytes;  // workspace
};

// The weights kind's tiles, `tile` rows by `cols` columns (f32: tile by tile),
// and the parts that each segment's rows are split into.  A few tiles of long
// segments leave SMs idle: parts give each SM one (bf16) or two (f32), of 1024
// rows at least (bf16; 256, f32), since each costs a write and a read of its f32
// sums.  Of one segment of 65536 rows, 512 x 512: 61 us in 9 parts, 260 in one,
// bf16; 622 in 18 parts, 2240 in one, f32.  8 segments of 1024 rows, 128 x 128:
// 22 us in parts of 512 rows, 14 in one, bf16.
struct WeightsPlan {
  int tile, cols, splits;
};

int parts_of(int64_t slots, int64_t tiles, int64_t rows, int64_t least) {
  return static_cast<int>(std::max<int64_t>(1, std::min(slots / tiles, rows / least)));
}

WeightsPlan plan_weights(int dtype, int64_t k, int64_t m, int64_t n, int64_t b) {
  if (dtype == RG_DTYPE_BF16) {
    const int cols = m > 64 ? 128 : 64;
    return {128, cols, parts_of(148, b * ceil_div(k, 128) * ceil_div(m, cols), n / b, 1024)};
  }
  const int64_t large = b * ceil_div(k, 128) * ceil_div(m, 128), small = b * ceil_div(k, 64) * ceil_div(m, 64);
  if (large >= 148) return {128, 128, 1};
  if (small >= 296) return {64, 64, 1};
  // 128 x 128 in parts that fill three quarters of the SMs, else 64 x 64 (one
  // segment as above: 872 us; 8 segments of 1024 rows, 128 x 128: 22 and 43 us).
  const int parts = parts_of(296, large, n / b, 256);
  if (large * parts >= 111) return {128, 128, parts};
  return {64, 64, parts_of(296, small, n / b, 256)};
}

int64_t status_bytes() { return 1024 * 8; }

bool takes_tma(const void *p, int64_t cols) { return cols % 8 == 0 && aligned(p, 16); }

// Whether a forward product goes row by row of the weights (columns in whole
// 16-byte vectors).  f32: up to 16 rows a segment on average.  1024 x 2048
// weights, 16 segments: 32 rows 37 us, 137 with tiles of 64; 256 rows 72 and 137;
// 1024 rows 225 and 219; all of 1024 rows in one segment 213 and 150.  bf16: up
// to two rows a segment, 256 in all.  There 16 rows 20.5 us, 26.6 with tensor-core
// tiles; 32 rows 24.6 and 28.7; 48 rows 30.7 and 28.7; 512 rows in 256 segments of
// 512 x 512 43 and 37; 512 rows in one segment 94 and 14.
// (Decided once, on the caller's operands: a copy of them is aligned and has
// another pitch.)
bool takes_few(int kind, int dtype, int64_t m, int64_t n, int64_t b, const void *right) {
  if (kind != MATMUL_FORWARD || m % (16 / elem_bytes(dtype)) || !aligned(right, 16)) return false;
  return dtype == RG_DTYPE_F32 ? n <= 16 * b : n <= 2 * b && n <= 256;
}

MatmulShape make_shape(int kind, int dtype, int64_t k, int64_t m, int64_t n, int64_t b, const void *left,
                       const void *right) {
  MatmulShape s{};
  s.rows = kind == MATMUL_GRAD_WEIGHTS ? k : n;
  s.cols = kind == MATMUL_GRAD_VALUES ? k : m;
  s.depth = kind == MATMUL_FORWARD ? k : kind == MATMUL_GRAD_VALUES ? m : n;
  s.left_rows = n;
  s.left_cols = kind == MATMUL_GRAD_VALUES ? m : k;
  s.right_rows = kind == MATMUL_GRAD_WEIGHTS ? n : b * k;
  s.right_cols = m;
  s.left_pitch = s.left_cols;
  s.right_pitch = s.right_cols;
  s.splits = kind == MATMUL_GRAD_WEIGHTS && b ? plan_weights(dtype, k, m, n, b).splits : 1;
  if (s.splits > 1) {
    s.parts_at = status_bytes();
    s.bytes = align256(s.parts_at + s.splits * b * k * m * 4);
  }
  s.few = takes_few(kind, dtype, m, n, b, right);
  if (dtype == RG_DTYPE_F32 || s.few) return s;
  if (!s.bytes) s.bytes = status_bytes();
  if (!takes_tma(left, s.left_cols)) {
    s.pack_left = true;
    s.left_pitch = (s.left_cols + 7) / 8 * 8;
    s.left_at = s.bytes;
    s.bytes = align256(s.bytes + s.left_rows * s.left_pitch * 2);
  }
  if (!takes_tma(right, s.right_cols)) {
    s.pack_right = true;
    s.right_pitch = (s.right_cols + 7) / 8 * 8;
    s.right_at = s.bytes;
    s.bytes = align256(s.bytes + s.right_rows * s.right_pitch * 2);
  }
  return s;
}

int check_shape(int kind, int dtype, int index_dtype, int64_t k, int64_t m, int64_t n, int64_t b) {
  if (kind < MATMUL_FORWARD || kind > MATMUL_GRAD_WEIGHTS)
    return fail(RG_ERR_INVALID_ARGUMENT, "kind must be forward, gradient of values or gradient of weights");
  if (dtype != RG_DTYPE_F32 && dtype != RG_DTYPE_BF16) return fail(RG_ERR_INVALID_ARGUMENT, "dtype must be f32 or bf16");
  if (index_dtype != RG_INDEX_I32 && index_dtype != RG_INDEX_I64)
    return fail(RG_ERR_INVALID_ARGUMENT, "offsets dtype must be i32 or i64");
  if (k < 1 || k > kMaxWidth || m < 1 || m > kMaxWidth)
    return fail(RG_ERR_INVALID_ARGUMENT, "K and M must lie in [1, 65536]");
  if (n < 0 || b < 0) return fail(RG_ERR_INVALID_ARGUMENT, "N and B must be nonnegative");
  if (b == 0 && n != 0) return fail(RG_ERR_INVALID_ARGUMENT, "B=0 requires N=0");
  if (n > 2147483647LL || b > 2147483647LL)
    return fail(RG_ERR_INVALID_ARGUMENT, "a matrix product takes up to 2^31 - 1 rows and segments");
  if (b > INT64_MAX / 16 / (k * m)) return fail(RG_ERR_INVALID_ARGUMENT, "tensor byte size overflows signed 64-bit");
  return RG_OK;
}

// Row tiles of `tile` rows, at most: a segment has one that is not full.
int64_t most_row_tiles(int kind, const MatmulArgs &p, int tile) {
  return kind == MATMUL_GRAD_WEIGHTS ? p.splits * p.b * ceil_div(p.k, tile) : p.n / tile + std::min(p.n, p.b);
}

template <typename OffT, int KIND, int TILE, int SIZE>
int launch_simt_tile(MatmulArgs p, const DeviceProps &dev, cudaStream_t stream, rg_report *report) {
  const auto kernel = matmul_simt_kernel<OffT, KIND, TILE, SIZE>;
  int per_sm = 0;
  constexpr int smem = simt_smem_bytes(TILE);
  const int status =
      prepare_kernel(reinterpret_cast<const void *>(kernel), dev.device, kSimtThreads, smem, smem, &per_sm);
  if (status) return status;
  p.col_tiles = static_cast<int>(ceil_div(p.cols, TILE));
  p.row_tiles = static_cast<int>(ceil_div(p.k, TILE));
  const int64_t tiles = most_row_tiles(KIND, p, TILE) * p.col_tiles;
  const dim3 grid(static_cast<unsigned>(std::min(tiles, static_cast<int64_t>(per_sm) * dev.sm_count)), 1, 1);
  kernel<<<grid, kSimtThreads, smem, stream>>>(p);
  record_launch(report, K_MATMUL_SIMT, grid, kSimtThreads, smem);
  return check_cuda(cudaGetLastError(), "matmul_simt_kernel launch");
}

// 128 x 128 tiles where they give two thirds of the SMs one, else 64 x 64: 8192
// rows x 512 x 512 in 16 segments 104 us, 150 with tiles of 64; 4096 rows in 8
// segments 57 and 80; 1024 rows in 8 segments (32 tiles) 55 and 43; 2048 rows in
// 64 segments (64 tiles, a quarter full) 98 and 76.  16-byte pieces where all
// rows start at 16-byte boundaries.
template <typename OffT, int KIND>
int launch_simt(const MatmulArgs &p, const DeviceProps &dev, cudaStream_t stream, rg_report *report) {
  const bool large = KIND == MATMUL_GRAD_WEIGHTS
                         ? plan_weights(RG_DTYPE_F32, p.k, p.m, p.n, p.b).tile == 128
                         : ceil_div(p.n, 128) * ceil_div(p.cols, 128) >= dev.sm_count * 2 / 3;
  if (p.k % 4 == 0 && p.m % 4 == 0 && aligned(p.left, 16) && aligned(p.right, 16) && aligned(p.out, 16)) {
    if (large) return launch_simt_tile<OffT, KIND, 128, 4>(p, dev, stream, report);
    return launch_simt_tile<OffT, KIND, 64, 4>(p, dev, stream, report);
  }
  if (large) return launch_simt_tile<OffT, KIND, 128, 1>(p, dev, stream, report);
  return launch_simt_tile<OffT, KIND, 64, 1>(p, dev, stream, report);
}

// Tensor maps of the operands: boxes of 128 rows of the left one (32 for the
// last rows of a segment) and `right` columns of the right one.
template <int KIND>
int make_maps(TensorMaps &maps, const MatmulArgs &p, int right) {
  int status = RG_OK;
  std::memset(&maps, 0, sizeof maps);
  constexpr bool weights = KIND == MATMUL_GRAD_WEIGHTS;
  const int64_t left_cols = KIND == MATMUL_GRAD_VALUES ? p.m : p.k;
  if (weights && left_cols % 64 == 0) {
    const int64_t dims[3] = {64, p.n, left_cols / 64}, strides[2] = {p.left_pitch, 64};
    const int box[3] = {64, kTensorDepth, 128 / 64};
    status = make_tensor_map(&maps.left, p.left, 3, dims, strides, box);
    maps.left_slabs = 1;
  } else {
    const int64_t dims[2] = {left_cols, p.n};
    const int box[2] = {64, weights ? kTensorDepth : 128}, part[2] = {64, 32};
    status = make_tensor_map(&maps.left, p.left, 2, dims, &p.left_pitch, box);
    if (!status && !weights) status = make_tensor_map(&maps.left_part, p.left, 2, dims, &p.left_pitch, part);
  }
  if (status) return status;
  maps.right_slabs = KIND != MATMUL_GRAD_VALUES && p.m % 64 == 0;
  if (weights && maps.right_slabs) {
    const int64_t dims[3] = {64, p.n, p.m / 64}, strides[2] = {p.right_pitch, 64};
    const int box[3] = {64, kTensorDepth, right / 64};
    status = make_tensor_map(&maps.right, p.right, 3, dims, strides, box);
  } else if (weights) {
    const int64_t dims[2] = {p.m, p.n};
    const int box[2] = {64, kTensorDepth};
    status = make_tensor_map(&maps.right, p.right, 2, dims, &p.right_pitch, box);
  } else if (maps.right_slabs) {
    const int64_t dims[4] = {64, p.k, p.m / 64, p.b}, strides[3] = {p.right_pitch, 64, p.right_pitch * p.k};
    const int box[4] = {64, kTensorDepth, right / 64, 1};
    status = make_tensor_map(&maps.right, p.right, 4, dims, strides, box);
  } else {
    const int64_t dims[3] = {p.m, p.k, p.b}, strides[2] = {p.right_pitch, p.right_pitch * p.k};
    const int box[3] = {64, KIND == MATMUL_FORWARD ? kTensorDepth : right, 1};
    status = make_tensor_map(&maps.right, p.right, 3, dims, strides, box);
  }
  if (status) return status;
  return RG_OK;
}

// After a pack launch the product may start before that ends (its roles wait).
int launch_after_pack(void (*kernel)(MatmulArgs, TensorMaps), dim3 grid, int smem, const MatmulArgs &p,
                      const TensorMaps &maps, cudaStream_t stream) {
  cudaLaunchAttribute serial;
  serial.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  serial.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(kTensorThreads, 1, 1);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &serial;
  config.numAttrs = p.packed ? 1 : 0;
  return check_cuda(cudaLaunchKernelEx(&config, kernel, p, maps), "segmented product launch");
}

template <typename OffT, int KIND, int COLS>
int launch_tensor_cols(MatmulArgs p, const DeviceProps &dev, cudaStream_t stream, rg_report *report) {
  const auto kernel = matmul_tensor_kernel<OffT, KIND, COLS>;
  const int smem = tensor_smem_bytes(COLS);
  int per_sm = 0;
  int status = prepare_kernel(reinterpret_cast<const void *>(kernel), dev.device, kTensorThreads, smem, smem, &per_sm);
  TensorMaps maps;
  if (!status) status = make_maps<KIND>(maps, p, COLS);
  if (status) return status;
  p.col_tiles = static_cast<int>(ceil_div(p.cols, COLS));
  p.row_tiles = static_cast<int>(ceil_div(p.k, kTensorRows));
  const int64_t tiles = most_row_tiles(KIND, p, kTensorRows) * p.col_tiles;
  const dim3 grid(static_cast<unsigned>(std::min(tiles, static_cast<int64_t>(std::min(dev.sm_count * tensor_ctas(COLS), 1024)))), 1, 1);
  record_launch(report, K_MATMUL_TENSOR, grid, kTensorThreads, smem);
  return launch_after_pack(kernel, grid, smem, p, maps, stream);
}

template <typename OffT, int KIND>
int launch_pair(MatmulArgs p, const DeviceProps &dev, cudaStream_t stream, rg_report *report) {
  const auto kernel = matmul_pair_kernel<OffT, KIND>;
  int per_sm = 0;
  int status =
      prepare_kernel(reinterpret_cast<const void *>(kernel), dev.device, kTensorThreads, kPairSmem, kPairSmem, &per_sm);
  TensorMaps maps;
  if (!status) status = make_maps<KIND>(maps, p, kPairCols / 2);
  if (status) return status;
  p.col_tiles = static_cast<int>(ceil_div(p.cols, kPairCols));
  p.row_tiles = static_cast<int>(ceil_div(p.k, kPairRows));
  const int64_t tiles = most_row_tiles(KIND, p, kPairRows) * p.col_tiles;
  const dim3 grid(static_cast<unsigned>(2 * std::min(tiles, static_cast<int64_t>(std::min(dev.sm_count, 1024) / 2))), 1, 1);
  record_launch(report, K_MATMUL_PAIR, grid, kTensorThreads, kPairSmem);
  return launch_after_pack(kernel, grid, kPairSmem, p, maps, stream);
}

// Pairs of SMs where their tiles of 256 x 256 keep all SMs busy twice over and few
// of a tile's rows are past a segment's end; else the widest tiles of one SM that
// give every SM one (128 columns: half of the SMs, which computes 2048 rows x 512
// x 512 in 8 segments in 10 us, 12 with 64).  In us, for pairs, 256 and 128
// columns: 65536 rows x 2048 x 2048 in 16 segments 360, 379, 526; 16384 rows x 1024
// x 2048 in 8 segments 64, 68, 88; in 32 segments 72, 74, 98; 8192 rows in 32
// segments 55, 53, 61.
template <typename OffT, int KIND>
int launch_tensor(const MatmulArgs &p, const DeviceProps &dev, cudaStream_t stream, rg_report *report) {
  // (a segment's last row tile is counted half)
  const int64_t row_tiles = KIND == MATMUL_GRAD_WEIGHTS ? p.b * ceil_div(p.k, kTensorRows)
                                                         : p.n / kTensorRows + std::max<int64_t>(std::min(p.n, p.b) / 2, 1);
  const int64_t pair_rows = KIND == MATMUL_GRAD_WEIGHTS ? p.b * ceil_div(p.k, kPairRows) : p.n / kPairRows;
  const bool full = KIND == MATMUL_GRAD_WEIGHTS ? p.k > 128 : p.n >= 512 * std::min(p.n, p.b);
  if (p.cols > 128 && full && pair_rows * ceil_div(p.cols, kPairCols) >= dev.sm_count)
    return launch_pair<OffT, KIND>(p, dev, stream, report);
  if (p.cols > 128 && row_tiles * ceil_div(p.cols, 256) >= dev.sm_count)
    return launch_tensor_cols<OffT, KIND, 256>(p, dev, stream, report);
  const bool wide = KIND == MATMUL_GRAD_WEIGHTS ? plan_weights(RG_DTYPE_BF16, p.k, p.m, p.n, p.b).cols == 128
                                                 : p.cols > 64 && row_tiles * ceil_div(p.cols, 128) >= dev.sm_count / 2;
  if (wide) return launch_tensor_cols<OffT, KIND, 128>(p, dev, stream, report);
  return launch_tensor_cols<OffT, KIND, 64>(p, dev, stream, report);
}

template <typename T, typename OffT>
int launch_few(MatmulArgs p, const DeviceProps &dev, cudaStream_t stream, rg_report *report) {
  const auto kernel = matmul_few_kernel<T, OffT>;
  constexpr int smem = kFewSmem;
  int per_sm = 0;
  const int status = prepare_kernel(reinterpret_cast<const void *>(kernel), dev.device, kFewThreads, smem, smem, &per_sm);
  if (status) return status;
  p.col_tiles = static_cast<int>(ceil_div(p.cols, few_cols<T>()));
  const int64_t tiles = most_row_tiles(MATMUL_FORWARD, p, kFewRows) * p.col_tiles;
  const dim3 grid(static_cast<unsigned>(std::min(tiles, static_cast<int64_t>(per_sm) * dev.sm_count)), 1, 1);
  kernel<<<grid, kFewThreads, smem, stream>>>(p);
  record_launch(report, K_MATMUL_FEW, grid, kFewThreads, smem);
  return check_cuda(cudaGetLastError(), "matmul_few_kernel launch");
}

template <typename OffT>
int launch_kind(int kind, int dtype, bool few, const MatmulArgs &p, const DeviceProps &dev, cudaStream_t stream,
                rg_report *report) {
  if (few) {
    if (dtype == RG_DTYPE_F32) return launch_few<float, OffT>(p, dev, stream, report);
    return launch_few<__nv_bfloat16, OffT>(p, dev, stream, report);
  }
  if (dtype == RG_DTYPE_F32) {
    if (kind == MATMUL_FORWARD) return launch_simt<OffT, MATMUL_FORWARD>(p, dev, stream, report);
    if (kind == MATMUL_GRAD_VALUES) return launch_simt<OffT, MATMUL_GRAD_VALUES>(p, dev, stream, report);
    return launch_simt<OffT, MATMUL_GRAD_WEIGHTS>(p, dev, stream, report);
  }
  if (kind == MATMUL_FORWARD) return launch_tensor<OffT, MATMUL_FORWARD>(p, dev, stream, report);
  if (kind == MATMUL_GRAD_VALUES) return launch_tensor<OffT, MATMUL_GRAD_VALUES>(p, dev, stream, report);
  return launch_tensor<OffT, MATMUL_GRAD_WEIGHTS>(p, dev, stream, report);
}

int pack(const PackArgs &left, const PackArgs &right, const DeviceProps &dev, cudaStream_t stream, rg_report *report) {
  const int64_t rows = left.rows + right.rows;
  if (rows == 0) return RG_OK;
  const dim3 grid(static_cast<unsigned>(std::min(ceil_div(rows, 8), static_cast<int64_t>(dev.sm_count) * 8)), 1, 1);
  matmul_pack_kernel<<<grid, 256, 0, stream>>>(left, right);
  record_launch(report, K_MATMUL_PACK, grid, 256, 0);
  return check_cuda(cudaGetLastError(), "matmul_pack_kernel launch");
}

}  // namespace

}  // namespace rgb

using namespace rgb;

extern "C" {

int rg_matmul_workspace_bytes(int kind, int dtype, int index_dtype, int64_t k, int64_t m, int64_t n, int64_t b,
                              const void *left, const void *right, int64_t *bytes) {
  if (!bytes) return fail(RG_ERR_INVALID_ARGUMENT, "bytes is NULL");
  const int status = check_shape(kind, dtype, index_dtype, k, m, n, b);
  if (status) return status;
  *bytes = make_shape(kind, dtype, k, m, n, b, left, right).bytes;
  return RG_OK;
}

int rg_matmul(int kind, int dtype, int index_dtype, int64_t k, int64_t m, int64_t n, int64_t b, const void *left,
              const void *right, const void *offsets, void *out, void *workspace, int64_t workspace_bytes,
              void *stream, rg_report *report) {
  clear_report(report);
  const bool clear_rest = dtype & RG_CLEAR_REST;
  dtype &= ~RG_CLEAR_REST;
  int status = check_shape(kind, dtype, index_dtype, k, m, n, b);
  if (status) return status;
  const MatmulShape s = make_shape(kind, dtype, k, m, n, b, left, right);
  const int esize = elem_bytes(dtype), isize = index_dtype == RG_INDEX_I32 ? 4 : 8;
  const int64_t out_bytes = (kind == MATMUL_GRAD_WEIGHTS ? b * k * m : n * s.cols) * esize;
  if (b == 0 || out_bytes == 0) return RG_OK;
  const TensorRange ranges[] = {
      {"the left operand", left, s.left_rows * s.left_cols * esize, esize, false},
      {"the right operand", right, s.right_rows * s.right_cols * esize, esize, false},
      {"offsets", offsets, (b + 1) * isize, isize, false},
      {"out", out, out_bytes, esize, true}};
  status = check_ranges(ranges, 4);
  if (status) return status;
  DeviceProps dev;
  status = check_device(&dev);
  if (status) return status;
  cudaStream_t on = static_cast<cudaStream_t>(stream);
  if (kind == MATMUL_GRAD_WEIGHTS && n == 0) {  // no rows at all: no operand to map
    if (report) report->memsets = 1;
    return check_cuda(cudaMemsetAsync(out, 0, out_bytes, on), "cudaMemsetAsync");
  }
  if (report) {
    report->workspace_bytes = s.bytes;
    report->d_vector = 1;
    report->d_tile = 1;
    report->status_offset = dtype == RG_DTYPE_BF16 && !s.few ? 0 : -1;
  }
  if (s.bytes) {
    if (!workspace || workspace_bytes < s.bytes) return fail(RG_ERR_WORKSPACE, "workspace missing or too small");
    if (!aligned(workspace, 256)) return fail(RG_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  }
  MatmulArgs p{};
  p.left = left;
  p.right = right;
  p.offsets = offsets;
  p.out = out;
  p.n = n;
  p.b = b;
  p.k = k;
  p.m = m;
  p.rows = s.rows;
  p.cols = s.cols;
  p.depth = s.depth;
  p.left_pitch = s.left_pitch;
  p.right_pitch = s.right_pitch;
  p.out_pitch = s.cols;
  p.splits = s.splits;
  p.parts = s.splits > 1 ? reinterpret_cast<float *>(static_cast<char *>(workspace) + s.parts_at) : nullptr;
  p.status = static_cast<unsigned long long *>(workspace);
  p.packed = s.pack_left || s.pack_right;
  p.clear_rest = clear_rest && kind != MATMUL_GRAD_WEIGHTS;
  char *scratch = static_cast<char *>(workspace);
  if (s.pack_left || s.pack_right) {
    PackArgs packed[2] = {};
    if (s.pack_left) {
      p.left = scratch + s.left_at;
      packed[0] = {static_cast<const __nv_bfloat16 *>(left), reinterpret_cast<__nv_bfloat16 *>(scratch + s.left_at),
                   s.left_rows, s.left_cols, s.left_pitch};
    }
    if (s.pack_right) {
      p.right = scratch + s.right_at;
      packed[1] = {static_cast<const __nv_bfloat16 *>(right), reinterpret_cast<__nv_bfloat16 *>(scratch + s.right_at),
                   s.right_rows, s.right_cols, s.right_pitch};
    }
    status = pack(packed[0], packed[1], dev, on, report);
    if (status) return status;
  }
  status = index_dtype == RG_INDEX_I32 ? launch_kind<int32_t>(kind, dtype, s.few, p, dev, on, report)
                                       : launch_kind<int64_t>(kind, dtype, s.few, p, dev, on, report);
  if (status || s.splits == 1) return status;
  const int64_t count = b * k * m;
  const dim3 grid(static_cast<unsigned>(std::min(ceil_div(count, 256), static_cast<int64_t>(dev.sm_count) * 8)), 1, 1);
  if (dtype == RG_DTYPE_F32)
    matmul_parts_kernel<float><<<grid, 256, 0, on>>>(p.parts, static_cast<float *>(out), count, s.splits);
  else
    matmul_parts_kernel<__nv_bfloat16><<<grid, 256, 0, on>>>(p.parts, static_cast<__nv_bfloat16 *>(out), count, s.splits);
  record_launch(report, K_MATMUL_PARTS, grid, 256, 0);
  return check_cuda(cudaGetLastError(), "matmul_parts_kernel launch");
}

}  // extern "C"
