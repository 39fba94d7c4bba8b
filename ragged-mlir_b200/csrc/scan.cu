// Launch code of the segmented scan (kernels and mathematics: scan.cuh).
#include <algorithm>
#include <cstdio>
#include <cstring>

#include "internal.h"
#include "scan.cuh"

namespace rgb {

namespace {

constexpr int64_t kMaxScanDim = 65536;

struct ScanShape {
  int vec, tiles, shift, lane_rows, row_shift;
  int64_t slabs, blocks;
};

// Whether walk is the only launch: up to 128 rows, or 512 of up to four a segment
// on average, where catching up costs less than two more launches.  In us, alone
// and in three launches, 1024 columns of bf16: 256 rows in 256 segments 16 and 27
// (backward 29 and 37), 512 in 128 14 and 21; 128 in 4 14 and 16; 256 in 4 18 and
// 16 (23 and 18); 512 in 4, the most that rows of unlike lengths can lose, 35 and 16.
bool walks_alone(int64_t n, int64_t b) { return n <= 128 || (n <= 512 && n <= 4 * b); }

// 32 lanes, or as many as cover a row, of one vector each: 8 bytes where they
// fill the lanes, else 4 (one element where D is odd).  8 bytes take two thirds
// of the instructions: bf16 65536 x 1024 139 us (backward 186), 166 (227) with 4;
// f32 262144 x 100 117 (158) and 131 (326), with a slower join than today's.  A lane takes 64 rows of a slab, fewer
// where that would leave resident warps without a task: f32 262144 x 100 117 us,
// 158 with 16; 4096 x 512 20 (23) with 16, 29 (35) with 64.  `align`: elements that
// all tensors are aligned for.
ScanShape make_shape(int dtype, int64_t d, int64_t n, int64_t b, int align) {
  ScanShape s;
  s.vec = 8 / elem_bytes(dtype);
  while (s.vec > align || d % s.vec || (s.vec * elem_bytes(dtype) == 8 && d < 32 * s.vec)) s.vec /= 2;
  s.shift = 0;
  while ((int64_t{1} << s.shift) * s.vec < d && s.shift < 5) ++s.shift;
  s.tiles = static_cast<int>(ceil_div(d, (int64_t{1} << s.shift) * s.vec));
  const int groups = 32 >> s.shift;
  constexpr int64_t warps = 148 * 24;  // of a B200 (the workspace is asked for without a device)
  s.lane_rows = 64;
  while (s.lane_rows > 16 && (ceil_div(n, s.lane_rows * groups) * s.tiles < warps || s.lane_rows * groups > 512))
    s.lane_rows /= 2;
  s.row_shift = 0;
  while ((1 << s.row_shift) < s.lane_rows * groups) ++s.row_shift;
  s.slabs = ceil_div(n, int64_t{1} << s.row_shift);
  // Empty segments are shared out over the tasks; 1024 of them keep one busy.
  s.blocks = s.slabs;
  if (s.blocks < ceil_div(b, 1024)) s.blocks = ceil_div(b, 1024);
  if (s.blocks < 1) s.blocks = 1;
  return s;
}

// Pairs, then states of each slab.
int64_t layout_bytes(const ScanShape &s, int64_t n, int64_t d, int64_t b) {
  return walks_alone(n, b) ? 0 : align256(s.slabs * d * 12);
}

int check_shape(int dtype, int index_dtype, int64_t d, int64_t n, int64_t b) {
  if (dtype != RG_DTYPE_F32 && dtype != RG_DTYPE_BF16) return fail(RG_ERR_INVALID_ARGUMENT, "dtype must be f32 or bf16");
  if (index_dtype != RG_INDEX_I32 && index_dtype != RG_INDEX_I64)
    return fail(RG_ERR_INVALID_ARGUMENT, "offsets dtype must be i32 or i64");
  if (d < 1 || d > kMaxScanDim) return fail(RG_ERR_INVALID_ARGUMENT, "D must lie in [1, 65536]");
  if (n < 0 || b < 0) return fail(RG_ERR_INVALID_ARGUMENT, "N and B must be nonnegative");
  if (b == 0 && n != 0) return fail(RG_ERR_INVALID_ARGUMENT, "B=0 requires N=0");
  if (b >= 2147483647LL) return fail(RG_ERR_INVALID_ARGUMENT, "a scan takes fewer than 2^31 - 1 segments");
  if (index_dtype == RG_INDEX_I32 && n > 2147483647LL)
    return fail(RG_ERR_INVALID_ARGUMENT, "N exceeds the i32 offsets range");
  if (n > INT64_MAX / d / 8 || b > INT64_MAX / d / 8)
    return fail(RG_ERR_INVALID_ARGUMENT, "tensor byte size overflows signed 64-bit");
  return RG_OK;
}

// Elements (4, 2 or 1) that all tensors are aligned for (in `r`: one's alignment).
int aligned_elements(const TensorRange *r, int count) {
  int most = 4;
  for (int i = 0; i < count; ++i)
    while (std::strcmp(r[i].name, "offsets") && r[i].bytes && !aligned(r[i].ptr, r[i].align * most)) most /= 2;
  return most;
}

template <typename T, typename OffT, int VEC, bool BACKWARD>
int launch(const ScanArgs &p, const ScanShape &s, const DeviceProps &dev, cudaStream_t stream, rg_report *report) {
  const int smem = kScanWarps * scan_marks_words(1 << s.row_shift) * 4;
  constexpr int usual = kScanWarps * scan_marks_words(64) * 4, limit = kScanWarps * scan_marks_words(512) * 4;
  // The second and third launch may start before the one before them ends.
  auto start = [&](void (*kernel)(ScanArgs), int id, int64_t ctas, int threads, int bytes, bool after) {
    cudaLaunchAttribute serial;
    serial.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    serial.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = bytes;
    config.stream = stream;
    config.attrs = &serial;
    config.numAttrs = after ? 1 : 0;
    record_launch(report, id, config.gridDim, threads, bytes);
    return check_cuda(cudaLaunchKernelEx(&config, kernel, p), "scan kernel launch");
  };
  auto run = [&](void (*kernel)(ScanArgs), int id, int64_t slabs, bool after) {
    int per_sm = 0;
    int status = prepare_kernel(reinterpret_cast<const void *>(kernel), dev.device, kScanThreads, usual, limit, &per_sm);
    if (status) return status;
    return start(kernel, id, std::min(static_cast<int64_t>(per_sm) * dev.sm_count, ceil_div(slabs * s.tiles, kScanWarps)),
                 kScanThreads, smem, after);
  };
  if (p.pairs) {
    int status = run(scan_fold_kernel<T, OffT, VEC, BACKWARD>, BACKWARD ? K_SCAN_FOLD_BACKWARD : K_SCAN_FOLD, s.slabs,
                     false);
    if (status) return status;
    status = start(scan_join_kernel, K_SCAN_JOIN, ceil_div(p.d, kJoinCols), kJoinCols * kJoinParts, 0, true);
    if (status) return status;
  }
  return run(scan_walk_kernel<T, OffT, VEC, BACKWARD>, BACKWARD ? K_SCAN_BACKWARD : K_SCAN, s.blocks,
             p.pairs != nullptr);
}

template <typename OffT, bool BACKWARD>
int launch_vec(int dtype, const ScanArgs &p, const ScanShape &s, const DeviceProps &dev, cudaStream_t stream,
               rg_report *report) {
  if (dtype == RG_DTYPE_F32) {
    if (s.vec == 2) return launch<float, OffT, 2, BACKWARD>(p, s, dev, stream, report);
    return launch<float, OffT, 1, BACKWARD>(p, s, dev, stream, report);
  }
  if (s.vec == 4) return launch<__nv_bfloat16, OffT, 4, BACKWARD>(p, s, dev, stream, report);
  if (s.vec == 2) return launch<__nv_bfloat16, OffT, 2, BACKWARD>(p, s, dev, stream, report);
  return launch<__nv_bfloat16, OffT, 1, BACKWARD>(p, s, dev, stream, report);
}

// Takes RG_CLEAR_REST out of a dtype.
bool take_clear_rest(int &dtype) {
  const bool clear = dtype & RG_CLEAR_REST;
  dtype &= ~RG_CLEAR_REST;
  return clear;
}

template <bool BACKWARD>
int run_scan(int dtype, int index_dtype, int align, ScanArgs &p, void *workspace, int64_t workspace_bytes,
             cudaStream_t stream, rg_report *report) {
  DeviceProps dev;
  int status = check_device(&dev);
  if (status) return status;
  const ScanShape s = make_shape(dtype, p.d, p.n, p.b, align);
  if (s.blocks > 2000000000LL / s.tiles) return fail(RG_ERR_INVALID_ARGUMENT, "the call needs more than 2e9 tasks");
  const int64_t need = layout_bytes(s, p.n, p.d, p.b);
  if (report) {
    report->workspace_bytes = need;
    report->d_vector = s.vec;
    report->d_tile = 1 << s.shift;
  }
  p.shift = s.shift;
  p.lane_rows = s.lane_rows;
  p.row_shift = s.row_shift;
  p.tiles = s.tiles;
  p.slabs = s.slabs;
  p.blocks = s.blocks;
  p.per_block = ceil_div(p.b, s.blocks);
  if (need) {
    if (!workspace || workspace_bytes < need) return fail(RG_ERR_WORKSPACE, "workspace missing or too small");
    if (!aligned(workspace, 256)) return fail(RG_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    p.pairs = static_cast<float2 *>(workspace);
    p.states = reinterpret_cast<float *>(p.pairs + s.slabs * p.d);
  }
  if (index_dtype == RG_INDEX_I32) return launch_vec<int32_t, BACKWARD>(dtype, p, s, dev, stream, report);
  return launch_vec<int64_t, BACKWARD>(dtype, p, s, dev, stream, report);
}

}  // namespace

}  // namespace rgb

using namespace rgb;

extern "C" {

int rg_scan_workspace_bytes(int dtype, int index_dtype, int64_t d, int64_t n, int64_t b, int64_t *bytes) {
  if (!bytes) return fail(RG_ERR_INVALID_ARGUMENT, "bytes is NULL");
  const int status = check_shape(dtype, index_dtype, d, n, b);
  if (status) return status;
  // (the slabs go by the tensors' alignment)
  *bytes = 0;
  for (int align = 1; align <= 4; align *= 2)
    *bytes = std::max(*bytes, layout_bytes(make_shape(dtype, d, n, b, align), n, d, b));
  return RG_OK;
}

int rg_scan(int dtype, int index_dtype, int64_t d, int64_t n, int64_t b, const void *values, const void *gates,
            const void *offsets, const float *initial, void *out, float *final_state, float *carries, void *workspace,
            int64_t workspace_bytes, void *stream, rg_report *report) {
  clear_report(report);
  const bool clear_rest = take_clear_rest(dtype);
  int status = check_shape(dtype, index_dtype, d, n, b);
  if (status) return status;
  if (b == 0) return RG_OK;
  const int esize = elem_bytes(dtype);
  const int isize = index_dtype == RG_INDEX_I32 ? 4 : 8;
  const int64_t full = n * d * esize, states = b * d * 4;
  const TensorRange ranges[] = {{"values", values, full, esize, false},
                          {"gates", gates, full, esize, false},
                          {"offsets", offsets, (b + 1) * isize, isize, false},
                          {"initial", initial, initial ? states : 0, 4, false},
                          {"out", out, full, esize, true},
                          {"final", final_state, final_state ? states : 0, 4, true},
                          {"carries", carries, carries ? ceil_div(n, kScanBatch) * d * 4 : 0, 4, true}};
  status = check_ranges(ranges, 7);
  if (status) return status;
  const int align = aligned_elements(ranges, 7);
  ScanArgs p{};
  p.values = values;
  p.gates = gates;
  p.offsets = offsets;
  p.initial = initial;
  p.n = n;
  p.d = d;
  p.b = b;
  p.clear_rest = clear_rest;
  p.carries = carries;
  p.out = out;
  p.final_state = final_state;
  return run_scan<false>(dtype, index_dtype, align, p, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), report);
}

int rg_scan_backward(int dtype, int index_dtype, int64_t d, int64_t n, int64_t b, const void *values,
                     const void *gates, const void *offsets, const float *initial, const float *carries,
                     const void *grad_out, const float *grad_final, void *grad_values, void *grad_gates,
                     float *grad_initial, void *workspace, int64_t workspace_bytes, void *stream,
                     rg_report *report) {
  clear_report(report);
  const bool clear_rest = take_clear_rest(dtype);
  int status = check_shape(dtype, index_dtype, d, n, b);
  if (status) return status;
  if (b == 0) return RG_OK;
  if (grad_initial && !initial) return fail(RG_ERR_INVALID_ARGUMENT, "grad_initial needs initial");
  const int esize = elem_bytes(dtype);
  const int isize = index_dtype == RG_INDEX_I32 ? 4 : 8;
  const int64_t full = n * d * esize, states = b * d * 4;
  const TensorRange ranges[] = {{"values", values, full, esize, false},
                          {"gates", gates, full, esize, false},
                          {"offsets", offsets, (b + 1) * isize, isize, false},
                          {"initial", initial, initial ? states : 0, 4, false},
                          {"carries", carries, ceil_div(n, kScanBatch) * d * 4, 4, false},
                          {"grad_out", grad_out, full, esize, false},
                          {"grad_final", grad_final, grad_final ? states : 0, 4, false},
                          {"grad_values", grad_values, grad_values ? full : 0, esize, true},
                          {"grad_gates", grad_gates, grad_gates ? full : 0, esize, true},
                          {"grad_initial", grad_initial, grad_initial ? states : 0, 4, true}};
  status = check_ranges(ranges, 10);
  if (status) return status;
  const int align = aligned_elements(ranges, 10);
  ScanArgs p{};
  p.values = values;
  p.gates = gates;
  p.offsets = offsets;
  p.initial = initial;
  p.n = n;
  p.d = d;
  p.b = b;
  p.clear_rest = clear_rest;
  p.carries = const_cast<float *>(carries);
  p.grad_out = grad_out;
  p.grad_final = grad_final;
  p.grad_values = grad_values;
  p.grad_gates = grad_gates;
  p.grad_initial = grad_initial;
  return run_scan<true>(dtype, index_dtype, align, p, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), report);
}

}  // extern "C"
