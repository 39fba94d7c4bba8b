// Launch code of the segmented scan (kernels and mathematics: scan.cuh).
#include <cstdio>
#include <cstring>

#include "internal.h"
#include "scan.cuh"

namespace rgb {

namespace {

constexpr int64_t kMaxScanDim = 65536;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

struct ScanShape {
  int vec, shift, tiles, rows;
  int64_t chunks, groups, supers, blocks;
};

// Column vectors of up to 16 bytes that divide D; a tile of at most 128 bytes
// and 32 lanes of them; the rest of the CTA's threads are row groups.
ScanShape make_shape(int dtype, int64_t d, int64_t n, int64_t b, uint32_t flags) {
  const int esize = elem_bytes(dtype);
  ScanShape s;
  s.vec = 1;
  if (!(flags & RG_FLAG_NO_VECTORIZE))
    while (2 * s.vec * esize <= 16 && d % (2 * s.vec) == 0) s.vec *= 2;
  const int64_t cols = d / s.vec;
  s.shift = 0;
  while ((1 << s.shift) < cols && s.shift < 5 && (2 << s.shift) * s.vec * esize <= 128) ++s.shift;
  s.tiles = static_cast<int>(ceil_div(cols, int64_t{1} << s.shift));
  s.rows = (kScanThreads >> s.shift) * scan_rows(esize, s.vec);
  s.chunks = ceil_div(n, s.rows);
  s.groups = ceil_div(s.chunks, kScanFan);
  s.supers = ceil_div(s.groups, kScanFan);
  // Empty segments are shared out over the CTAs; 4096 of them keep one busy.
  s.blocks = s.chunks;
  if (s.blocks < ceil_div(b, 4096)) s.blocks = ceil_div(b, 4096);
  if (s.blocks < 1) s.blocks = 1;
  return s;
}

struct ScanLayout {
  int64_t flags, pairs, supers, bytes, cleared;
};

// Status word at 0, ticket at 8, then flags (cleared before each call), pairs
// and supergroup states.  A single chunk waits for nothing and needs none.
ScanLayout make_layout(const ScanShape &s) {
  ScanLayout l{};
  if (s.chunks <= 1) return l;
  const int64_t slots = static_cast<int64_t>(s.tiles) * 2;
  l.flags = 256;
  l.cleared = align256(l.flags + (s.chunks + s.groups + s.supers) * slots * 4);
  l.pairs = l.cleared;
  l.supers = align256(l.pairs + (s.chunks + s.groups) * s.tiles * kScanCols * 8);
  l.bytes = align256(l.supers + s.supers * s.tiles * kScanCols * 4);
  return l;
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

struct Range {
  const char *name;
  const void *ptr;
  int64_t bytes;
  int align;
  bool written;
};

// Null pointers of tensors with bytes, misaligned ones, and written tensors
// that overlap any other.
int check_ranges(const Range *r, int count) {
  char buffer[200];
  for (int i = 0; i < count; ++i) {
    if (!r[i].bytes) continue;
    if (!r[i].ptr) {
      std::snprintf(buffer, sizeof buffer, "%s pointer is NULL", r[i].name);
      return fail(RG_ERR_INVALID_ARGUMENT, buffer);
    }
    if (!aligned(r[i].ptr, r[i].align)) {
      std::snprintf(buffer, sizeof buffer, "%s must be %d-byte aligned", r[i].name, r[i].align);
      return fail(RG_ERR_INVALID_ARGUMENT, buffer);
    }
  }
  for (int i = 0; i < count; ++i)
    for (int j = 0; j < count; ++j) {
      if (i == j || !r[i].written || !r[i].bytes || !r[j].bytes) continue;
      const uintptr_t a = reinterpret_cast<uintptr_t>(r[i].ptr), b = reinterpret_cast<uintptr_t>(r[j].ptr);
      if (a < b + r[j].bytes && b < a + r[i].bytes) {
        std::snprintf(buffer, sizeof buffer, "%s overlaps %s", r[i].name, r[j].name);
        return fail(RG_ERR_INVALID_ARGUMENT, buffer);
      }
    }
  return RG_OK;
}

template <typename T, typename OffT, int VEC, bool BACKWARD>
int launch(const ScanArgs &p, const ScanShape &s, cudaStream_t stream, rg_report *report) {
  const int smem = 2 * (s.rows + 1) * 4;
  const dim3 grid(static_cast<unsigned>(s.blocks * s.tiles), 1, 1);
  scan_kernel<T, OffT, VEC, BACKWARD><<<grid, kScanThreads, smem, stream>>>(p);
  record_launch(report, BACKWARD ? K_SCAN_BACKWARD : K_SCAN, grid, kScanThreads, smem);
  return check_cuda(cudaGetLastError(), "scan_kernel launch");
}

template <typename OffT, bool BACKWARD>
int launch_vec(int dtype, const ScanArgs &p, const ScanShape &s, cudaStream_t stream, rg_report *report) {
  if (dtype == RG_DTYPE_F32) {
    if (s.vec == 4) return launch<float, OffT, 4, BACKWARD>(p, s, stream, report);
    if (s.vec == 2) return launch<float, OffT, 2, BACKWARD>(p, s, stream, report);
    return launch<float, OffT, 1, BACKWARD>(p, s, stream, report);
  }
  if (s.vec == 8) return launch<__nv_bfloat16, OffT, 8, BACKWARD>(p, s, stream, report);
  if (s.vec == 4) return launch<__nv_bfloat16, OffT, 4, BACKWARD>(p, s, stream, report);
  if (s.vec == 2) return launch<__nv_bfloat16, OffT, 2, BACKWARD>(p, s, stream, report);
  return launch<__nv_bfloat16, OffT, 1, BACKWARD>(p, s, stream, report);
}

template <bool BACKWARD>
int run_scan(int dtype, int index_dtype, const ScanShape &s, ScanArgs &p, void *workspace, int64_t workspace_bytes,
             cudaStream_t stream, rg_report *report) {
  DeviceProps dev;
  int status = check_device(&dev);
  if (status) return status;
  if (s.blocks > 2147483647LL / s.tiles) return fail(RG_ERR_INVALID_ARGUMENT, "the call needs more than 2^31 - 1 CTAs");
  const ScanLayout l = make_layout(s);
  if (report) {
    report->workspace_bytes = l.bytes;
    report->d_vector = s.vec;
    report->d_tile = 1 << s.shift;
    report->status_offset = l.bytes ? 0 : -1;
  }
  p.shift = s.shift;
  p.vec_cols = static_cast<int>(p.d / s.vec);
  p.tiles = s.tiles;
  p.chunks = s.chunks;
  p.blocks = s.blocks;
  if (l.bytes) {
    if (!workspace || workspace_bytes < l.bytes) return fail(RG_ERR_WORKSPACE, "workspace missing or too small");
    if (!aligned(workspace, 256)) return fail(RG_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    char *base = static_cast<char *>(workspace);
    p.status = reinterpret_cast<unsigned long long *>(base);
    p.ticket = reinterpret_cast<unsigned *>(base + 8);
    p.flags = reinterpret_cast<unsigned *>(base + l.flags);
    p.pairs = reinterpret_cast<float2 *>(base + l.pairs);
    p.supers = reinterpret_cast<float *>(base + l.supers);
    status = check_cuda(cudaMemsetAsync(base, 0, l.cleared, stream), "cudaMemsetAsync");
    if (status) return status;
    if (report) ++report->memsets;
  }
  if (index_dtype == RG_INDEX_I32) return launch_vec<int32_t, BACKWARD>(dtype, p, s, stream, report);
  return launch_vec<int64_t, BACKWARD>(dtype, p, s, stream, report);
}

void clear_report(rg_report *report) {
  if (!report) return;
  std::memset(report, 0, sizeof *report);
  report->status_offset = -1;
  report->streams = 1;
}

}  // namespace

}  // namespace rgb

using namespace rgb;

extern "C" {

int rg_scan_workspace_bytes(int dtype, int index_dtype, int64_t d, int64_t n, int64_t b, uint32_t flags,
                            int64_t *bytes, int64_t *carry_rows) {
  if (!bytes || !carry_rows) return fail(RG_ERR_INVALID_ARGUMENT, "bytes and carry_rows must not be NULL");
  const int status = check_shape(dtype, index_dtype, d, n, b);
  if (status) return status;
  const ScanShape s = make_shape(dtype, d, n, b, flags);
  *bytes = make_layout(s).bytes;
  *carry_rows = s.chunks;
  return RG_OK;
}

int rg_scan(int dtype, int index_dtype, int64_t d, int64_t n, int64_t b, const void *values, const void *gates,
            const void *offsets, const float *initial, void *out, float *final_state, float *carries, void *workspace,
            int64_t workspace_bytes, uint32_t flags, void *stream, rg_report *report) {
  clear_report(report);
  int status = check_shape(dtype, index_dtype, d, n, b);
  if (status) return status;
  if (b == 0) return RG_OK;
  const ScanShape s = make_shape(dtype, d, n, b, flags);
  const int esize = elem_bytes(dtype), vec = s.vec * esize, state = (s.vec < 4 ? s.vec : 4) * 4;
  const int isize = index_dtype == RG_INDEX_I32 ? 4 : 8;
  const int64_t full = n * d * esize, states = b * d * 4;
  const Range ranges[] = {{"values", values, full, vec, false},
                          {"gates", gates, full, vec, false},
                          {"offsets", offsets, (b + 1) * isize, isize, false},
                          {"initial", initial, initial ? states : 0, state, false},
                          {"out", out, full, vec, true},
                          {"final", final_state, final_state ? states : 0, state, true},
                          {"carries", carries, carries ? s.chunks * d * 4 : 0, 4, true}};
  status = check_ranges(ranges, 7);
  if (status) return status;
  ScanArgs p{};
  p.values = values;
  p.gates = gates;
  p.offsets = offsets;
  p.initial = initial;
  p.n = n;
  p.d = d;
  p.b = b;
  p.carries = carries;
  p.out = out;
  p.final_state = final_state;
  return run_scan<false>(dtype, index_dtype, s, p, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), report);
}

int rg_scan_backward(int dtype, int index_dtype, int64_t d, int64_t n, int64_t b, const void *values,
                     const void *gates, const void *offsets, const float *initial, const float *carries,
                     const void *grad_out, const float *grad_final, void *grad_values, void *grad_gates,
                     float *grad_initial, void *workspace, int64_t workspace_bytes, uint32_t flags, void *stream,
                     rg_report *report) {
  clear_report(report);
  int status = check_shape(dtype, index_dtype, d, n, b);
  if (status) return status;
  if (b == 0) return RG_OK;
  if (grad_initial && !initial) return fail(RG_ERR_INVALID_ARGUMENT, "grad_initial needs initial");
  const ScanShape s = make_shape(dtype, d, n, b, flags);
  const int esize = elem_bytes(dtype), vec = s.vec * esize, state = (s.vec < 4 ? s.vec : 4) * 4;
  const int isize = index_dtype == RG_INDEX_I32 ? 4 : 8;
  const int64_t full = n * d * esize, states = b * d * 4;
  const Range ranges[] = {{"values", values, full, vec, false},
                          {"gates", gates, full, vec, false},
                          {"offsets", offsets, (b + 1) * isize, isize, false},
                          {"initial", initial, initial ? states : 0, state, false},
                          {"carries", carries, s.chunks * d * 4, 4, false},
                          {"grad_out", grad_out, full, vec, false},
                          {"grad_final", grad_final, grad_final ? states : 0, state, false},
                          {"grad_values", grad_values, grad_values ? full : 0, vec, true},
                          {"grad_gates", grad_gates, grad_gates ? full : 0, vec, true},
                          {"grad_initial", grad_initial, grad_initial ? states : 0, state, true}};
  status = check_ranges(ranges, 10);
  if (status) return status;
  ScanArgs p{};
  p.values = values;
  p.gates = gates;
  p.offsets = offsets;
  p.initial = initial;
  p.n = n;
  p.d = d;
  p.b = b;
  p.carries = const_cast<float *>(carries);
  p.grad_out = grad_out;
  p.grad_final = grad_final;
  p.grad_values = grad_values;
  p.grad_gates = grad_gates;
  p.grad_initial = grad_initial;
  return run_scan<true>(dtype, index_dtype, s, p, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), report);
}

}  // extern "C"
