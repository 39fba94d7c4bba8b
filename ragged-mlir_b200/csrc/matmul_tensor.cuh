// Segmented matrix products of bf16 tensors on the 5th-generation tensor cores.
//
// A persistent CTA computes 128 x COLS tiles of the output.  One warp brings
// slices of 64 of the contraction into a ring of shared-memory stages by TMA
// (128-byte swizzle), one warp issues tcgen05.mma on them into one of two
// accumulators in tensor memory, and four warps empty the other one: round to
// bf16 once, turn 32 x 64 blocks through shared memory, store whole 128-byte
// lines.  Loads, products and stores of neighbouring tiles overlap.
//
// Operands are read as they lie in memory, K-major or MN-major by descriptor:
//   kind      left                          right
//   forward   values: K-major               weights[s]: MN-major
//   values    grad_out: K-major             weights[s]: K-major
//   weights   values_s: MN-major            grad_out_s: MN-major
// Columns past a width are zero (TMA's fill, in both operands).  Rows of the
// next segment that a tile of rows reaches into only make rows of the
// accumulator that are not stored, and boxes of 32 rows without a row of the
// segment are not loaded: a segment of few rows costs its weights and little
// more.  In the weights kind a slice of the contraction can reach into the
// next segment: its rows there are set to zero in both operands (in the last
// slice of a segment, up to the next multiple of the instruction's 16).
//
// Sums are f32 in tensor memory.  Every wait is bounded; one that gives up
// sets the call's status word, and all roles leave.
//
// With some hundred rows a segment neither device memory nor the tensor cores are at
// their limit (16384 rows x 1024 x 1024 in 64 segments of unlike lengths: 48 us, 53 %
// of the tensor cores' cycles, a quarter of them for rows past a segment's end, 48 %
// of the memory's); with few rows each CTA's way to its first tile, along the offsets,
// counts (8192 rows x 1024 x 64 in 256 segments: 13 us, 17 with cold inputs, where
// the bytes take 8); in large products the operands
// that L2 delivers to an SM, which pairs of SMs halve (matmul_pair.cuh).
#pragma once

#include <cuda.h>

#include "matmul.cuh"

namespace rgb {

constexpr int kTensorThreads = 192;  // warps: copies, products, 4 x stores
constexpr int kStoreThreads = 128;
constexpr int kTensorRows = 128;
constexpr int kTensorDepth = 64;     // of a stage: 128 bytes of bf16
constexpr int kLeftBytes = kTensorRows * 128;
constexpr int kStoreBytes = 4 * 32 * 128;

constexpr int tensor_stages(int cols) { return cols == 256 ? 4 : cols == 128 ? 6 : 3; }
// Narrow tiles are small work each: two CTAs an SM overlap their starts and ends.
constexpr int tensor_ctas(int cols) { return cols == 64 ? 2 : 1; }
constexpr int tensor_smem_bytes(int cols) { return tensor_stages(cols) * (kLeftBytes + cols * 128) + kStoreBytes + 1024; }

struct TensorMaps {
  CUtensorMap left, left_part, right;  // left_part: boxes of 32 rows
  // MN-major operands whose width is a multiple of 64 are mapped with their
  // slabs of 64 as a dimension of their own, and a tile's slabs come in one box.
  int left_slabs, right_slabs;
};

__device__ __forceinline__ void tma_load_3d(void *smem_dst, const void *map, int x, int y, int z, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n" ::"r"(
          smem_u32(smem_dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ void tma_load_4d(void *smem_dst, const void *map, int x, int y, int z, int w, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n" ::"r"(
          smem_u32(smem_dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Orders ordinary writes to global memory before copies by TMA that read them.
__device__ __forceinline__ void fence_proxy_async_global() { asm volatile("fence.proxy.async.global;\n" ::: "memory"); }

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}

// Shared-memory operand with 128-byte swizzle.  K-major: rows of 128 bytes,
// groups of 8 rows 1024 bytes apart.  MN-major: slabs of 64 elements, each a
// row of 128 bytes per step of the contraction; `lead` bytes from slab to slab,
// groups of 8 steps 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_operand(uint32_t smem, uint32_t lead) {
  return (uint64_t{2} << 61) | (uint64_t{1} << 46) | (uint64_t{1024 >> 4} << 32) |
         (static_cast<uint64_t>(lead >> 4) << 16) | ((smem >> 4) & 0x3fff);
}

// kind::f16: f32 accumulator, bf16 operands.
__device__ __forceinline__ uint32_t umma_instruction(int rows, int cols, bool left_mn, bool right_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(left_mn) << 15) |
         (static_cast<uint32_t>(right_mn) << 16) | (static_cast<uint32_t>(cols >> 3) << 17) |
         (static_cast<uint32_t>(rows >> 4) << 24);
}

__device__ __forceinline__ void umma(uint32_t acc, uint64_t left, uint64_t right, uint32_t instruction, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(acc),
      "l"(left), "l"(right), "r"(instruction), "r"(static_cast<uint32_t>(add))
      : "memory");
}

// Likewise on a pair of SMs (matmul_pair.cuh).
__device__ __forceinline__ void umma_pair(uint32_t acc, uint64_t left, uint64_t right, uint32_t instruction, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(acc),
      "l"(left), "l"(right), "r"(instruction), "r"(static_cast<uint32_t>(add))
      : "memory");
}

// Arrives on `bar` when the products issued so far are done.
__device__ __forceinline__ void umma_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void tmem_load_32(uint32_t at, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at));
}

// True in one lane of a converged warp, the same one each time.  Roles run their
// inner loops in that lane alone: products that the compiler knows to come from
// one thread are issued back to back, a branch on the lane's number costs a
// hundred clocks around each.
__device__ __forceinline__ bool elect_lane() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// Place in the ring of stages.
template <int STAGES>
struct RingPlace {
  int stage;
  uint32_t phase;
  __device__ __forceinline__ void next() {
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1;
    }
  }
  __device__ __forceinline__ void skip(uint32_t count) {
    const uint32_t at = stage + count;
    phase ^= at / STAGES & 1;
    stage = static_cast<int>(at % STAGES);
  }
};

// The products of a stage, `steps` times 16 of the contraction: 32 bytes along a
// K-major row, 16 rows of an MN-major slab.
template <bool PAIR, bool LEFT_MN, bool RIGHT_MN>
__device__ __forceinline__ void umma_stage(uint32_t to, uint32_t left, uint32_t right, uint32_t slab,
                                           uint32_t instruction, bool add, int steps) {
  const uint64_t a = umma_operand(left, LEFT_MN ? slab : 16), b = umma_operand(right, RIGHT_MN ? slab : 16);
#pragma unroll
  for (int i = 0; i < kTensorDepth / 16; ++i) {
    if (i < steps) {
      const uint64_t ai = a + i * (LEFT_MN ? 2048 >> 4 : 32 >> 4), bi = b + i * (RIGHT_MN ? 2048 >> 4 : 32 >> 4);
      if constexpr (PAIR)
        umma_pair(to, ai, bi, instruction, add || i > 0);
      else
        umma(to, ai, bi, instruction, add || i > 0);
    }
  }
}

// Bounded wait by a role; on giving up marks the CTA so that all roles leave.
// `status` is the CTA's own word.  `slices`: what the wait may have to see
// through, where that has no bound of its own.
struct TensorGate {
  volatile int *abandoned;
  unsigned long long *status;
  __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, int64_t slices = 0) const {
    for (int64_t left = kMbarWaitLimit * (1 + (slices >> 14)); left > 0; --left) {
      if (mbar_try_wait(bar, parity)) return true;
      if (*abandoned) return false;
    }
    *abandoned = 1;
    *status = 1;
    return false;
  }
  // By all lanes of a warp, which go on, or give up, as one: what comes next
  // (votes, tensor-memory loads) needs all of them.
  __device__ __forceinline__ bool wait_together(uint64_t *bar, uint32_t parity, int64_t slices = 0) const {
    return __all_sync(~0u, wait(bar, parity, slices)) != 0;
  }
};

// Empties a warp's 32 rows (`quarter`: of the accumulator's 128, those this warp
// can read) of a tile of COLS columns: rounds to bf16, turns 32 x 64 blocks
// through shared memory, stores whole 128-byte lines.
template <int KIND, int COLS>
struct TensorStore {
  const MatmulArgs &p;
  unsigned char *turn;
  int quarter;
  __nv_bfloat16 *out;
  bool whole;  // rows start at 16-byte boundaries
  __device__ __forceinline__ TensorStore(const MatmulArgs &args, unsigned char *smem, int q)
      : p(args), turn(smem + q * 32 * 128), quarter(q), out(static_cast<__nv_bfloat16 *>(args.out)) {
    whole = p.out_pitch % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  }
  // The accumulator's rows are the output's from `first` on, up to the tile's end.
  __device__ __forceinline__ void tile(const MatmulTile &t, int64_t first, bool nothing, uint32_t acc) const {
    const int lane = threadIdx.x & 31;
    const int64_t row0 = first + quarter * 32;
    const int rows = static_cast<int>(min(max(t.row_end - row0, int64_t{0}), int64_t{32}));
    __nv_bfloat16 *to = out + (KIND == MATMUL_GRAD_WEIGHTS ? t.seg * p.rows + row0 : row0) * p.out_pitch;
#pragma unroll 1
    for (int c = 0; c < COLS; c += 64) {
      const int64_t col0 = static_cast<int64_t>(t.col_tile) * COLS + c;
      if (col0 >= p.cols) break;
      uint32_t v[2][32];
      if (nothing) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[0][i] = v[1][i] = 0;
      } else {
        const uint32_t at = acc + c + (static_cast<uint32_t>(quarter * 32) << 16);
        tmem_load_32(at, v[0]);
        tmem_load_32(at + 32, v[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
      }
      if constexpr (KIND == MATMUL_GRAD_WEIGHTS) {
        if (p.parts) {  // a part's sum, f32: a row a lane (few and small tiles alone are split)
          float *row = p.parts + ((t.split * p.b + t.seg) * p.rows + row0 + lane) * p.cols;
          if (lane < rows && p.cols % 4 == 0) {
#pragma unroll
            for (int i = 0; i < 64; i += 4) {
              const uint32_t *x = &v[i / 32][i % 32];
              if (col0 + i < p.cols) *reinterpret_cast<uint4 *>(row + col0 + i) = uint4{x[0], x[1], x[2], x[3]};
            }
          } else if (lane < rows) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (col0 + i < p.cols) row[col0 + i] = __uint_as_float(v[i / 32][i % 32]);
          }
          __syncwarp();  // the next load of tensor memory is one of all lanes
          continue;
        }
      }
      // Row `lane`, 8 pieces of 16 bytes, permuted so that neither this nor
      // the reading across rows meets a bank twice.
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t *x = &v[i / 4][i % 4 * 8];
        uint4 piece;
        piece.x = pack_bf16x2(__uint_as_float(x[0]), __uint_as_float(x[1]));
        piece.y = pack_bf16x2(__uint_as_float(x[2]), __uint_as_float(x[3]));
        piece.z = pack_bf16x2(__uint_as_float(x[4]), __uint_as_float(x[5]));
        piece.w = pack_bf16x2(__uint_as_float(x[6]), __uint_as_float(x[7]));
        *reinterpret_cast<uint4 *>(turn + lane * 128 + ((i ^ (lane & 7)) * 16)) = piece;
      }
      __syncwarp();
      if (whole) {
        const int piece = lane & 7;
        const bool col_ok = col0 + piece * 8 < p.cols;  // widths are multiples of 8 here
#pragma unroll
        for (int r = 0; r < 32; r += 4) {
          const int row = r + lane / 8;
          const uint4 x = *reinterpret_cast<const uint4 *>(turn + row * 128 + ((piece ^ (row & 7)) * 16));
          if (row < rows && col_ok) *reinterpret_cast<uint4 *>(to + row * p.out_pitch + col0 + piece * 8) = x;
        }
      } else {
#pragma unroll 4
        for (int row = 0; row < rows; ++row) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int col = half * 32 + lane;
            const __nv_bfloat16 x = *reinterpret_cast<const __nv_bfloat16 *>(
                turn + row * 128 + (((col / 8) ^ (row & 7)) * 16) + col % 8 * 2);
            if (col0 + col < p.cols) to[row * p.out_pitch + col0 + col] = x;
          }
        }
      }
      __syncwarp();
    }
  }
};

template <typename OffT, int KIND, int COLS>
__global__ void __launch_bounds__(kTensorThreads, tensor_ctas(COLS))
matmul_tensor_kernel(const MatmulArgs p, const __grid_constant__ TensorMaps maps) {
  constexpr int STAGES = tensor_stages(COLS);
  constexpr int DEPTH = kTensorDepth, ROWS = kTensorRows;
  constexpr int kRight = COLS * 128, kStage = kLeftBytes + kRight;
  constexpr bool LEFT_MN = KIND == MATMUL_GRAD_WEIGHTS, RIGHT_MN = KIND != MATMUL_GRAD_VALUES;
  constexpr uint32_t kSlab = DEPTH * 128;  // bytes of an MN-major slab of 64 elements
  __shared__ uint64_t full[STAGES], empty[STAGES], ready[2], drained[2], settled;
  __shared__ uint32_t tmem_base;
  __shared__ int abandoned;
  extern __shared__ unsigned char tensor_smem_raw[];
  unsigned char *smem = tensor_smem_raw + ((1024 - (smem_u32(tensor_smem_raw) & 1023)) & 1023);
  unsigned char *store_smem = smem + STAGES * kStage;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ready[i], 1);
      mbar_init(&drained[i], 4);
    }
    mbar_init(&settled, 1);
    abandoned = 0;
    p.status[blockIdx.x] = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_base)),
                 "n"(2 * COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tmem = tmem_base;
  const TensorGate gate{&abandoned, p.status + blockIdx.x};
  // (One load by a warp that has just met in __syncwarp: the same for all lanes.  A
  // vote on it takes 2 us more at 32768 rows x 1024 x 2048.)
  auto abandoned_now = [&]() { return *gate.abandoned != 0; };

  MatmulWalk<OffT, KIND, ROWS> walk(p.offsets, p.b);
  MatmulTile t;
  auto slices = [&](const MatmulTile &tile) {
    const int64_t depth = KIND == MATMUL_GRAD_WEIGHTS ? tile.end - tile.begin : p.depth;
    return (depth + DEPTH - 1) / DEPTH;
  };

  // On operands that are being packed, all roles: the waits below are bounded,
  // and a pack launch may take longer than that.
  grid_dependency_wait();
  if (warp == 0) {
    // ------------------------------------------------------------ copies --
    fence_proxy_async_global();  // (operands that a launch has packed)
    RingPlace<STAGES> at{0, 1};
    bool going = true;
    for (int64_t index = blockIdx.x; going && walk.find(p, index, t); index += gridDim.x) {
      const int count = static_cast<int>(slices(t));
      const int col0 = t.col_tile * COLS;
      const int boxes = LEFT_MN ? 2 : static_cast<int>((t.row_end - t.row + 31) / 32);
      const uint32_t bytes = (LEFT_MN ? kLeftBytes : boxes * 32 * 128) + kRight;
      if (elect_lane()) {
        RingPlace<STAGES> here = at;
        for (int k = 0; k < count; ++k, here.next()) {
          const int stage = here.stage;
          if (!gate.wait(&empty[stage], here.phase)) break;
          unsigned char *left = smem + stage * kStage, *right = left + kLeftBytes;
          mbar_expect_tx(&full[stage], bytes);
          const int d0 = k * DEPTH;
          if constexpr (LEFT_MN) {
            const int row = static_cast<int>(t.begin) + d0;
            if (maps.left_slabs) {
              tma_load_3d(left, &maps.left, 0, row, static_cast<int>(t.row) / 64, &full[stage]);
            } else {
              for (int i = 0; i < ROWS / 64; ++i)
                tma_load_2d(left + i * kSlab, &maps.left, static_cast<int>(t.row) + i * 64, row, &full[stage]);
            }
            if (maps.right_slabs) {
              tma_load_3d(right, &maps.right, 0, row, col0 / 64, &full[stage]);
            } else {
              for (int i = 0; i < COLS / 64; ++i)
                tma_load_2d(right + i * kSlab, &maps.right, col0 + i * 64, row, &full[stage]);
            }
          } else {
            if (boxes == 4) {
              tma_load_2d(left, &maps.left, d0, static_cast<int>(t.row), &full[stage]);
            } else {
              for (int i = 0; i < boxes; ++i)
                tma_load_2d(left + i * 32 * 128, &maps.left_part, d0, static_cast<int>(t.row) + i * 32, &full[stage]);
            }
            if constexpr (RIGHT_MN) {
              if (maps.right_slabs) {
                tma_load_4d(right, &maps.right, 0, d0, col0 / 64, static_cast<int>(t.seg), &full[stage]);
              } else {
                for (int i = 0; i < COLS / 64; ++i)
                  tma_load_3d(right + i * kSlab, &maps.right, col0 + i * 64, d0, static_cast<int>(t.seg), &full[stage]);
              }
            } else {
              tma_load_3d(right, &maps.right, d0, col0, static_cast<int>(t.seg), &full[stage]);
            }
          }
        }
      }
      __syncwarp();
      at.skip(static_cast<uint32_t>(count));
      going = !abandoned_now();
    }
    // Given up: copies in flight write this CTA's shared memory, so they get
    // a millisecond to end before it does.
    if (!going)
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  } else if (warp == 1) {
    // ---------------------------------------------------------- products --
    const uint32_t instruction = umma_instruction(ROWS, COLS, LEFT_MN, RIGHT_MN);
    RingPlace<STAGES> at{0, 0};
    int acc = 0;
    uint32_t acc_phase = 1;
    bool going = true;
    for (int64_t index = blockIdx.x; going && walk.find(p, index, t); index += gridDim.x) {
      const int count = static_cast<int>(slices(t));
      if (count == 0) continue;  // (weights kind: the stores write zeros)
      // Slices that are whole; in the weights kind the last one may not be.
      const int whole = KIND == MATMUL_GRAD_WEIGHTS ? static_cast<int>((t.end - t.begin) / DEPTH) : count;
      const uint32_t to = tmem + acc * COLS;
      if (elect_lane()) {
        bool there = gate.wait(&drained[acc], acc_phase);
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        RingPlace<STAGES> here = at;
        for (int k = 0; there && k < whole; ++k, here.next()) {
          there = gate.wait(&full[here.stage], here.phase);
          if (!there) break;
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          const uint32_t left = smem_u32(smem + here.stage * kStage);
          umma_stage<false, LEFT_MN, RIGHT_MN>(to, left, left + kLeftBytes, kSlab, instruction, k > 0, DEPTH / 16);
          umma_commit(&empty[here.stage]);
        }
        if (there && whole == count) umma_commit(&ready[acc]);
      }
      __syncwarp();
      at.skip(static_cast<uint32_t>(whole));
      going = !abandoned_now();
      if (KIND == MATMUL_GRAD_WEIGHTS && going && whole < count) {
        going = gate.wait_together(&full[at.stage], at.phase);
        if (!going) break;
        unsigned char *left = smem + at.stage * kStage, *right = left + kLeftBytes;
        const int from = static_cast<int>(t.end - t.begin - int64_t{whole} * DEPTH), steps = (from + 15) / 16;
        const int rows = steps * 16 - from;
        for (int i = lane; i < rows * 8 * (2 + COLS / 64); i += 32) {
          const int slab = i / (rows * 8), row = from + i / 8 % rows;
          *reinterpret_cast<uint4 *>((slab < 2 ? left + slab * kSlab : right + (slab - 2) * kSlab) + row * 128 +
                                     i % 8 * 16) = uint4{0, 0, 0, 0};
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (elect_lane()) {
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          umma_stage<false, LEFT_MN, RIGHT_MN>(to, smem_u32(left), smem_u32(right), kSlab, instruction, whole > 0, steps);
          umma_commit(&empty[at.stage]);
          umma_commit(&ready[acc]);
        }
        __syncwarp();
        at.next();
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (!going) {  // given up: the products in flight end before tensor memory is freed
      if (elect_lane()) umma_commit(&settled);
      __syncwarp();
      mbar_wait(&settled, 0);
    }
  } else {
    // ------------------------------------------------------------ stores --
    TensorStore<KIND, COLS> store(p, store_smem, warp & 3);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool going = true;
    for (int64_t index = blockIdx.x; going && walk.find(p, index, t); index += gridDim.x) {
      const bool nothing = KIND == MATMUL_GRAD_WEIGHTS && t.end == t.begin;
      if (!nothing) {
        going = gate.wait_together(&ready[acc], acc_phase, slices(t));
        if (!going) break;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      }
      store.tile(t, t.row, nothing, tmem + acc * COLS);
      if (!nothing) {
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        if (lane == 0) mbar_arrive(&drained[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
    if constexpr (KIND != MATMUL_GRAD_WEIGHTS)
      matmul_clear_rest<__nv_bfloat16, OffT>(
          p, int64_t{blockIdx.x} * kStoreThreads + threadIdx.x - (kTensorThreads - kStoreThreads),
          int64_t{gridDim.x} * kStoreThreads);
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "n"(2 * COLS) : "memory");
}

// Rows of `cols` elements, `pitch` apart in `to`: for widths or addresses that
// TMA does not take (its rows start at 16-byte boundaries).  The elements past
// `cols` are never read.
struct PackArgs {
  const __nv_bfloat16 *from;  // null: nothing
  __nv_bfloat16 *to;
  int64_t rows, cols, pitch;
};

// One launch for both operands, all weights among them, 16 loads a lane at once; the
// product's launch may start before it ends.  (5003 rows x 501 x 333 in 12 segments:
// 17 us a call in a replayed graph, 18 with cold inputs, 19 with a launch each; 16001
// rows x 1001 x 777 87 and 93.)
__global__ void __launch_bounds__(256) matmul_pack_kernel(const PackArgs left, const PackArgs right) {
  grid_dependents_launch();
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 8;
  const int64_t total = left.rows + right.rows;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32; i < total; i += stride) {
    const bool second = i >= left.rows;
    const PackArgs &p = second ? right : left;
    const int64_t r = second ? i - left.rows : i;
    const __nv_bfloat16 *from = p.from + r * p.cols;
    __nv_bfloat16 *to = p.to + r * p.pitch;
    for (int64_t c0 = threadIdx.x % 32; c0 < p.cols; c0 += 512) {
      __nv_bfloat16 x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c0 + j * 32 < p.cols) x[j] = from[c0 + j * 32];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c0 + j * 32 < p.cols) to[c0 + j * 32] = x[j];
    }
  }
  fence_proxy_async_global();
}

}  // namespace rgb
