// Large segmented matrix products of bf16 tensors: tiles of 256 x 256 on pairs
// of SMs.
//
// A 128 x 256 tile of one SM takes in 48 KB of operands for each 64 of the
// contraction, 768 clocks of the 64 bytes a clock that L2 delivers to an SM,
// and computes on them for 512.  A cluster of two CTAs computes 256 x 256
// instead (tcgen05 with cta_group::2): each loads its 128 rows of the left
// operand and its 128 columns of the right one, 32 KB, and tensor cores read
// the other SM's half from there.  Roles are those of the tile of one SM
// (matmul_tensor.cuh): copies and stores in both CTAs, each for itself, but all
// copies of a stage are counted on the first CTA's barrier, and the first CTA
// issues the products.  Where a slice reaches past a segment's end (weights
// kind, a segment's last slice), each CTA has its own copies counted on its own
// barrier and clears its rows, and the second one says so by a remote arrival.
//
// 65536 rows x 2048 x 2048 in 16 segments: 357 to 365 us forward, 353 to 363 and 358
// to 375 for the gradients of values and weights on several GPUs (single calls; 1.5
// PFLOP/s, 0.92 of a library's dense product; 390 in a row, under the power limit);
// on tiles of one SM 379, 385 and 404.  Bound: the tensor cores (74 %
// busy at 16384 x 1024 x 2048, where the first and last tiles weigh more).  Copies
// of a stage counted by relayed arrivals instead of on the first CTA's barrier
// took 965 us; products issued behind a branch on the lane 430.
#pragma once

#include "matmul_tensor.cuh"

namespace rgb {

constexpr int kPairStages = 6;
constexpr int kPairRows = 256, kPairCols = 256;
constexpr int kPairHalf = 128 * 128;  // bytes of a CTA's half of an operand's stage
constexpr int kPairSmem = kPairStages * 2 * kPairHalf + kStoreBytes + 1024;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// Arrives on the first CTA's barrier at this place.
__device__ __forceinline__ void mbar_arrive_first(uint64_t *bar) {
  asm volatile(
      "{\n .reg .b32 at;\n mapa.shared::cluster.u32 at, %0, 0;\n"
      " mbarrier.arrive.release.cluster.shared::cluster.b64 _, [at];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}
// A box into this CTA's shared memory, counted on a barrier of the first CTA
// (`bar`: its address in the cluster).
__device__ __forceinline__ void pair_load_2d(void *smem_dst, const void *map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n" ::"r"(
          smem_u32(smem_dst)),
      "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void pair_load_3d(void *smem_dst, const void *map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];\n" ::"r"(smem_u32(smem_dst)),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void pair_load_4d(void *smem_dst, const void *map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, "
      "%6}], [%2];\n" ::"r"(smem_u32(smem_dst)),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// Address in the cluster of a barrier of CTA `rank`.
__device__ __forceinline__ uint32_t cluster_address(uint64_t *bar, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_u32(bar)), "r"(rank));
  return at;
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t *bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
// Arrives on the barrier of both CTAs when the products issued so far are done.
__device__ __forceinline__ void umma_pair_commit(uint64_t *bar) {
  asm volatile(
      "{\n .reg .b16 both;\n mov.b16 both, 3;\n"
      " tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n}\n" ::"r"(
          smem_u32(bar))
      : "memory");
}

template <typename OffT, int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTensorThreads, 1)
matmul_pair_kernel(const MatmulArgs p, const __grid_constant__ TensorMaps maps) {
  constexpr int STAGES = kPairStages, DEPTH = kTensorDepth, COLS = kPairCols;
  constexpr int kStage = 2 * kPairHalf;
  constexpr bool LEFT_MN = KIND == MATMUL_GRAD_WEIGHTS, RIGHT_MN = KIND != MATMUL_GRAD_VALUES;
  constexpr uint32_t kSlab = DEPTH * 128;
  // `full`, `theirs` and `drained` are used in the first CTA, `tail` in the second.
  __shared__ uint64_t full[STAGES], tail[STAGES], theirs[STAGES], empty[STAGES], ready[2], drained[2], settled;
  __shared__ uint32_t tmem_base;
  __shared__ int abandoned;
  extern __shared__ unsigned char pair_smem_raw[];
  unsigned char *smem = pair_smem_raw + ((1024 - (smem_u32(pair_smem_raw) & 1023)) & 1023);
  unsigned char *store_smem = smem + STAGES * kStage;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&tail[i], 1);
      mbar_init(&theirs[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ready[i], 1);
      mbar_init(&drained[i], 8);
    }
    mbar_init(&settled, 1);
    abandoned = 0;
    p.status[blockIdx.x] = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_base)),
                 "n"(2 * COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are there
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tmem = tmem_base;
  const TensorGate gate{&abandoned, p.status + blockIdx.x};
  // (One load by a warp that has just met in __syncwarp: the same for all lanes.  A
  // vote on it takes 2 us more at 32768 rows x 1024 x 2048.)
  auto abandoned_now = [&]() { return *gate.abandoned != 0; };

  MatmulWalk<OffT, KIND, kPairRows> walk(p.offsets, p.b);
  MatmulTile t;
  const int64_t first = blockIdx.x / 2, stride = gridDim.x / 2;
  auto slices = [&](const MatmulTile &tile) {
    const int64_t depth = KIND == MATMUL_GRAD_WEIGHTS ? tile.end - tile.begin : p.depth;
    return (depth + DEPTH - 1) / DEPTH;
  };

  // Whether slice k reaches past the segment's end.
  auto is_tail = [&](const MatmulTile &tile, int k) {
    return KIND == MATMUL_GRAD_WEIGHTS && tile.end - tile.begin - int64_t{k} * DEPTH < DEPTH;
  };

  // On operands that are being packed, all roles: the waits below are bounded,
  // and a pack launch may take longer than that.
  grid_dependency_wait();
  if (warp == 0) {
    // ------------------------------------------------------------ copies --
    fence_proxy_async_global();  // (operands that a launch has packed)
    RingPlace<STAGES> at{0, 1};
    bool going = true;
    for (int64_t index = first; going && walk.find(p, index, t); index += stride) {
      const int count = static_cast<int>(slices(t));
      const int row0 = static_cast<int>(t.row) + rank * 128, col0 = t.col_tile * COLS + rank * 128;
      auto boxes_of = [&](int r) {  // of 32 rows, of CTA r
        return static_cast<int>((min(max(t.row_end - t.row - r * 128, int64_t{0}), int64_t{128}) + 31) / 32);
      };
      const int boxes = LEFT_MN ? 0 : boxes_of(rank);
      const uint32_t both = (LEFT_MN ? 2 * kPairHalf : (boxes_of(0) + boxes_of(1)) * 32 * 128) + 2 * kPairHalf;
      if (elect_lane()) {
        RingPlace<STAGES> here = at;
        for (int k = 0; k < count; ++k, here.next()) {
          const int stage = here.stage;
          if (!gate.wait(&empty[stage], here.phase)) break;
          unsigned char *left = smem + stage * kStage, *right = left + kPairHalf;
          const int d0 = k * DEPTH;
          const bool alone = is_tail(t, k);
          uint64_t *own = rank == 0 ? &full[stage] : &tail[stage];
          if (alone)
            mbar_expect_tx(own, 2 * kPairHalf);
          else if (rank == 0)
            mbar_expect_tx(own, both);
          const uint32_t bar = alone ? cluster_address(own, rank) : cluster_address(&full[stage], 0);
          if constexpr (LEFT_MN) {
            const int row = static_cast<int>(t.begin) + d0;
            if (maps.left_slabs) {
              pair_load_3d(left, &maps.left, 0, row, row0 / 64, bar);
            } else {
              for (int i = 0; i < 2; ++i) pair_load_2d(left + i * kSlab, &maps.left, row0 + i * 64, row, bar);
            }
            if (maps.right_slabs) {
              pair_load_3d(right, &maps.right, 0, row, col0 / 64, bar);
            } else {
              for (int i = 0; i < 2; ++i) pair_load_2d(right + i * kSlab, &maps.right, col0 + i * 64, row, bar);
            }
          } else {
            if (boxes == 4) {
              pair_load_2d(left, &maps.left, d0, row0, bar);
            } else {
              for (int i = 0; i < boxes; ++i) pair_load_2d(left + i * 32 * 128, &maps.left_part, d0, row0 + i * 32, bar);
            }
            if constexpr (RIGHT_MN) {
              if (maps.right_slabs) {
                pair_load_4d(right, &maps.right, 0, d0, col0 / 64, static_cast<int>(t.seg), bar);
              } else {
                for (int i = 0; i < 2; ++i)
                  pair_load_3d(right + i * kSlab, &maps.right, col0 + i * 64, d0, static_cast<int>(t.seg), bar);
              }
            } else {
              pair_load_3d(right, &maps.right, d0, col0, static_cast<int>(t.seg), bar);
            }
          }
        }
      }
      __syncwarp();
      at.skip(static_cast<uint32_t>(count));
      going = !abandoned_now();
    }
    if (!going)
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // given up: copies in flight get a millisecond to end
  } else if (warp == 1) {
    // ---------------------------------------------------------- products --
    const uint32_t instruction = umma_instruction(kPairRows, COLS, LEFT_MN, RIGHT_MN);
    RingPlace<STAGES> at{0, 0};
    int acc = 0;
    uint32_t acc_phase = 1, tails = 0;  // tails: bit s, the phase of stage s's tail barriers
    bool going = true;
    auto wait_cluster = [&](uint64_t *bar, uint32_t parity) {
      for (int i = 0; i < kMbarWaitLimit; ++i) {
        if (mbar_try_wait_cluster(bar, parity)) return true;
        if (*gate.abandoned) return false;
      }
      *gate.abandoned = 1;
      *gate.status = 1;
      return false;
    };
    for (int64_t index = first; going && walk.find(p, index, t); index += stride) {
      const int count = static_cast<int>(slices(t));
      if (count == 0) continue;  // (weights kind: the stores write zeros)
      // Slices that are whole; in the weights kind the last one may not be.
      const int whole = KIND == MATMUL_GRAD_WEIGHTS ? static_cast<int>((t.end - t.begin) / DEPTH) : count;
      const uint32_t to = tmem + acc * COLS;
      if (rank == 0 && elect_lane()) {
        bool there = wait_cluster(&drained[acc], acc_phase);
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        RingPlace<STAGES> here = at;
        for (int k = 0; there && k < whole; ++k, here.next()) {
          there = wait_cluster(&full[here.stage], here.phase);
          if (!there) break;
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          const uint32_t left = smem_u32(smem + here.stage * kStage);
          umma_stage<true, LEFT_MN, RIGHT_MN>(to, left, left + kPairHalf, kSlab, instruction, k > 0, DEPTH / 16);
          umma_pair_commit(&empty[here.stage]);
        }
        if (there && whole == count) umma_pair_commit(&ready[acc]);
      }
      __syncwarp();
      at.skip(static_cast<uint32_t>(whole));
      going = !abandoned_now();
      if (KIND == MATMUL_GRAD_WEIGHTS && going && whole < count) {
        const int stage = at.stage;
        // (the second CTA has not waited for the whole slices before this one)
        going = rank == 0 ? gate.wait_together(&full[stage], at.phase)
                          : gate.wait_together(&tail[stage], (tails >> stage) & 1, whole);
        if (!going) break;
        unsigned char *left = smem + stage * kStage, *right = left + kPairHalf;
        const int from = static_cast<int>(t.end - t.begin - int64_t{whole} * DEPTH), steps = (from + 15) / 16;
        const int rows = steps * 16 - from;
        for (int i = lane; i < rows * 8 * 4; i += 32) {  // two slabs of each operand
          const int slab = i / (rows * 8), row = from + i / 8 % rows;
          *reinterpret_cast<uint4 *>((slab < 2 ? left + slab * kSlab : right + (slab - 2) * kSlab) + row * 128 +
                                     i % 8 * 16) = uint4{0, 0, 0, 0};
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (rank == 0) {
          going = __all_sync(~0u, wait_cluster(&theirs[stage], (tails >> stage) & 1)) != 0;
          if (!going) break;
          if (elect_lane()) {
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            umma_stage<true, LEFT_MN, RIGHT_MN>(to, smem_u32(left), smem_u32(right), kSlab, instruction, whole > 0, steps);
            umma_pair_commit(&empty[stage]);
            umma_pair_commit(&ready[acc]);
          }
        } else if (elect_lane()) {
          mbar_arrive_first(&theirs[stage]);
        }
        __syncwarp();
        tails ^= 1u << stage;
        at.next();
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (!going && rank == 0) {  // given up: the products in flight end before tensor memory is freed
      if (elect_lane()) umma_pair_commit(&settled);
      __syncwarp();
      mbar_wait(&settled, 0);
    }
  } else {
    // ------------------------------------------------------------ stores --
    TensorStore<KIND, COLS> store(p, store_smem, warp & 3);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool going = true;
    for (int64_t index = first; going && walk.find(p, index, t); index += stride) {
      const bool nothing = KIND == MATMUL_GRAD_WEIGHTS && t.end == t.begin;
      if (!nothing) {
        going = gate.wait_together(&ready[acc], acc_phase, slices(t));
        if (!going) break;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      }
      store.tile(t, t.row + rank * 128, nothing, tmem + acc * COLS);
      if (!nothing) {
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        if (lane == 0) mbar_arrive_first(&drained[acc]);
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
  cluster_sync();  // no one reads or signals this CTA's shared memory any more
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "n"(2 * COLS) : "memory");
}

}  // namespace rgb
