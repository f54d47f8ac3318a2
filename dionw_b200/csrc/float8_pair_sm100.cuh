// The 8-bit product of float8_sm100.cuh on SM pairs: a cluster of two CTAs computes 256 x 256 tiles with
// tcgen05.mma.cta_group::2.  Each CTA loads its 128 rows of A and half of B's 256, and scales and adds the blocks' sums of
// its 128 rows: 128 fp32 sums a thread, in pairs (fma.rn.f32x2).
//
// The bound: a block of 128 is 512 cycles of MMA for 32 KB of codes a CTA.  In that time its eight summing warps read 128 x
// 256 accumulators from TMEM (128 bytes each cycle and sub-partition: 256 cycles) and add them (64 packed
// multiply-adds a thread, 128 issue cycles; twice that where each row of B has a scale of its own).  Two
// accumulators of 256 columns are all of TMEM, so the warps give one back as soon as it is in registers.  Measured with scales
// that are no powers of two: 8192 x 14336 x 4096 490 us with B's in tiles, 826 to 880 with a scale for each row of both, the look at
// them included (the tensor cores apply powers of two in 350, float8_scaled_sm100.cuh).  What takes the rest of the time has not been found.
#pragma once

#include "float8_sm100.cuh"
#include "gemm2_sm100.cuh"

namespace dionw {
namespace float8 {
namespace pair {

constexpr int kPairM = 256, kPairN = 256;
constexpr int kThreads = 384;            // warp 0: TMA, warp 1: MMA + TMEM owner, warps 4-11: sums and output
// Registers: 384 threads are launched with 168 each; 128 * 40 + 256 * 232 = 384 * 168.
constexpr int kHelperRegisters = 40, kSumRegisters = 232;
constexpr int kStages = 5;
constexpr int kColumns = kPairN / 2;     // of a summing warp
constexpr uint32_t kStageBytes = 2 * kABytes;          // 128 rows of A, 128 of B
constexpr uint32_t kStagingBytes = kSumWarps * 32 * 128;
template <bool kRowScales>
using Queue = ScaleQueue<kRowScales ? kColumns : 0, kRowScales ? 4 : 8>;
template <bool kRowScales>
constexpr size_t kSmemBytes =
    size_t(kStages) * kStageBytes + kStagingBytes + kSumWarps * Queue<kRowScales>::kBytes + 256 + 1024;

__device__ __forceinline__ void tma_load_pair(uint32_t smem_dst, const CUtensorMap* map, uint32_t leader_bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(leader_bar), "r"(c0), "r"(c1)
      : "memory");
}

__device__ __forceinline__ void umma2_f8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// kRowScales: each row of B has its own scales; otherwise 128 share one.
template <typename T, bool kRowScales>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
  using namespace gemm;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + size_t(kStages) * kStageBytes;
  uint8_t* queues = staging + kStagingBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(queues + kSumWarps * Queue<kRowScales>::kBytes);  // leader's: both CTAs' codes landed
  uint64_t* empty_bar = full_bar + kStages;            // both: the pair's MMAs on this stage completed
  uint64_t* acc_full = empty_bar + kStages;            // [2] both
  uint64_t* acc_empty = acc_full + 2;                  // [2] leader's: both CTAs have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int first_tile = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  int total_tiles = p.tiles_m * p.tiles_n;
  const int k_blocks = (p.k + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kSumWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (k_blocks > 0) {
      prefetch_map(&map_a);
      prefetch_map(&map_b);
    }
  }
  if (warp == 1) gemm2::tmem_alloc2(tmem_slot, kTmemCols);
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // both CTAs' barriers exist before anyone arrives on a peer's
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch();
  // Scales that are all powers of two have been left to the tensor cores: nothing is left to do.
  if (p.odd_scales != nullptr && !any_odd_scale(p)) total_tiles = 0;

  auto warp_wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, p.wait_ns)) != 0;
  };

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kHelperRegisters));
  if (warp == 0) {
    // ---------------------------------------------------------- TMA producer (both CTAs)
    int s = 0;
    uint32_t released = 1;
    bool ok = true;
    const uint32_t ring = smem_u32(smem), leader_full = peer_address(full_bar, 0);
    for (int t = first_tile; t < total_tiles && ok; t += pairs) {
      int tm, tn;
      tile_at(t, p, tm, tn);
      const int m0 = tm * kPairM + int(rank) * kBM, n0 = tn * kPairN + int(rank) * (kPairN / 2);
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!warp_wait(&empty_bar[s], released)) { ok = false; break; }
        if (gemm2::elect_one()) {
          const uint32_t dst = ring + uint32_t(s) * kStageBytes;
          const uint32_t landed = leader_full + uint32_t(s) * uint32_t(sizeof(uint64_t));
          // The peer's bytes may land before the leader announces them: the phase cannot complete before its arrive.
          if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * kStageBytes);
          tma_load_pair(dst, &map_a, landed, kb * kBK, m0);
          tma_load_pair(dst + kABytes, &map_b, landed, kb * kBK, n0);
        }
        __syncwarp();
        if (++s == kStages) s = 0, released ^= 1u;
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {   // the second CTA's MMA warp has nothing to issue
      // ---------------------------------------------------------- MMA issuer (leader)
      constexpr uint32_t idesc = make_idesc(kPairM, kPairN);
      int s = 0;
      uint32_t loaded = 0, it = 0;
      bool ok = true;
      const uint32_t ring = smem_u32(smem);
      for (int t = first_tile; t < total_tiles && ok; t += pairs) {
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const uint32_t acc = it & 1u;
          if (!warp_wait(&acc_empty[acc], ((it >> 1) & 1u) ^ 1u)) { ok = false; break; }
          if (!warp_wait(&full_bar[s], loaded)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = ring + uint32_t(s) * kStageBytes;
          const uint64_t a_desc = make_smem_desc(a_addr, 16, 1024), b_desc = make_smem_desc(a_addr + kABytes, 16, 1024);
          if (gemm2::elect_one()) {
#pragma unroll
            for (int j = 0; j < kBK / 32; ++j)
              umma2_f8(tmem_base + acc * uint32_t(kPairN), a_desc + 2 * j, b_desc + 2 * j, idesc, j > 0 ? 1u : 0u);
            gemm2::umma2_commit_both(&empty_bar[s]);
            gemm2::umma2_commit_both(&acc_full[acc]);
          }
          __syncwarp();
          if (++s == kStages) s = 0, loaded ^= 1u;
        }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ sums and output (both CTAs)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegisters));
    const int sub = warp & 3, half = (warp - 4) >> 2;
    uint8_t* stage_out = staging + (warp - 4) * 32 * 128;
    const uint32_t tmem_mine = tmem_base + uint32_t(half * kColumns) + (uint32_t(sub * 32) << 16);
    const uint32_t leader_empty = peer_address(acc_empty, 0);
    Queue<kRowScales> queue(queues + (warp - 4) * Queue<kRowScales>::kBytes);
    const int row_in_tile = int(rank) * kBM + sub * 32, col_in_tile = half * kColumns;
    uint32_t it = 0;
    bool ok = true;
    int tm, tn;
    if (first_tile < total_tiles) {
      tile_at(first_tile, p, tm, tn);
      queue.start(p, tm * kPairM + row_in_tile, tn * kPairN + col_in_tile, 0, k_blocks, lane);
    }
    for (int t = first_tile; t < total_tiles; t += pairs) {
      uint64_t sum[kColumns / 2];
#pragma unroll
      for (int c = 0; c < kColumns / 2; ++c) sum[c] = 0;
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        const uint32_t acc = it & 1u;
        if (!warp_wait(&acc_full[acc], (it >> 1) & 1u)) { ok = false; break; }
        tc_fence_after();
        add_block<kColumns, kRowScales ? 8 : 16, kRowScales>(
            tmem_mine + acc * uint32_t(kPairN), lane, sum, [&] { return queue.take(p, k_blocks - 1 - kb, lane); },
            [&] {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) gemm2::remote_arrive(leader_empty + acc * uint32_t(sizeof(uint64_t)));
            });
      }
      if (!ok) break;
      const int row0 = tm * kPairM + row_in_tile, col0 = tn * kPairN + col_in_tile;
      if (t + pairs < total_tiles) {   // the next tile's first scales come while this one's sums go out
        tile_at(t + pairs, p, tm, tn);
        queue.start(p, tm * kPairM + row_in_tile, tn * kPairN + col_in_tile, 0, k_blocks, lane);
      }
      write_sums<T, kColumns>(p, stage_out, row0, col0, lane, [&](int c) {
        const float2 f = apart(sum[c / 2]);
        return (c & 1) != 0 ? f.y : f.x;
      });
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }

  // ------------------------------------------------------------ teardown
  __syncthreads();
  if (*abort_flag != 0 && threadIdx.x == 0) {
    const uint64_t start = global_ns();
    while (global_ns() - start < 200000ull) {
    }
  }
  cluster_sync();   // the peer may still be reading this CTA's shared memory through the pair's MMAs
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    gemm2::tmem_dealloc2(tmem_base, kTmemCols);
  }
}

}  // namespace pair
}  // namespace float8
}  // namespace dionw
