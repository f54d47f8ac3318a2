// The 8-bit product with powers of two for scales, on SM pairs: the tensor cores apply the scales themselves
// (tcgen05.mma kind::mxf8f6f4, block_scale), so that a tile's sums stay in TMEM and the warps that write them
// out have next to nothing to do in the main loop.  For what the quantizer makes; scales of any value take
// float8_pair_sm100.cuh, whose warps add 256 x 256 sums for each block of 128.
//
// Exponents travel as words of 32 bits with the scale's exponent in the low byte (UE8M0, the same bias as fp32's), 128 rows of a
// block together, in the order that the tensor cores want them: word 4 l + c is row 32 c + l.  TMA brings 128 of A and 256 of B
// into each CTA with the codes of a block, tcgen05.cp from there into TMEM, where each 32 lanes get a copy.  The hardware takes
// one scale for 32 codes of a row; the four MMAs of a block use the same ones.
//
// The tensor cores cut off what an addition to their fp32 sums leaves behind the last place, up to 2^-23 of the sum for each 32
// products, so that sums of one sign fall behind: 1e-3 of one of half a million.  After kPiece blocks the sums are therefore taken into
// registers, where the pieces are added to nearest: at most 128 * 2^-23 = 1.5e-5 for a piece, and 2^-24 for each addition of one.
// Measured on positive values of a wide range, 2304 x 2304 sums of 4096 to 131072 products: 1.35e-6 on average, 2.4e-6 at most (sums in
// registers block by block, as float8_sm100.cuh does: 7e-8 to 3.7e-7 on average, 2.4e-6 at most).
//
// A tile's 256 columns are half of TMEM and there is one of them: the eight warps take it into registers at once, and
// convert and store while the next tile is computed.  Tiles of 256 x 128 are for products that have too few of the wide ones.
//
// 8192 x 14336 x 4096 takes 350 us in short runs, 2.75 PFLOP/s; 577 cycles a block where the MMAs alone are 512, at some 1.3 GHz:
// the power cap sets the clock, and long runs take 420 to 440 us.
#pragma once

#include "float8_pair_sm100.cuh"

namespace dionw {
namespace float8 {
namespace scaled {

using pair::kPairM;
constexpr int kThreads = pair::kThreads;
constexpr uint32_t kAtomBytes = 512;                       // the exponents of 128 rows
constexpr uint32_t kStagingBytes = kSumWarps * 32 * 128;
constexpr uint32_t kScaleColumns = 16;                     // of TMEM, for a block's exponents: 4 of A, 4 for each 128 of B
constexpr uint32_t kScaleBuffers = 8;
constexpr int kPiece = 32;                                 // blocks of 128 that are summed in TMEM
constexpr uint32_t kScalesAt = 256;                        // the columns behind the sums

// kTileN: 256 or 128.
template <int kTileN>
struct Shape {
  static constexpr int kColumns = kTileN / 2;                               // of a warp
  static constexpr int kStages = kTileN == 256 ? 5 : 6;
  static constexpr uint32_t kCodeBytes = kABytes + kTileN / 2 * kBK;        // 128 rows of A, half of B's
  static constexpr uint32_t kAtoms = 1 + kTileN / 128;
  static constexpr uint32_t kLoadBytes = kCodeBytes + kAtoms * kAtomBytes;
  static constexpr uint32_t kStageBytes = (kLoadBytes + 1023) / 1024 * 1024;
  static constexpr uint32_t kSums = 256 / kTileN;                           // accumulators
  static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + kStagingBytes + 256 + 1024;
};

struct Maps {
  CUtensorMap a, b, a_scales, b_scales;
};

// Shared memory to TMEM, in both CTAs of the pair: 32 rows of 16 bytes, to each 32 lanes.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// 16-byte rows one after the other, no swizzle: 128 bytes between groups of eight.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}

__device__ __forceinline__ void umma2_scaled(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                             uint32_t tmem_sa, uint32_t tmem_sb, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(tmem_sa), "r"(tmem_sb), "r"(accumulate)
      : "memory");
}

// Instruction descriptor: e4m3 operands (format 0), both K-major, UE8M0 scales (bit 23), the low byte of their words.
constexpr uint32_t make_idesc(int m, int n) {
  return (uint32_t(n >> 3) << 17) | (1u << 23) | (uint32_t(m >> 4) << 24);
}

// Adds the accumulator at `taddr` to this lane's sums (in pairs); `release` is called once it is in registers.
template <int kColumns, typename Release>
__device__ __forceinline__ void add_pieces(uint32_t taddr, uint64_t (&sum)[kColumns / 2], Release&& release) {
  uint32_t v[2][16];
  tmem_load<16>(taddr, v[0]);
  tmem_load<16>(taddr + 16, v[1]);
#pragma unroll
  for (int c0 = 0; c0 < kColumns; c0 += 32) {
    tmem_wait<16>(v[0]);
    tmem_pass<16>(v[1]);
    if (c0 + 32 == kColumns) release();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        uint64_t& s = sum[(c0 + 16 * h + i) / 2];
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(s) : "l"(two(v[h][i], v[h][i + 1])));
      }
      if (c0 + 32 < kColumns) tmem_load<16>(taddr + c0 + 32 + 16 * h, v[h]);
    }
  }
}

template <typename T, int kTileN>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ Maps maps, const Params p) {
  using namespace gemm;
  using S = Shape<kTileN>;
  constexpr int kStages = S::kStages, kColumns = S::kColumns;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + size_t(kStages) * S::kStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(staging + kStagingBytes);  // leader's: both CTAs' stage landed
  uint64_t* empty_bar = full_bar + kStages;            // both: the pair's MMAs on this stage completed
  uint64_t* acc_full = empty_bar + kStages;            // [kSums] both: a tile's sums are complete
  uint64_t* acc_empty = acc_full + S::kSums;           // [kSums] leader's: both CTAs have them in registers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + S::kSums);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int first_tile = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  int total_tiles = p.tiles_m * p.tiles_n;
  const int k_blocks = (p.k + kBK - 1) / kBK;          // at least one

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (uint32_t a = 0; a < S::kSums; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kSumWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    prefetch_map(&maps.a);
    prefetch_map(&maps.b);
    prefetch_map(&maps.a_scales);
    prefetch_map(&maps.b_scales);
  }
  if (warp == 1) gemm2::tmem_alloc2(tmem_slot, kTmemCols);
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // both CTAs' barriers exist before anyone arrives on a peer's
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch();
  // With a scale of any other value the kernel after this one does the work.
  if (p.odd_scales != nullptr && any_odd_scale(p)) total_tiles = 0;

  auto warp_wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, p.wait_ns)) != 0;
  };

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(pair::kHelperRegisters));
  if (warp == 0) {
    // ---------------------------------------------------------- TMA producer (both CTAs)
    int s = 0;
    uint32_t released = 1;
    bool ok = true;
    const uint32_t ring = smem_u32(smem), leader_full = peer_address(full_bar, 0);
    const int a_atoms = (p.m + 127) / 128, b_atoms = (p.n + 127) / 128;
    for (int t = first_tile; t < total_tiles && ok; t += pairs) {
      int tm, tn;
      tile_at(t, p, tm, tn);
      const int m0 = tm * kPairM + int(rank) * kBM, n0 = tn * kTileN + int(rank) * (kTileN / 2);
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!warp_wait(&empty_bar[s], released)) { ok = false; break; }
        if (gemm2::elect_one()) {
          const uint32_t dst = ring + uint32_t(s) * S::kStageBytes;
          const uint32_t landed = leader_full + uint32_t(s) * uint32_t(sizeof(uint64_t));
          // The peer's bytes may land before the leader announces them: the phase cannot complete before its arrive.
          if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * S::kLoadBytes);
          pair::tma_load_pair(dst, &maps.a, landed, kb * kBK, m0);
          pair::tma_load_pair(dst + kABytes, &maps.b, landed, kb * kBK, n0);
          // (the second half of a last tile may be past its block's exponents: those rows are not stored)
          pair::tma_load_pair(dst + S::kCodeBytes, &maps.a_scales, landed, 0, kb * a_atoms + m0 / 128);
          pair::tma_load_pair(dst + S::kCodeBytes + kAtomBytes, &maps.b_scales, landed, 0, kb * b_atoms + tn * (kTileN / 128));
        }
        __syncwarp();
        if (++s == kStages) s = 0, released ^= 1u;
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {   // the second CTA's MMA warp has nothing to issue
      // ---------------------------------------------------------- MMA issuer (leader)
      constexpr uint32_t idesc = make_idesc(kPairM, kTileN);
      int s = 0;
      uint32_t loaded = 0, local = 0, buffer = 0;
      bool ok = true;
      const uint32_t ring = smem_u32(smem);
      for (int t = first_tile; t < total_tiles && ok; t += pairs) {
        uint32_t acc = 0;
        for (int kb = 0; kb < k_blocks; ++kb) {
          const bool first = kb % kPiece == 0, last = (kb + 1) % kPiece == 0 || kb + 1 == k_blocks;   // of a piece
          if (first) {
            acc = local % S::kSums;
            if (!warp_wait(&acc_empty[acc], ((local / S::kSums) & 1u) ^ 1u)) { ok = false; break; }
            tc_fence_after();
            ++local;
          }
          if (!warp_wait(&full_bar[s], loaded)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = ring + uint32_t(s) * S::kStageBytes;
          const uint64_t a_desc = make_smem_desc(a_addr, 16, 1024), b_desc = make_smem_desc(a_addr + kABytes, 16, 1024);
          const uint64_t scales = scale_desc(a_addr + S::kCodeBytes);
          const uint32_t sa = tmem_base + kScalesAt + buffer * kScaleColumns, sb = sa + 4;
          if (gemm2::elect_one()) {
            copy_scales(sa, scales);
            copy_scales(sb, scales + (kAtomBytes >> 4));
            if (kTileN == 256) copy_scales(sb + 4, scales + (2 * kAtomBytes >> 4));
#pragma unroll
            for (int j = 0; j < kBK / 32; ++j)
              umma2_scaled(tmem_base + acc * kTileN, a_desc + 2 * j, b_desc + 2 * j, idesc, sa, sb, !first || j > 0 ? 1u : 0u);
            gemm2::umma2_commit_both(&empty_bar[s]);
            if (last) gemm2::umma2_commit_both(&acc_full[acc]);
          }
          __syncwarp();
          buffer = (buffer + 1) % kScaleBuffers;
          if (++s == kStages) s = 0, loaded ^= 1u;
        }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ output (both CTAs)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(pair::kSumRegisters));
    const int sub = warp & 3, half = (warp - 4) >> 2;
    uint8_t* stage_out = staging + (warp - 4) * 32 * 128;
    const uint32_t tmem_mine = tmem_base + uint32_t(half * kColumns) + (uint32_t(sub * 32) << 16);
    const uint32_t leader_empty = peer_address(acc_empty, 0);
    uint32_t local = 0;
    bool ok = true;
    for (int t = first_tile; t < total_tiles; t += pairs) {
      uint64_t sum[kColumns / 2];
#pragma unroll
      for (int c = 0; c < kColumns / 2; ++c) sum[c] = 0;
      for (int kb = 0; kb < k_blocks; kb += kPiece, ++local) {
        const uint32_t acc = local % S::kSums;
        if (!warp_wait(&acc_full[acc], (local / S::kSums) & 1u)) { ok = false; break; }
        tc_fence_after();
        const uint32_t from = tmem_mine + acc * kTileN;
        add_pieces<kColumns>(from, sum, [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) gemm2::remote_arrive(leader_empty + acc * uint32_t(sizeof(uint64_t)));
        });
      }
      if (!ok) break;
      int tm, tn;
      tile_at(t, p, tm, tn);
      write_sums<T, kColumns>(p, stage_out, tm * kPairM + int(rank) * kBM + sub * 32, tn * kTileN + half * kColumns, lane,
                              [&](int c) {
                                const float2 f = apart(sum[c / 2]);
                                return (c & 1) != 0 ? f.y : f.x;
                              });
    }
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

}  // namespace scaled
}  // namespace float8
}  // namespace dionw
