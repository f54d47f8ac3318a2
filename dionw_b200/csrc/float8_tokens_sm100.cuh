// The 8-bit product of float8_sm100.cuh for up to 64 rows on the left, a few tokens: `out` is the transposed tile of 128 rows of
// the weights (operand A here) times all tokens (operand B).
//
// Bound by the weights' bytes, 16 KB for each block and SM: at 6.5 TB/s and 148 SMs some 700 cycles.  With a barrier for
// each block, in the ring, to the summing warps and back, the warp that issues the MMAs took 780 cycles a block whatever the
// ring's depth (1 x 4096 x 14336 45.7 us, without the summing warps' barriers 34, with one MMA of the four 26): so stages and
// accumulators are of four blocks, with a barrier for all four.  A lane fetches its row's scales of four blocks at once, 16 bytes
// where they lie so: 4-byte copies of 32 rows are 32 lines each, and 64 x 14336 x 4096 took 23.5 us with them instead of 16.9.
// Where tiles are few, a cluster of two to eight CTAs shares a tile, each with a part of the blocks, and adds the parts in the
// order of their ranks through one another's shared memory.
//
// 1 x 14336 x 4096, call after call, takes 13.1 us where the calls go round ten matrices of weights, 4.5 TB/s from HBM, and 11.8 with the
// same one, whose 58.7 MB stay in L2 (recorded in a graph 12.8 and 9.2).  Some 3 of that are a launch that reads next to nothing.
// Leaving out the sums took 0.4 off; more bytes in flight (three stages) and tiles of fewer rows on more SMs changed nothing.  112 of
// the 148 SMs have a tile.
#pragma once

#include "float8_sm100.cuh"

namespace dionw {
namespace float8 {
namespace tokens {

constexpr int kGroup = 4;                // blocks of a stage, and of a set of accumulators
constexpr int kSets = 2;

template <int kTokens, bool kRowScales>
struct Shape {
  static constexpr int kColumns = kTokens / 2;                     // of a summing warp
  static constexpr uint32_t kBlockBytes = kABytes + kTokens * kBK;
  static constexpr uint32_t kStageBytes = kGroup * kBlockBytes;
  static constexpr int kStages = 2;
  static constexpr uint32_t kTmemCols = kSets * kGroup * kTokens;  // 128, 256 or 512
  // The tokens' scales of four blocks, block after block, twice, for each summing warp.
  static constexpr uint32_t kScaleBytes = kRowScales ? 2 * kGroup * kColumns * 4 : 0;
  static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + kSumWarps * kScaleBytes + 256 + 1024;
  static_assert(kTokens * kBM * 4 <= kStages * kStageBytes, "the parts of a tile lie where the ring was");
};

// The scales of one row of an operand, four blocks at a time.
struct RowScales {
  const float* at;           // nullptr: the row is not there, its scales are zero
  int64_t block_stride;
  bool whole;                // four blocks' lie in 16 aligned bytes

  __device__ __forceinline__ RowScales(const Scales& s, int row, int rows, int first_block)
      : at(row < rows ? s.base + int64_t(row >> s.shift) * s.row_stride + first_block * s.block_stride : nullptr),
        block_stride(s.block_stride), whole(s.block_stride == 1 && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {}
  // Of blocks k0 .. k0 + 3; zero from block `blocks` on.
  __device__ __forceinline__ float4 four(int k0, int blocks) const {
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (at == nullptr || k0 >= blocks) return f;
    const float* from = at + k0 * block_stride;
    if (whole && k0 + kGroup <= blocks) return __ldg(reinterpret_cast<const float4*>(from));
    f.x = __ldg(from);
    if (k0 + 1 < blocks) f.y = __ldg(from + block_stride);
    if (k0 + 2 < blocks) f.z = __ldg(from + 2 * block_stride);
    if (k0 + 3 < blocks) f.w = __ldg(from + 3 * block_stride);
    return f;
  }
};

template <typename T, int kTokens, bool kRowScales>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
  using namespace gemm;
  using S = Shape<kTokens, kRowScales>;
  constexpr int kStages = S::kStages, kColumns = S::kColumns;
  constexpr int kChunk = kColumns < 16 ? kColumns : 16, kChunks = kColumns / kChunk;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* token_scales = reinterpret_cast<float*>(smem + size_t(kStages) * S::kStageBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(token_scales + kSumWarps * S::kScaleBytes / 4);   // a stage's codes are there
  uint64_t* empty_bar = full_bar + kStages;     // its MMAs are done
  uint64_t* acc_full = empty_bar + kStages;     // [kSets] the sums of four blocks are complete
  uint64_t* acc_empty = acc_full + kSets;       // [kSets] they are read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + kSets);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // A cluster's CTAs share a tile: CTA `rank` takes the blocks from first_block on.  (One tile a cluster of several CTAs.)
  const int parts = int(cluster_size()), rank = int(cluster_rank());
  const int all_blocks = (p.k + kBK - 1) / kBK, share = ((all_blocks + parts - 1) / parts + kGroup - 1) / kGroup * kGroup;
  const int first_block = min(rank * share, all_blocks), k_blocks = min(share, all_blocks - first_block);
  const int first_tile = int(blockIdx.x) / parts, stride = int(gridDim.x) / parts;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < kSets; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], kSumWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (all_blocks > 0) {
      prefetch_map(&map_a);
      prefetch_map(&map_b);
    }
  }
  if (warp == 1) tmem_alloc(tmem_slot, S::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch();

  auto warp_wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, p.wait_ns)) != 0;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    uint32_t it = 0;
    bool ok = true;
    for (int t = first_tile; t < p.tiles_m && ok; t += stride) {
      for (int k0 = 0; k0 < k_blocks; k0 += kGroup, ++it) {
        const int s = it % kStages, count = min(kGroup, k_blocks - k0);
        if (!warp_wait(&empty_bar[s], ((it / kStages) & 1u) ^ 1u)) { ok = false; break; }
        uint8_t* dst = smem + size_t(s) * S::kStageBytes;
        if (gemm2::elect_one()) {
          mbar_expect_tx(&full_bar[s], uint32_t(count) * S::kBlockBytes);
#pragma unroll
          for (int j = 0; j < kGroup; ++j) {
            if (j >= count) break;
            const int at = (first_block + k0 + j) * kBK;
            tma_load_2d(dst + j * S::kBlockBytes, &map_a, &full_bar[s], at, t * kBM);
            tma_load_2d(dst + j * S::kBlockBytes + kABytes, &map_b, &full_bar[s], at, 0);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = make_idesc(kBM, kTokens);
    uint32_t it = 0;
    bool ok = true;
    for (int t = first_tile; t < p.tiles_m && ok; t += stride) {
      for (int k0 = 0; k0 < k_blocks; k0 += kGroup, ++it) {
        const int s = it % kStages, count = min(kGroup, k_blocks - k0);
        const uint32_t set = it % kSets;
        if (!warp_wait(&acc_empty[set], ((it / kSets) & 1u) ^ 1u)) { ok = false; break; }
        if (!warp_wait(&full_bar[s], (it / kStages) & 1u)) { ok = false; break; }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(smem + size_t(s) * S::kStageBytes);
        const uint64_t a_desc = make_smem_desc(a_addr, 16, 1024), b_desc = make_smem_desc(a_addr + kABytes, 16, 1024);
        if (gemm2::elect_one()) {
#pragma unroll
          for (int j = 0; j < kGroup; ++j) {
            if (j >= count) break;
            const uint64_t step = uint64_t(j) * (S::kBlockBytes >> 4);
            const uint32_t acc = tmem_base + (set * kGroup + j) * kTokens;
#pragma unroll
            for (int i = 0; i < kBK / 32; ++i)    // 32 codes further along each 128-byte row
              umma_f8(acc, a_desc + step + 2 * i, b_desc + step + 2 * i, idesc, i > 0 ? 1u : 0u);
          }
          umma_commit(&empty_bar[s]);
          umma_commit(&acc_full[set]);
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------ sums and output
    // Two warps for each TMEM sub-partition (a warp reads the 32 lanes 32 * (warp % 4) ..): half of the tokens each.
    const int sub = warp & 3;
    const int first_token = ((warp - 2) >> 2) * kColumns;
    const uint32_t tmem_mine = tmem_base + uint32_t(first_token) + (uint32_t(sub * 32) << 16);
    float* const scales_here = token_scales + (warp - 2) * (S::kScaleBytes / 4);
    uint32_t it = 0;
    bool ok = true;
    for (int t = first_tile; t < p.tiles_m; t += stride) {
      const int row0 = t * kBM + sub * 32;
      // Scales are two groups of blocks ahead, in registers: a row's for its lane, and a token's each for the first kColumns lanes.
      const RowScales weights(p.a, row0 + lane, p.m, first_block);
      const RowScales tokens(p.b, kRowScales ? first_token + (lane < kColumns ? lane : 0) : 0, p.n, first_block);
      float4 row_scales[3], token_scales4[3];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        row_scales[i] = weights.four(kGroup * i, k_blocks);
        token_scales4[i] = tokens.four(kGroup * i, k_blocks);
      }
      uint64_t sum[kColumns / 2];
#pragma unroll
      for (int c = 0; c < kColumns / 2; ++c) sum[c] = 0;
      for (int k0 = 0; k0 < k_blocks; k0 += kGroup, ++it) {
        const uint32_t set = it % kSets;
        const int count = min(kGroup, k_blocks - k0);
        row_scales[2] = weights.four(k0 + 2 * kGroup, k_blocks);
        token_scales4[2] = tokens.four(k0 + 2 * kGroup, k_blocks);
        float factor[kGroup] = {row_scales[0].x, row_scales[0].y, row_scales[0].z, row_scales[0].w};
        const float4 of_token = token_scales4[0];
        float* const by_block = scales_here + (it & 1u) * (kGroup * kColumns);
        if constexpr (kRowScales) {
          if (lane < kColumns) {       // (the other half of the room may still be read)
            by_block[lane] = of_token.x;
            by_block[kColumns + lane] = of_token.y;
            by_block[2 * kColumns + lane] = of_token.z;
            by_block[3 * kColumns + lane] = of_token.w;
          }
        } else {
          factor[0] *= of_token.x; factor[1] *= of_token.y; factor[2] *= of_token.z; factor[3] *= of_token.w;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          row_scales[i] = row_scales[i + 1];
          token_scales4[i] = token_scales4[i + 1];
        }
        if (!warp_wait(&acc_full[set], (it / kSets) & 1u)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        // A chunk of a block's sums is on its way from TMEM while the one before is added.
        const uint32_t accumulators = tmem_mine + set * kGroup * kTokens;
        uint32_t v[2][kChunk];
        tmem_load<kChunk>(accumulators, v[0]);
#pragma unroll
        for (int i = 0; i < kGroup * kChunks; ++i) {
          const int j = i / kChunks, c0 = i % kChunks * kChunk, next = i + 1;
          if (j >= count) break;
          tmem_wait<kChunk>(v[i & 1]);
          if (next < count * kChunks) {
            if (next < kGroup * kChunks)
              tmem_load<kChunk>(accumulators + uint32_t(next / kChunks * kTokens + next % kChunks * kChunk), v[next & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[set]);
          }
          add_columns<kChunk, kRowScales>(v[i & 1], two(__float_as_uint(factor[j]), __float_as_uint(factor[j])),
                                          by_block + j * kColumns + c0, sum + c0 / 2);
        }
      }
      if (!ok) break;
      const int column = row0 + lane;            // of the output: 32 lanes write neighbours
      if (parts == 1) {
        const float bias = p.bias != nullptr && column < p.m ? bias_at(p, column) : 0.0f;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
          const int row = first_token + c;
          if (row >= p.n || column >= p.m) continue;
          T* at = static_cast<T*>(p.out) + int64_t(row) * p.ldo + column;
          const float2 pair = apart(sum[c / 2]);
          float f = ((c & 1) != 0 ? pair.y : pair.x) + bias;
          if (p.accumulate) f += to_float<T>(*at);
          *at = from_float<T>(f);
        }
      } else {
        // The ring is done with: every MMA that read it has been waited for.
        float* part = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
          const float2 pair = apart(sum[c / 2]);
          part[(first_token + c) * kBM + sub * 32 + lane] = (c & 1) != 0 ? pair.y : pair.x;
        }
      }
    }
  }

  // ------------------------------------------------------------ a tile's parts
  if (parts > 1) {
    cluster_sync();
    const float* part = reinterpret_cast<const float*>(smem);
    const bool complete = *abort_flag == 0;
    for (int i = rank * kThreads + int(threadIdx.x); complete && i < p.n * kBM; i += parts * kThreads) {
      const int row = i / kBM, column = first_tile * kBM + i % kBM;
      if (column >= p.m) continue;
      float f = 0.0f;
      for (int q = 0; q < parts; ++q) f += __uint_as_float(peer_load(part + i, q));
      T* at = static_cast<T*>(p.out) + int64_t(row) * p.ldo + column;
      if (p.bias != nullptr) f += bias_at(p, column);
      if (p.accumulate) f += to_float<T>(*at);
      *at = from_float<T>(f);
    }
    cluster_sync();   // nobody's shared memory is read any more
  }

  // ------------------------------------------------------------ teardown
  __syncthreads();
  if (*abort_flag != 0 && threadIdx.x == 0) {
    // copies that may still be in flight land before the shared memory is released
    const uint64_t start = global_ns();
    while (global_ns() - start < 200000ull) {
    }
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

}  // namespace tokens
}  // namespace float8
}  // namespace dionw
