// Products of e4m3 matrices with a scale for each block of 128 along the summed side, on tcgen05:
//
//   out[i, j] = sum over blocks b of  sa[i, b] * sb[j, b] * (sum over k in b of a[i, k] * b[j, k])   (+ bias, + out)
//
// The tensor cores sum one block of 128 (four MMAs of 32) into an accumulator of its own in TMEM; eight warps read it
// back, scale it by its row's and its column's factor and add it in fp32 registers, while the tensor cores work on the next
// blocks in the other accumulators.  Scales travel with their block: the producer warp brings the 128-byte rows of both operands
// by TMA and the block's scales by 4-byte asynchronous copies (any strides) into the same stage of the ring.
//
// A is [m, k], B is [n, k], both with rows of k codes: 128 of A times kTileN of B make a tile.  With kSwap A holds the
// weights and B a few tokens, and `out` is the transposed tile.
//
// Every spin-wait is bounded, as in gemm_sm100.cuh.
#pragma once

#include "cluster.cuh"
#include "gemm_sm100.cuh"

namespace dionw {
namespace float8 {

constexpr int kBM = 128;
constexpr int kBK = 128;                 // codes, and bytes, of a block
constexpr int kThreads = 320;            // warp 0: TMA and scales, warp 1: MMA + TMEM owner, warps 2-9: sums and output
constexpr int kSumWarps = 8;
constexpr uint32_t kABytes = kBM * kBK;  // 16 KB
constexpr int kAccumulators = 4;

// Scale of row i of an operand in block b: base[(i >> shift) * row_stride + b * block_stride].
struct Scales {
  const float* base;
  int64_t row_stride, block_stride;
  int shift;                             // 0: each row has its own; 7: 128 rows share one
};

struct Params {
  Scales a, b;
  void* out;
  int64_t ldo;
  const void* bias;                      // nullable: one for each column of `out`
  int out_dtype, bias_dtype;             // DIONW_F32, _F16, _BF16
  int accumulate;                        // add to what `out` holds
  int m, n, k;                           // rows of A, rows of B, summed length
  int tiles_m, tiles_n;
  int* status;
  uint64_t wait_ns;
};

template <int kTileN>
struct Shape {
  static constexpr int kColumns = kTileN / 2;                      // of a summing warp: half of the tile's
  static constexpr uint32_t kBBytes = kTileN * kBK;
  static constexpr uint32_t kScaleBytes = (kBM + kTileN) * 4;
  static constexpr uint32_t kStageBytes = (kABytes + kBBytes + kScaleBytes + 1023) / 1024 * 1024;
  static constexpr int kStages = kTileN == 128 ? 5 : 8;
  static constexpr uint32_t kTmemCols = kAccumulators * kTileN < 32 ? 32 : kAccumulators * kTileN;
  static constexpr uint32_t kStagingBytes = kTileN == 128 ? kSumWarps * 32 * 128 : 0;   // 32 rows of 32 floats a warp
  static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + kStagingBytes + 256 + 1024;
};

__device__ __forceinline__ void tma_load_2d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(gemm::smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(gemm::smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}

// Four bytes; zero instead where `there` is false (nothing is read then).
__device__ __forceinline__ void copy4(void* smem_dst, const float* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
               ::"r"(gemm::smem_u32(smem_dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}
// Arrives on `bar` once this thread's asynchronous copies so far are there.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(gemm::smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor for kind::f8f6f4: fp32 accumulate, e4m3 operands (format 0), both K-major.
constexpr uint32_t make_idesc(int m, int n) {
  return (1u << 4) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// kCount consecutive accumulator columns of this lane's row.  Valid after tmem_wait.
template <int kCount>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t* v);
template <>
__device__ __forceinline__ void tmem_load<8>(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr) : "memory");
}
template <>
__device__ __forceinline__ void tmem_load<16>(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(taddr) : "memory");
}
template <>
__device__ __forceinline__ void tmem_load<32>(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                 "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                 "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
               : "r"(taddr) : "memory");
}
// The registers pass through the wait, so that no use of them can be moved in front of it.
template <int kCount>
__device__ __forceinline__ void tmem_wait(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < kCount; i += 8)
    asm volatile("" : "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]),
                      "+r"(v[i + 6]), "+r"(v[i + 7]));
}

// One value in each of the three types.
__device__ __forceinline__ float load_as(const void* base, int64_t at, int dtype) {
  if (dtype == DIONW_F32) return static_cast<const float*>(base)[at];
  if (dtype == DIONW_F16) return __half2float(static_cast<const __half*>(base)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at]);
}
__device__ __forceinline__ void store_as(void* base, int64_t at, int dtype, float v) {
  if (dtype == DIONW_F32) static_cast<float*>(base)[at] = v;
  else if (dtype == DIONW_F16) static_cast<__half*>(base)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(v);
}

// Four values at out[row, col ..]: bias and what is there are added in fp32, the sum is rounded once.
__device__ __forceinline__ void put4(const Params& p, int row, int col, float4 v, bool vec) {
  const int cols = p.n;
  if (row >= p.m || col >= cols) return;
  float f[4] = {v.x, v.y, v.z, v.w};
  const int64_t at = int64_t(row) * p.ldo + col;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (col + i >= cols) continue;
    if (p.bias != nullptr) f[i] += load_as(p.bias, col + i, p.bias_dtype);
    if (p.accumulate) f[i] += load_as(p.out, at + i, p.out_dtype);
  }
  if (vec && col + 4 <= cols) {
    if (p.out_dtype == DIONW_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(f[0], f[1], f[2], f[3]);
    } else if (p.out_dtype == DIONW_F16) {
      *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) =
          make_uint2(gemm::pack2<__half>(f[0], f[1]), gemm::pack2<__half>(f[2], f[3]));
    } else {
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
          make_uint2(gemm::pack2<__nv_bfloat16>(f[0], f[1]), gemm::pack2<__nv_bfloat16>(f[2], f[3]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < cols) store_as(p.out, at + i, p.out_dtype, f[i]);
}

// Tiles in groups of eight tile rows that sweep the columns: a wave of CTAs shares its operands in L2.
__device__ __forceinline__ void tile_at(int t, const Params& p, int& tm, int& tn) {
  constexpr int kGroup = 8;
  const int per_group = kGroup * p.tiles_n, g = t / per_group;
  const int rows_here = min(kGroup, p.tiles_m - g * kGroup);
  const int r = t - g * per_group;
  tm = g * kGroup + r % rows_here;
  tn = r / rows_here;
}

template <int kTileN, bool kSwap>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
  using namespace gemm;
  using S = Shape<kTileN>;
  constexpr int kStages = S::kStages;
  constexpr int kAcc = kAccumulators;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + size_t(kStages) * S::kStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(staging + S::kStagingBytes);   // codes and scales of a stage are there
  uint64_t* empty_bar = full_bar + kStages;     // its MMAs are done, its scales read
  uint64_t* acc_full = empty_bar + kStages;     // [kAcc] a block's sums are complete
  uint64_t* acc_empty = acc_full + kAcc;        // [kAcc] they are read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + kAcc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total_tiles = p.tiles_m * p.tiles_n;
  const int k_blocks = (p.k + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1 + 32);          // the byte count, and the copies of each lane
      mbar_init(&empty_bar[s], 1 + kSumWarps);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], kSumWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (k_blocks > 0) {
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
    // ------------------------------------------------------------ TMA and scale producer
    uint32_t it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total_tiles && ok; t += gridDim.x) {
      int tm, tn;
      tile_at(t, p, tm, tn);
      const int m0 = tm * kBM, n0 = tn * kTileN;
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        const int s = it % kStages;
        if (!warp_wait(&empty_bar[s], ((it / kStages) & 1u) ^ 1u)) { ok = false; break; }
        uint8_t* a_dst = smem + size_t(s) * S::kStageBytes;
        uint8_t* b_dst = a_dst + kABytes;
        float* scale_dst = reinterpret_cast<float*>(b_dst + S::kBBytes);
        if (lane == 0) {
          mbar_expect_tx(&full_bar[s], kABytes + S::kBBytes);
          tma_load_2d(a_dst, &map_a, &full_bar[s], kb * kBK, m0);
          tma_load_2d(b_dst, &map_b, &full_bar[s], kb * kBK, n0);
        }
#pragma unroll
        for (int i = 0; i < kBM; i += 32) {
          const int row = m0 + i + lane;
          const bool there = row < p.m;
          copy4(scale_dst + i + lane,
                p.a.base + (there ? int64_t(row >> p.a.shift) * p.a.row_stride + kb * p.a.block_stride : 0), there);
        }
#pragma unroll
        for (int i = 0; i < kTileN; i += 32) {
          if (kTileN < 32 && lane >= kTileN) break;
          const int row = n0 + i + lane;
          const bool there = row < p.n;
          copy4(scale_dst + kBM + i + lane,
                p.b.base + (there ? int64_t(row >> p.b.shift) * p.b.row_stride + kb * p.b.block_stride : 0), there);
        }
        copies_arrive(&full_bar[s]);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = make_idesc(kBM, kTileN);
    uint32_t it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total_tiles && ok; t += gridDim.x) {
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        const int s = it % kStages;
        const uint32_t acc = it % kAcc;
        if (!warp_wait(&acc_empty[acc], ((it / kAcc) & 1u) ^ 1u)) { ok = false; break; }
        if (!warp_wait(&full_bar[s], (it / kStages) & 1u)) { ok = false; break; }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(smem + size_t(s) * S::kStageBytes);
        const uint64_t a_desc = make_smem_desc(a_addr, 16, 1024), b_desc = make_smem_desc(a_addr + kABytes, 16, 1024);
        if (lane == 0) {
#pragma unroll
          for (int j = 0; j < kBK / 32; ++j)    // 32 codes further along each 128-byte row
            umma_f8(tmem_base + acc * kTileN, a_desc + 2 * j, b_desc + 2 * j, idesc, j > 0 ? 1u : 0u);
          umma_commit(&empty_bar[s]);
          umma_commit(&acc_full[acc]);
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------ sums and output
    // Two warps for each TMEM sub-partition (a warp reads the 32 lanes 32 * (warp % 4) ..): half of the columns each.
    constexpr int kColumns = S::kColumns;
    constexpr int kPiece = kColumns < 32 ? kColumns : 32;
    const int sub = warp & 3;
    const int first_column = ((warp - 2) >> 2) * kColumns;
    uint8_t* stage_out = staging + (warp - 2) * 32 * 128;
    const bool vec = (p.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0;
    uint32_t it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total_tiles && ok; t += gridDim.x) {
      float sum[kColumns];
#pragma unroll
      for (int c = 0; c < kColumns; ++c) sum[c] = 0.0f;
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        const int s = it % kStages;
        const uint32_t acc = it % kAcc;
        if (!warp_wait(&full_bar[s], (it / kStages) & 1u)) { ok = false; break; }
        const float* scales = reinterpret_cast<const float*>(smem + size_t(s) * S::kStageBytes + kABytes + S::kBBytes);
        const float row_scale = scales[sub * 32 + lane];
        const float4* column_scales = reinterpret_cast<const float4*>(scales + kBM + first_column);
        if (!warp_wait(&acc_full[acc], (it / kAcc) & 1u)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int c0 = 0; c0 < kColumns; c0 += kPiece) {
          uint32_t v[kPiece];
          tmem_load<kPiece>(tmem_base + acc * kTileN + uint32_t(first_column + c0) + (uint32_t(sub * 32) << 16), v);
          tmem_wait<kPiece>(v);
#pragma unroll
          for (int c = 0; c < kPiece; c += 4) {
            const float4 f = column_scales[(c0 + c) / 4];
            sum[c0 + c] = fmaf(__uint_as_float(v[c]), row_scale * f.x, sum[c0 + c]);
            sum[c0 + c + 1] = fmaf(__uint_as_float(v[c + 1]), row_scale * f.y, sum[c0 + c + 1]);
            sum[c0 + c + 2] = fmaf(__uint_as_float(v[c + 2]), row_scale * f.z, sum[c0 + c + 2]);
            sum[c0 + c + 3] = fmaf(__uint_as_float(v[c + 3]), row_scale * f.w, sum[c0 + c + 3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&acc_empty[acc]);
          mbar_arrive(&empty_bar[s]);
        }
      }
      if (!ok) break;
      int tm, tn;
      tile_at(t, p, tm, tn);
      const int row0 = tm * kBM + sub * 32, col0 = tn * kTileN + first_column;
      if constexpr (kSwap) {
        // rows of A are columns of the output: 32 lanes write neighbours
        const int column = row0 + lane;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
          const int row = col0 + c;
          if (row >= p.n || column >= p.m) continue;
          const int64_t at = int64_t(row) * p.ldo + column;
          float f = sum[c];
          if (p.bias != nullptr) f += load_as(p.bias, column, p.bias_dtype);
          if (p.accumulate) f += load_as(p.out, at, p.out_dtype);
          store_as(p.out, at, p.out_dtype, f);
        }
      } else {
        // 32 columns at a time through shared memory: eight lanes write 32 neighbours of a row
#pragma unroll
        for (int c0 = 0; c0 < kColumns; c0 += 32) {
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<float4*>(stage_out + lane * 128 + ((u ^ (lane & 7)) << 4)) =
                make_float4(sum[c0 + 4 * u], sum[c0 + 4 * u + 1], sum[c0 + 4 * u + 2], sum[c0 + 4 * u + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3), u = lane & 7;
            const float4 f = *reinterpret_cast<const float4*>(stage_out + r * 128 + ((u ^ (r & 7)) << 4));
            put4(p, row0 + r, col0 + c0 + 4 * u, f, vec);
          }
        }
      }
    }
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

}  // namespace float8
}  // namespace dionw
