// Products of e4m3 matrices with a scale for each block of 128 along the summed side, on tcgen05:
//
//   out[i, j] = sum over blocks b of  sa[i, b] * sb[j, b] * (sum over k in b of a[i, k] * b[j, k])   (+ bias, + out)
//
// The tensor cores sum one block of 128 (four MMAs of 32) into an accumulator of its own in TMEM; eight warps read it
// back, scale it by its row's and its column's factor and add it in fp32 registers, while the tensor cores work on the next
// blocks in the other accumulators.  The codes come by TMA; each summing warp fetches the scales it needs itself, a few blocks
// ahead, by 4-byte asynchronous copies (any strides) into a queue of its own.
//
// A is [m, k], B is [n, k], both with rows of k codes: 128 of each make a tile.  (Few rows on the left: float8_tokens_sm100.cuh.)
//
// Every spin-wait is bounded, as in gemm_sm100.cuh.
#pragma once

#include "cluster.cuh"
#include "gemm2_sm100.cuh"
#include "gemm_sm100.cuh"

namespace dionw {
namespace float8 {

constexpr int kBM = 128;
constexpr int kBK = 128;                 // codes, and bytes, of a block
constexpr int kThreads = 320;            // warp 0: TMA, warp 1: MMA + TMEM owner, warps 2-9: sums and output
constexpr int kSumWarps = 8;
constexpr uint32_t kABytes = kBM * kBK;  // 16 KB
constexpr int kTileN = 128;
constexpr int kAccumulators = 4;
constexpr int kMaxParts = 8;             // CTAs of a cluster that share a tile

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
  int bias_dtype;                        // DIONW_F32, _F16, _BF16
  int accumulate;                        // add to what `out` holds
  int m, n, k;                           // rows of A, rows of B, summed length
  int tiles_m, tiles_n;
  const int* odd_scales;                 // nullable: `odd_parts` words, not all zero if some scale is no power of two
  int odd_parts;
  int* status;
  uint64_t wait_ns;
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
__device__ __forceinline__ void tmem_pass(uint32_t* v) {
#pragma unroll
  for (int i = 0; i < kCount; i += 8)
    asm volatile("" : "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]),
                      "+r"(v[i + 6]), "+r"(v[i + 7]));
}
template <int kCount>
__device__ __forceinline__ void tmem_wait(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  tmem_pass<kCount>(v);
}

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float bias_at(const Params& p, int at) {
  if (p.bias_dtype == DIONW_F32) return static_cast<const float*>(p.bias)[at];
  if (p.bias_dtype == DIONW_F16) return __half2float(static_cast<const __half*>(p.bias)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[at]);
}

// Four neighbours of an output row.
template <typename T>
struct Four {
  uint32_t w[2];
  __device__ __forceinline__ void load(const T* at) {
    const uint2 raw = *reinterpret_cast<const uint2*>(at);
    w[0] = raw.x; w[1] = raw.y;
  }
  __device__ __forceinline__ void set(int i, T v) {
    const uint32_t bits = *reinterpret_cast<const uint16_t*>(&v);
    w[i >> 1] = i & 1 ? (w[i >> 1] & 0xFFFFu) | (bits << 16) : bits;
  }
  __device__ __forceinline__ float value(int i) const {
    const float2 v = gemm::unpack2<T>(w[i >> 1]);
    return i & 1 ? v.y : v.x;
  }
  static __device__ __forceinline__ void store(T* at, const float (&f)[4]) {
    *reinterpret_cast<uint2*>(at) = make_uint2(gemm::pack2<T>(f[0], f[1]), gemm::pack2<T>(f[2], f[3]));
  }
};
template <>
struct Four<float> {
  float f[4];
  __device__ __forceinline__ void load(const float* at) {
    const float4 v = *reinterpret_cast<const float4*>(at);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
  __device__ __forceinline__ void set(int i, float v) { f[i] = v; }
  __device__ __forceinline__ float value(int i) const { return f[i]; }
  static __device__ __forceinline__ void store(float* at, const float (&v)[4]) {
    *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
  }
};

// The 32 x kColumns sums of a warp (lane l: row row0 + l, columns col0 ..; get(c) is the sum of column c) into `out`, through
// 4 KB of the warp's shared memory: 128 bytes of each row at a time, kept at unit ^ (row % 8) of 16 bytes, so that
// neither the rows on the way in nor the lines on the way out meet in a bank.  Eight lanes then write 128 bytes of a row.
// Bias and what is there are added to the fp32 sums, which are rounded once.
template <typename T, int kColumns, typename Get>
__device__ __forceinline__ void write_sums(const Params& p, uint8_t* stage, int row0, int col0, int lane, Get&& get) {
  T* out = static_cast<T*>(p.out);
  constexpr int kUnit = 16 / sizeof(T);
  const bool aligned = (p.ldo & (kUnit - 1)) == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  const bool whole = aligned && row0 + 32 <= p.m && col0 + kColumns <= p.n;
  uint8_t* const my_row = stage + lane * 128;
  const int turn = lane & 7;
  const int r0 = lane >> 3, u = lane & 7;
  if (whole && p.bias == nullptr && p.accumulate == 0) {
    constexpr int kPass = 128 / sizeof(T);
    T* const at = out + int64_t(row0 + r0) * p.ldo + col0 + u * kUnit;
#pragma unroll
    for (int c0 = 0; c0 < kColumns; c0 += kPass) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint4 w;
        if constexpr (sizeof(T) == 4) {
          w = make_uint4(__float_as_uint(get(c0 + 4 * i)), __float_as_uint(get(c0 + 4 * i + 1)),
                         __float_as_uint(get(c0 + 4 * i + 2)), __float_as_uint(get(c0 + 4 * i + 3)));
        } else {
          w = make_uint4(gemm::pack2<T>(get(c0 + 8 * i), get(c0 + 8 * i + 1)), gemm::pack2<T>(get(c0 + 8 * i + 2), get(c0 + 8 * i + 3)),
                         gemm::pack2<T>(get(c0 + 8 * i + 4), get(c0 + 8 * i + 5)), gemm::pack2<T>(get(c0 + 8 * i + 6), get(c0 + 8 * i + 7)));
        }
        *reinterpret_cast<uint4*>(my_row + ((i ^ turn) << 4)) = w;
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + r0;
        *reinterpret_cast<uint4*>(at + int64_t(4 * i) * p.ldo + c0) = *reinterpret_cast<const uint4*>(stage + r * 128 + ((u ^ (r & 7)) << 4));
      }
    }
    return;
  }
  // What is there is asked for before the sums go to shared memory, eight rows at a time: one after the other, each with
  // the way to memory, they took 7.6 of the 24 us of 1531 x 1100 x 2927 added to an fp32 result.
  const bool add = p.accumulate != 0;
  const bool vec = aligned && (col0 & 3) == 0;
#pragma unroll
  for (int c0 = 0; c0 < kColumns; c0 += 32) {
    const int col = col0 + c0 + 4 * u;
    const bool inside = vec && col + 4 <= p.n;
    T* const at = out + int64_t(row0 + r0) * p.ldo + col;
    Four<T> held[8];
    if (add) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (row0 + r0 + 4 * i >= p.m) continue;
        const T* from = at + int64_t(4 * i) * p.ldo;
        if (inside) {
          held[i].load(from);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (col + j < p.n) held[i].set(j, from[j]);
        }
      }
    }
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j) bias[j] = col + j < p.n ? bias_at(p, col + j) : 0.0f;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<float4*>(my_row + ((i ^ turn) << 4)) =
          make_float4(get(c0 + 4 * i), get(c0 + 4 * i + 1), get(c0 + 4 * i + 2), get(c0 + 4 * i + 3));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + r0;
      if (row0 + r >= p.m) continue;
      const float4 v = *reinterpret_cast<const float4*>(stage + r * 128 + ((u ^ (r & 7)) << 4));
      float f[4] = {v.x + bias[0], v.y + bias[1], v.z + bias[2], v.w + bias[3]};
      if (add) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] += held[i].value(j);
      }
      T* to = at + int64_t(4 * i) * p.ldo;
      if (inside) {
        Four<T>::store(to, f);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < p.n) to[j] = from_float<T>(f[j]);
      }
    }
  }
}

// The scales that a summing warp needs: one for each of its 32 rows, and kColumnScales for its columns (0: one for all of
// them), block after block, fetched kDepth - 1 blocks ahead into a queue in shared memory that only this warp uses.  (A ring
// filled by a warp of its own, released and awaited through barriers, cost each block some 400 cycles of barrier traffic:
// 8192 x 14336 x 4096 on SM pairs took 590 us with it, 466 without any scales.)
template <int kColumnScales, int kDepth>
struct ScaleQueue {
  static_assert((kDepth & (kDepth - 1)) == 0, "a power of two");
  static constexpr int kFloats = 32 + (kColumnScales == 0 ? 4 : kColumnScales);
  static constexpr uint32_t kBytes = kDepth * kFloats * 4;

  float* slots;
  const float* row_at;         // of the next block to fetch
  const float* column_at;
  int columns_there;           // of this warp, from its first one
  bool row_there;
  uint32_t taken;              // blocks, of all tiles

  __device__ __forceinline__ explicit ScaleQueue(void* at) : slots(static_cast<float*>(at)), taken(0) {}

  // Block taken + ahead of the queue, where the tile has it.
  __device__ __forceinline__ void fetch(const Params& p, uint32_t ahead, bool more, int lane) {
    if (more) {
      float* slot = slots + ((taken + ahead) & (kDepth - 1)) * kFloats;
      copy4(slot + lane, row_at, row_there);
      if constexpr (kColumnScales == 0) {
        if (lane == 0) copy4(slot + 32, column_at, columns_there > 0);
      } else {
#pragma unroll
        for (int i = 0; i < (kColumnScales + 31) / 32; ++i) {
          const int c = 32 * i + lane;
          const bool there = c < columns_there;
          if (kColumnScales % 32 == 0 || c < kColumnScales)
            copy4(slot + 32 + c, there ? column_at + i * 32 * p.b.row_stride : p.b.base, there);
        }
      }
      if (row_there) row_at += p.a.block_stride;
      if (columns_there > 0) column_at += p.b.block_stride;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // The first of `blocks` blocks, from first_block on, of a tile whose rows and columns start at row0 and col0 for this warp.
  __device__ __forceinline__ void start(const Params& p, int row0, int col0, int first_block, int blocks, int lane) {
    const int row = row0 + lane;
    row_there = row < p.m;
    row_at = p.a.base + (row_there ? int64_t(row >> p.a.shift) * p.a.row_stride + first_block * p.a.block_stride : 0);
    columns_there = p.n - col0;
    const int column = kColumnScales == 0 ? col0 : col0 + lane;
    column_at = p.b.base + (columns_there > 0 ? int64_t(column >> p.b.shift) * p.b.row_stride + first_block * p.b.block_stride : 0);
    __syncwarp();              // nobody reads the last tile's any more
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) fetch(p, i, i < blocks, lane);
  }

  // The scales of the next block, in the order of fetching; `after` blocks of the tile follow it.  The slot of the block
  // before is fetched into.
  __device__ __forceinline__ const float* take(const Params& p, int after, int lane) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
    __syncwarp();              // every lane's copies are there, and the slot before has been read
    fetch(p, kDepth - 1, after >= kDepth - 1, lane);
    return slots + (taken++ & (kDepth - 1)) * kFloats;
  }
};

// Two floats as one register pair.
__device__ __forceinline__ uint64_t two(uint32_t lo, uint32_t hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  return v;
}
__device__ __forceinline__ float2 apart(uint64_t v) {
  uint32_t lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
  return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ void fma2(uint64_t& sum, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sum) : "l"(a), "l"(b));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

// Adds kCount accumulator columns, times their factors, to sums (in pairs).
template <int kCount, bool kRowScales>
__device__ __forceinline__ void add_columns(const uint32_t* v, uint64_t factors, const float* column_scales, uint64_t* sum) {
#pragma unroll
  for (int c = 0; c < kCount; c += 4) {
    if constexpr (kRowScales) {
      const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(column_scales + c);
      fma2(sum[c / 2], two(v[c], v[c + 1]), mul2(factors, f.x));
      fma2(sum[c / 2 + 1], two(v[c + 2], v[c + 3]), mul2(factors, f.y));
    } else {
      fma2(sum[c / 2], two(v[c], v[c + 1]), factors);
      fma2(sum[c / 2 + 1], two(v[c + 2], v[c + 3]), factors);
    }
  }
}

// Adds a block's sums, times their factors, to this lane's kColumns sums: from the accumulator at `taddr`, two loads of kChunk
// columns under way at a time.  `take` gives the block's scales while the first are; `release` is called once the
// accumulator is in registers.
template <int kColumns, int kChunk, bool kRowScales, typename Take, typename Release>
__device__ __forceinline__ void add_block(uint32_t taddr, int lane, uint64_t (&sum)[kColumns / 2], Take&& take,
                                          Release&& release) {
  constexpr bool kTwo = kColumns > kChunk;
  constexpr int kStep = kTwo ? 2 * kChunk : kChunk;
  static_assert(kColumns % kStep == 0, "whole pairs of loads");
  uint32_t v0[kChunk], v1[kTwo ? kChunk : 1];
  tmem_load<kChunk>(taddr, v0);
  if constexpr (kTwo) tmem_load<kChunk>(taddr + kChunk, v1);
  const float* slot = take();
  const float factor = kRowScales ? slot[lane] : slot[lane] * slot[32];
  const uint64_t factors = two(__float_as_uint(factor), __float_as_uint(factor));
  const float* column_scales = slot + 32;
#pragma unroll
  for (int c0 = 0; c0 < kColumns; c0 += kStep) {
    tmem_wait<kChunk>(v0);
    if constexpr (kTwo) tmem_pass<kChunk>(v1);
    const bool last = c0 + kStep == kColumns;
    if (last) release();
    add_columns<kChunk, kRowScales>(v0, factors, column_scales + c0, sum + c0 / 2);
    if (!last) tmem_load<kChunk>(taddr + c0 + kStep, v0);
    if constexpr (kTwo) {
      add_columns<kChunk, kRowScales>(v1, factors, column_scales + c0 + kChunk, sum + (c0 + kChunk) / 2);
      if (!last) tmem_load<kChunk>(taddr + c0 + kStep + kChunk, v1);
    }
  }
}

// Four neighbours of a tile's row from the sums that a cluster's CTAs hold of them, in the order of their ranks.
template <typename T>
__device__ __forceinline__ void add_parts(const Params& p, const float* part, int parts, int row, int col) {
  float4 of[kMaxParts];
#pragma unroll
  for (int q = 0; q < kMaxParts; ++q)
    if (q < parts) of[q] = peer_load4(part, q);
  float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int q = 0; q < kMaxParts; ++q)
    if (q < parts) { f[0] += of[q].x; f[1] += of[q].y; f[2] += of[q].z; f[3] += of[q].w; }
  T* at = static_cast<T*>(p.out) + int64_t(row) * p.ldo + col;
  const bool inside = col + 4 <= p.n && (reinterpret_cast<uintptr_t>(at) & (4 * sizeof(T) - 1)) == 0;
  if (inside) {
    Four<T> held;
    if (p.accumulate) held.load(at);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (p.bias != nullptr) f[j] += bias_at(p, col + j);
      if (p.accumulate) f[j] += held.value(j);
    }
    Four<T>::store(at, f);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (col + j >= p.n) continue;
    if (p.bias != nullptr) f[j] += bias_at(p, col + j);
    if (p.accumulate) f[j] += to_float<T>(at[j]);
    at[j] = from_float<T>(f[j]);
  }
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

template <bool kRowScales>
struct Shape {
  static constexpr int kColumns = kTileN / 2;                      // of a summing warp: half of the tile's
  static constexpr uint32_t kStageBytes = kABytes + kTileN * kBK;
  static constexpr int kStages = 5;
  static constexpr uint32_t kTmemCols = kAccumulators * kTileN;
  static constexpr uint32_t kStagingBytes = kSumWarps * 32 * 128;  // 128 bytes of 32 rows a warp
  static constexpr int kPartStride = kTileN + 4;                   // of a part's rows, in floats: 16-byte writes of 32 rows do not meet
  static_assert(kBM * kPartStride * 4 <= kStages * kStageBytes, "a tile's part lies where the ring was");
  using Queue = ScaleQueue<kRowScales ? kColumns : 0, kRowScales ? 4 : 8>;
  static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + kStagingBytes + kSumWarps * Queue::kBytes + 256 + 1024;
};

// Whether some scale is no power of two, as the kernel before found out.  Called by all threads of a CTA, which are as many as parts at least.
__device__ __forceinline__ bool any_odd_scale(const Params& p) {
  const bool mine = int(threadIdx.x) < p.odd_parts && __ldcg(p.odd_scales + threadIdx.x) != 0;
  return __syncthreads_or(mine) != 0;
}

// kRowScales: each row of B has scales of its own; otherwise 128 share one.  kSplit: the CTAs of a cluster share a tile, each with a
// part of the blocks, and add the parts in the order of their ranks through one another's shared memory: for products that have
// few tiles (200 x 200 x 8192 in eight parts 42.7 -> 11.4 us).  A kernel of its own, because the other lost 1 us by having both.
template <typename T, bool kRowScales, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
  using namespace gemm;
  using S = Shape<kRowScales>;
  constexpr int kStages = S::kStages;
  constexpr int kAcc = kAccumulators;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + size_t(kStages) * S::kStageBytes;
  uint8_t* queues = staging + S::kStagingBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(queues + kSumWarps * S::Queue::kBytes);   // codes of a stage are there
  uint64_t* empty_bar = full_bar + kStages;     // its MMAs are done
  uint64_t* acc_full = empty_bar + kStages;     // [kAcc] a block's sums are complete
  uint64_t* acc_empty = acc_full + kAcc;        // [kAcc] they are read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + kAcc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int total_tiles = p.tiles_m * p.tiles_n;
  // CTA `rank` of a cluster takes the blocks from first_block on of the cluster's one tile.
  const int parts = kSplit ? int(cluster_size()) : 1, rank = kSplit ? int(cluster_rank()) : 0;
  const int all_blocks = (p.k + kBK - 1) / kBK, share = (all_blocks + parts - 1) / parts;
  const int first_block = min(rank * share, all_blocks), k_blocks = min(share, all_blocks - first_block);
  const int first_tile = int(blockIdx.x) / parts, stride = int(gridDim.x) / parts;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < kAcc; ++a) {
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
  // Scales that are all powers of two have been left to the tensor cores: nothing is left to do.
  if (p.odd_scales != nullptr && !any_odd_scale(p)) total_tiles = 0;

  auto warp_wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, p.wait_ns)) != 0;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    uint32_t it = 0;
    bool ok = true;
    for (int t = first_tile; t < total_tiles && ok; t += stride) {
      int tm, tn;
      tile_at(t, p, tm, tn);
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        const int s = it % kStages;
        if (!warp_wait(&empty_bar[s], ((it / kStages) & 1u) ^ 1u)) { ok = false; break; }
        uint8_t* dst = smem + size_t(s) * S::kStageBytes;
        if (gemm2::elect_one()) {
          mbar_expect_tx(&full_bar[s], S::kStageBytes);
          tma_load_2d(dst, &map_a, &full_bar[s], (first_block + kb) * kBK, tm * kBM);
          tma_load_2d(dst + kABytes, &map_b, &full_bar[s], (first_block + kb) * kBK, tn * kTileN);
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = make_idesc(kBM, kTileN);
    uint32_t it = 0;
    bool ok = true;
    for (int t = first_tile; t < total_tiles && ok; t += stride) {
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        const int s = it % kStages;
        const uint32_t acc = it % kAcc;
        if (!warp_wait(&acc_empty[acc], ((it / kAcc) & 1u) ^ 1u)) { ok = false; break; }
        if (!warp_wait(&full_bar[s], (it / kStages) & 1u)) { ok = false; break; }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(smem + size_t(s) * S::kStageBytes);
        const uint64_t a_desc = make_smem_desc(a_addr, 16, 1024), b_desc = make_smem_desc(a_addr + kABytes, 16, 1024);
        if (gemm2::elect_one()) {
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
    const int sub = warp & 3;
    const int first_column = ((warp - 2) >> 2) * kColumns;
    uint8_t* stage_out = staging + (warp - 2) * 32 * 128;
    typename S::Queue queue(queues + (warp - 2) * S::Queue::kBytes);
    uint32_t it = 0;
    bool ok = true;
    int tm, tn;
    if (first_tile < total_tiles) {
      tile_at(first_tile, p, tm, tn);
      queue.start(p, tm * kBM + sub * 32, tn * kTileN + first_column, first_block, k_blocks, lane);
    }
    for (int t = first_tile; t < total_tiles; t += stride) {
      uint64_t sum[kColumns / 2];
#pragma unroll
      for (int c = 0; c < kColumns / 2; ++c) sum[c] = 0;
      for (int kb = 0; kb < k_blocks; ++kb, ++it) {
        const uint32_t acc = it % kAcc;
        if (!warp_wait(&acc_full[acc], (it / kAcc) & 1u)) { ok = false; break; }
        tc_fence_after();
        add_block<kColumns, 16, kRowScales>(
            tmem_base + acc * kTileN + uint32_t(first_column) + (uint32_t(sub * 32) << 16), lane, sum,
            [&] { return queue.take(p, k_blocks - 1 - kb, lane); },
            [&] {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&acc_empty[acc]);
            });
      }
      if (!ok) break;
      if constexpr (kSplit) {
        // The ring is done with: every MMA that read it has been waited for.
        float* part = reinterpret_cast<float*>(smem) + (sub * 32 + lane) * S::kPartStride + first_column;
#pragma unroll
        for (int c = 0; c < kColumns; c += 4) {
          const float2 lo = apart(sum[c / 2]), hi = apart(sum[c / 2 + 1]);
          *reinterpret_cast<float4*>(part + c) = make_float4(lo.x, lo.y, hi.x, hi.y);
        }
        break;
      } else {
        const int row0 = tm * kBM + sub * 32, col0 = tn * kTileN + first_column;
        if (t + stride < total_tiles) {   // the next tile's first scales come while this one's sums go out
          tile_at(t + stride, p, tm, tn);
          queue.start(p, tm * kBM + sub * 32, tn * kTileN + first_column, 0, k_blocks, lane);
        }
        write_sums<T, kColumns>(p, stage_out, row0, col0, lane, [&](int c) {
          const float2 f = apart(sum[c / 2]);
          return (c & 1) != 0 ? f.y : f.x;
        });
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }

  // ------------------------------------------------------------ a tile's parts
  if (kSplit && first_tile < total_tiles) {
    cluster_sync();
    int tm, tn;
    tile_at(first_tile, p, tm, tn);
    const float* part = reinterpret_cast<const float*>(smem);
    const int rows_here = kBM / parts;          // that this CTA adds and writes, four columns a thread
    const bool complete = *abort_flag == 0;
    for (int i = int(threadIdx.x); complete && i < rows_here * (kTileN / 4); i += kThreads) {
      const int row_in = rank * rows_here + i / (kTileN / 4), col_in = i % (kTileN / 4) * 4;
      const int row = tm * kBM + row_in, col = tn * kTileN + col_in;
      if (row < p.m && col < p.n) add_parts<T>(p, part + row_in * S::kPartStride + col_in, parts, row, col);
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

}  // namespace float8
}  // namespace dionw
