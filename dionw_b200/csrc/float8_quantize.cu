// Matrices into e4m3 with a scale for each block of 128: 1 x 128 along the rows, or 128 x 128 tiles; with the
// transposed matrix from the same read, because a layer's backward products sum over the other side.
//
// A scale is the least power of two 2^k with max|x| <= 448 * 2^k over the block.  A power of two, because x / 2^k is
// then exact and each value is rounded once, to nearest even, in whatever order things are computed; it costs at most one
// of the format's 16 binades, and no precision.  A block of zeros has scale 1; one that holds an infinity or a NaN has the
// scale NaN, which every sum over the block then is.
//
// One CTA takes 128 x 128 elements, four rows by eight columns for each of its 512 threads, in registers and in the type they
// came in: row maxima are maxima over the 16 lanes of a row, column maxima over the 32 row groups go through shared
// memory, and so do the codes on their way into the transposed matrix.
//
// HBM-bound: 14336 x 4096 fp32 in tiles and both orders 61.3 us, 5.7 TB/s; 8192 x 4096 bf16 by rows 17.4 us, 5.8 TB/s.  Both orders
// of that, with a byte written for each byte read and two scales for each value, take 27.5 us, 4.9 TB/s: two thirds of the issue
// slots are taken, and three barriers a tile keep the rest from being filled.  With eight rows a thread, as fp32, an SM held 16
// warps of 104 registers: 46.8 us, and 69.6 for the tiles.  Asynchronous copies a tile ahead changed nothing (27.9), two ahead took
// 33.6.
#include <type_traits>

#include "cluster.cuh"
#include "common.cuh"

namespace dionw {
namespace {

constexpr int kBlock = 128;
constexpr int kThreads = 512;
constexpr int kRows = 4;              // of a thread

struct QuantizeParams {
  const void* x;
  int64_t ldx;
  uint8_t* q;          // nullable: [rows, ldq]
  int64_t ldq;
  uint8_t* qt;         // nullable: [cols, ldqt]
  int64_t ldqt;
  float* scales;       // rows: scale of (row, block) at block * lds + row; tiles: at row block * lds + block
  int64_t lds;
  float* scales_t;     // the same of the transposed matrix
  int64_t ldst;
  uint32_t* exponents;   // nullable: of the scales of 128 rows together, as float8_scaled_sm100.cuh wants them
  uint32_t* exponents_t;
  int rows, cols;
  int tiles_x, tiles_y, tiles;  // of 128 x 128
  int vec;             // 16-byte loads
};

// The scale's bits and the factor 1 / scale of a block whose largest magnitude has these bits.
__device__ __forceinline__ float scale_of(uint32_t largest, float& inverse) {
  if (largest == 0) {
    inverse = 1.0f;
    return 1.0f;
  }
  if (largest >= 0x7F800000u) {
    inverse = 0.0f;
    return __uint_as_float(0x7FFFFFFFu);
  }
  // 448 = 1.75 * 2^8; exponents of both 2^k and 2^-k stay those of normal numbers
  int k = int(largest >> 23) - 127 - 8 + ((largest & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  k = max(k, -126);
  inverse = __uint_as_float(uint32_t(127 - k) << 23);
  return __uint_as_float(uint32_t(127 + k) << 23);
}

// Word of row r's exponent among those of 128 rows, and the exponent with fp32's bias (NaN: 255).
__device__ __forceinline__ int exponent_at(int r) { return 4 * (r & 31) + (r >> 5); }
__device__ __forceinline__ uint32_t exponent_of(float scale) { return __float_as_uint(scale) >> 23; }

__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return uint32_t(lo) | (uint32_t(hi) << 16);
}

// Eight values of a row in the type they have, and what is done with them.  Magnitudes are compared as integers: infinity
// and NaN are above all numbers.
template <typename T>
struct Eight {
  static constexpr int kWords = 4;     // two columns each
  uint32_t w[4];
  __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0; }
  __device__ __forceinline__ void load(const T* at) {
    const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(at));
    w[0] = raw.x; w[1] = raw.y; w[2] = raw.z; w[3] = raw.w;
  }
  __device__ __forceinline__ void set(int i, T v) {
    w[i >> 1] |= uint32_t(*reinterpret_cast<const uint16_t*>(&v)) << (16 * (i & 1));
  }
  __device__ __forceinline__ uint32_t magnitude(int word) const { return w[word] & 0x7FFF7FFFu; }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  // The larger of a word's two, and one of them, as the bits of a float.
  static __device__ __forceinline__ uint32_t as_float(uint32_t half) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return half << 16;
    return __float_as_uint(__half2float(__ushort_as_half(uint16_t(half))));
  }
  static __device__ __forceinline__ uint32_t of_word(uint32_t word) { return as_float(max(word & 0xFFFFu, word >> 16)); }
  static __device__ __forceinline__ uint32_t of_column(uint32_t word, int c) { return as_float(c & 1 ? word >> 16 : word & 0xFFFFu); }
  // The word's two values, times a power of two each.
  __device__ __forceinline__ float2 scaled(int word, float fa, float fb) const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      // exact in bf16 too: what becomes too small for a normal number is far below the smallest code
      const uint32_t factors = __byte_perm(__float_as_uint(fa), __float_as_uint(fb), 0x7632);
      const __nv_bfloat162 product = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[word]),
                                             *reinterpret_cast<const __nv_bfloat162*>(&factors));
      const uint32_t bits = *reinterpret_cast<const uint32_t*>(&product);
      return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xFFFF0000u));
    }
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[word]));
    return make_float2(v.x * fa, v.y * fb);
  }
};
template <>
struct Eight<float> {
  static constexpr int kWords = 8;
  float v[8];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  }
  __device__ __forceinline__ void load(const float* at) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(at)), b = __ldcs(reinterpret_cast<const float4*>(at) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
  __device__ __forceinline__ uint32_t magnitude(int word) const { return __float_as_uint(v[word]) & 0x7FFFFFFFu; }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ uint32_t of_word(uint32_t word) { return word; }
  static __device__ __forceinline__ uint32_t of_column(uint32_t word, int) { return word; }
  __device__ __forceinline__ float2 scaled(int pair, float fa, float fb) const {
    return make_float2(v[2 * pair] * fa, v[2 * pair + 1] * fb);
  }
};

template <typename T>
__device__ __forceinline__ void load8(const QuantizeParams& p, int row, int col, Eight<T>& out) {
  const T* at = static_cast<const T*>(p.x) + int64_t(row) * p.ldx + col;
  if (p.vec && row < p.rows && col + 8 <= p.cols) {
    out.load(at);
    return;
  }
  out.clear();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (row < p.rows && col + i < p.cols) out.set(i, at[i]);
}

// A thread holds rows row0 .. row0 + 3 and columns col0 .. col0 + 7 of the CTA's tile: the 16 lanes of a half warp are
// the 128 columns of four rows.
template <typename T, bool kTiles>
__global__ void __launch_bounds__(kThreads, 2)
quantize_kernel(const QuantizeParams p) {
  constexpr int kWords = Eight<T>::kWords;
  __shared__ alignas(16) uint32_t column_part[kTiles ? 1 : 16][kTiles ? 1 : 16 * kWords];   // of a warp's eight rows
  __shared__ alignas(16) float column_inverse[kTiles ? 1 : kBlock];
  __shared__ alignas(16) uint32_t tile_part[kThreads / 32];
  __shared__ uint2 turned[kBlock][16];     // the transposed codes of eight rows: unit u of column c at u ^ (c / 8)
  after_previous();
  const int group = threadIdx.x >> 4, lane16 = threadIdx.x & 15, warp = threadIdx.x >> 5;
  Eight<T> x[kRows];
  auto load = [&](int tile) {
    const int ty = tile / p.tiles_x, row0 = ty * kBlock + group * kRows, col0 = (tile - ty * p.tiles_x) * kBlock + lane16 * 8;
#pragma unroll
    for (int r = 0; r < kRows; ++r) load8<T>(p, row0 + r, col0, x[r]);
  };
  load(blockIdx.x);
  for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
    const int ty = tile / p.tiles_x, tx = tile - ty * p.tiles_x;
    const int tile_row = ty * kBlock, tile_col = tx * kBlock;
    const int row0 = tile_row + group * kRows, col0 = tile_col + lane16 * 8;
    float inverse = 1.0f;                    // tiles: of all values
    if constexpr (kTiles) {
      uint32_t top = 0;
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < kWords; ++i) top = Eight<T>::larger(top, x[r].magnitude(i));
      top = __reduce_max_sync(0xffffffffu, Eight<T>::of_word(top));
      if ((threadIdx.x & 31) == 0) tile_part[warp] = top;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kThreads / 32; i += 4) {
        const uint4 four = *reinterpret_cast<const uint4*>(&tile_part[i]);
        top = max(top, max(max(four.x, four.y), max(four.z, four.w)));
      }
      const float scale = scale_of(top, inverse);
      if (threadIdx.x == 0) {
        if (p.q != nullptr) p.scales[int64_t(ty) * p.lds + tx] = scale;
        if (p.qt != nullptr) p.scales_t[int64_t(tx) * p.ldst + ty] = scale;
      }
      if (threadIdx.x < kBlock) {
        if (p.exponents != nullptr) p.exponents[(int64_t(tx) * p.tiles_y + ty) * kBlock + threadIdx.x] = exponent_of(scale);
        if (p.exponents_t != nullptr) p.exponents_t[(int64_t(ty) * p.tiles_x + tx) * kBlock + threadIdx.x] = exponent_of(scale);
      }
    } else if (p.qt != nullptr) {
      uint32_t top[kWords];
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        top[i] = x[0].magnitude(i);
#pragma unroll
        for (int r = 1; r < kRows; ++r) top[i] = Eight<T>::larger(top[i], x[r].magnitude(i));
        top[i] = Eight<T>::larger(top[i], __shfl_xor_sync(0xffffffffu, top[i], 16));
      }
      if ((threadIdx.x & 16) == 0) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4)
          *reinterpret_cast<uint4*>(&column_part[warp][lane16 * kWords + i]) = make_uint4(top[i], top[i + 1], top[i + 2], top[i + 3]);
      }
    }
    if (p.q != nullptr) {
      float row_inverse[kRows];
      if constexpr (!kTiles) {
        // The rows' maxima over 16 lanes; lane r of them then works out row r's scale.
        uint32_t top[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          uint32_t word = x[r].magnitude(0);
#pragma unroll
          for (int i = 1; i < kWords; ++i) word = Eight<T>::larger(word, x[r].magnitude(i));
          top[r] = word;
        }
        if constexpr (kWords == 4) {   // two rows to a word
#pragma unroll
          for (int r = 0; r < kRows; r += 2)
            top[r / 2] = __vmaxu2(__byte_perm(top[r], top[r + 1], 0x5410), __byte_perm(top[r], top[r + 1], 0x7632));
        }
        constexpr int kTops = kWords == 4 ? kRows / 2 : kRows;
#pragma unroll
        for (int step = 8; step > 0; step >>= 1)
#pragma unroll
          for (int i = 0; i < kTops; ++i) top[i] = Eight<T>::larger(top[i], __shfl_xor_sync(0xffffffffu, top[i], step));
        uint32_t mine;
        if constexpr (kWords == 4) mine = Eight<T>::of_column(lane16 & 2 ? top[1] : top[0], lane16);
        else mine = lane16 & 2 ? (lane16 & 1 ? top[3] : top[2]) : (lane16 & 1 ? top[1] : top[0]);
        float inv;
        const float scale = scale_of(mine, inv);
        if (lane16 < kRows) {
          if (row0 + lane16 < p.rows) p.scales[int64_t(tx) * p.lds + row0 + lane16] = scale;
          if (p.exponents != nullptr)
            p.exponents[(int64_t(tx) * p.tiles_y + ty) * kBlock + exponent_at(group * kRows + lane16)] = exponent_of(scale);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) row_inverse[r] = __shfl_sync(0xffffffffu, inv, r, 16);
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float f = kTiles ? inverse : row_inverse[r];
        float2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = x[r].scaled(i, f, f);
        // rows have room up to a multiple of 16 elements: codes behind the last column are zero
        if (row0 + r < p.rows && col0 < p.cols)
          *reinterpret_cast<uint2*>(p.q + int64_t(row0 + r) * p.ldq + col0) =
              make_uint2(to_codes(v[0].x, v[0].y, v[1].x, v[1].y), to_codes(v[2].x, v[2].y, v[3].x, v[3].y));
      }
    }
    if (p.qt == nullptr) {
      if (tile + int(gridDim.x) < p.tiles) load(tile + int(gridDim.x));
      if (kTiles) __syncthreads();           // the maxima are read
      continue;
    }
    if constexpr (!kTiles) {
      __syncthreads();
      if (threadIdx.x < kBlock) {
        const int c = threadIdx.x, word = kWords == 8 ? c : c >> 1;
        uint32_t top = column_part[0][word];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = Eight<T>::larger(top, column_part[i][word]);
        float inv;
        const float scale = scale_of(Eight<T>::of_column(top, c), inv);
        if (tile_col + c < p.cols) p.scales_t[int64_t(ty) * p.ldst + tile_col + c] = scale;
        if (p.exponents_t != nullptr) p.exponents_t[(int64_t(ty) * p.tiles_x + tx) * kBlock + exponent_at(c)] = exponent_of(scale);
        column_inverse[c] = inv;
      }
      __syncthreads();
    }
    float column[8];
#pragma unroll
    for (int c = 0; c < 8; c += 4) {
      if constexpr (kTiles) {
        column[c] = column[c + 1] = column[c + 2] = column[c + 3] = inverse;
      } else {
        const float4 f = *reinterpret_cast<const float4*>(&column_inverse[lane16 * 8 + c]);
        column[c] = f.x; column[c + 1] = f.y; column[c + 2] = f.z; column[c + 3] = f.w;
      }
    }
#pragma unroll
    for (int c = 0; c < 8; c += 2) {
      float2 v[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) v[r] = x[r].scaled(c / 2, column[c], column[c + 1]);
      uint32_t* unit = reinterpret_cast<uint32_t*>(&turned[lane16 * 8 + c][(group >> 1) ^ lane16]) + (group & 1);
      unit[0] = to_codes(v[0].x, v[1].x, v[2].x, v[3].x);
      unit[kBlock / 4] = to_codes(v[0].y, v[1].y, v[2].y, v[3].y);   // the next column
    }
    if (tile + int(gridDim.x) < p.tiles) load(tile + int(gridDim.x));
    __syncthreads();
    const int out_col = tile_row + lane16 * 8;   // of the transposed matrix
#pragma unroll
    for (int i = 0; i < kBlock / (kThreads / 16); ++i) {
      const int c = group + (kThreads / 16) * i, row = tile_col + c;
      if (row < p.cols && out_col < p.rows)
        *reinterpret_cast<uint2*>(p.qt + int64_t(row) * p.ldqt + out_col) = turned[c][lane16 ^ (c >> 3)];
    }
  }
}

template <bool kTiles>
int launch(const QuantizeParams& p, int dtype, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(p.tiles < 2 * sm_count() ? p.tiles : 2 * sm_count()));
  config.blockDim = dim3(kThreads);
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = use_dependent_launch() ? 1 : 0;
  auto kernel = dtype == DIONW_F32   ? quantize_kernel<float, kTiles>
                : dtype == DIONW_F16 ? quantize_kernel<__half, kTiles>
                                     : quantize_kernel<__nv_bfloat16, kTiles>;
  count_launch();
  return check_cuda(cudaLaunchKernelEx(&config, kernel, p), "quantize_kernel launch");
}

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" int dionw_float8_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int tiles,
                                     void* q, int64_t ldq, float* scales, int64_t lds, void* qt, int64_t ldqt,
                                     float* scales_t, int64_t ldst, uint32_t* exponents, uint32_t* exponents_t,
                                     void* stream_ptr) {
  DIONW_REQUIRE(dtype >= DIONW_F32 && dtype <= DIONW_BF16, "float8_quantize: bad dtype");
  DIONW_REQUIRE(rows >= 0 && cols >= 0 && rows <= 0x7FFFFF80ll && cols <= 0x7FFFFF80ll, "float8_quantize: bad shape %lld x %lld",
                (long long)rows, (long long)cols);
  const int64_t row_blocks = (rows + kBlock - 1) / kBlock, col_blocks = (cols + kBlock - 1) / kBlock;
  DIONW_REQUIRE(row_blocks * col_blocks < (1ll << 30), "float8_quantize: too large a matrix, %lld x %lld", (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return DIONW_OK;
  DIONW_REQUIRE(x != nullptr && ldx >= cols, "float8_quantize: leading dimension %lld of %lld columns", (long long)ldx,
                (long long)cols);
  DIONW_REQUIRE(q != nullptr || qt != nullptr, "float8_quantize: nothing to write");
  DIONW_REQUIRE(q == nullptr || (scales != nullptr && aligned16(q) && ldq % 16 == 0 && ldq >= cols && lds >= (tiles ? col_blocks : rows)),
                "float8_quantize: the codes need 16-byte aligned rows and a scale for each block");
  DIONW_REQUIRE(qt == nullptr || (scales_t != nullptr && aligned16(qt) && ldqt % 16 == 0 && ldqt >= rows && ldst >= (tiles ? row_blocks : cols)),
                "float8_quantize: the transposed codes need 16-byte aligned rows and a scale for each block");
  QuantizeParams p;
  p.x = x;
  p.ldx = ldx;
  p.q = static_cast<uint8_t*>(q);
  p.ldq = ldq;
  p.qt = static_cast<uint8_t*>(qt);
  p.ldqt = ldqt;
  p.scales = scales;
  p.lds = lds;
  p.scales_t = scales_t;
  p.ldst = ldst;
  p.exponents = q != nullptr ? exponents : nullptr;
  p.exponents_t = qt != nullptr ? exponents_t : nullptr;
  p.rows = int(rows);
  p.cols = int(cols);
  p.tiles_x = int(col_blocks);
  p.tiles_y = int(row_blocks);
  p.tiles = int(row_blocks * col_blocks);
  const int64_t size = dtype == DIONW_F32 ? 4 : 2;
  p.vec = aligned16(x) && (rows == 1 || (ldx * size) % 16 == 0);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  return tiles ? launch<true>(p, dtype, stream) : launch<false>(p, dtype, stream);
}
