// Matrices into e4m3 with a scale for each block of 128: 1 x 128 along the rows, or 128 x 128 tiles; with the
// transposed matrix from the same read, because a layer's backward products sum over the other side.
//
// A scale is the least power of two 2^k with max|x| <= 448 * 2^k over the block.  A power of two, because x / 2^k is
// then exact and each value is rounded once, to nearest even, in whatever order things are computed; it costs at most one
// of the format's 16 binades, and no precision.  A block of zeros has scale 1; one that holds an infinity or a NaN has the
// scale NaN, which every sum over the block then is.
//
// One CTA takes 128 x 128 elements, eight rows by eight columns for each of its 256 threads, in registers: row maxima are
// maxima over the 16 lanes of a row, column maxima over the 16 row groups go through shared memory, and so do the codes on
// their way into the transposed matrix.
#include <type_traits>

#include "cluster.cuh"
#include "common.cuh"

namespace dionw {
namespace {

constexpr int kBlock = 128;
constexpr int kThreads = 256;

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
  int rows, cols;
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

__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return uint32_t(lo) | (uint32_t(hi) << 16);
}

// Eight values of a row; those outside of the matrix are zero.
template <typename T>
__device__ __forceinline__ void load8(const QuantizeParams& p, int row, int col, float (&v)[8]) {
  const T* at = static_cast<const T*>(p.x) + int64_t(row) * p.ldx + col;
  if (p.vec && row < p.rows && col + 8 <= p.cols) {
    if constexpr (std::is_same<T, float>::value) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(at)), b = __ldg(reinterpret_cast<const float4*>(at) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(at));
      const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_float<T>(h[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = row < p.rows && col + i < p.cols ? to_float<T>(at[i]) : 0.0f;
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// A thread holds rows row0 .. row0 + 7 and columns col0 .. col0 + 7 of the CTA's tile: the 16 lanes of a half warp are
// the 128 columns of eight rows.
template <typename T, bool kTiles>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(const QuantizeParams p) {
  __shared__ uint32_t column_part[kTiles ? 1 : 16][kBlock + 4];
  __shared__ uint32_t tile_part[kThreads / 32];
  __shared__ uint2 turned[kBlock][16];     // the transposed codes: unit u of column c at u ^ (c / 8)
  after_previous();
  const int group = threadIdx.x >> 4, lane16 = threadIdx.x & 15;
  const int tile_row = int(blockIdx.y) * kBlock, tile_col = int(blockIdx.x) * kBlock;
  const int row0 = tile_row + group * 8, col0 = tile_col + lane16 * 8;
  float x[8][8];
#pragma unroll
  for (int r = 0; r < 8; ++r) load8<T>(p, row0 + r, col0, x[r]);

  uint2 codes[8];
  if constexpr (kTiles) {
    uint32_t top = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int c = 0; c < 8; ++c) top = max(top, magnitude(x[r][c]));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tile_part[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) top = max(top, tile_part[i]);
    float inverse;
    const float scale = scale_of(top, inverse);
    if (threadIdx.x == 0) {
      if (p.q != nullptr) p.scales[int64_t(blockIdx.y) * p.lds + blockIdx.x] = scale;
      if (p.qt != nullptr) p.scales_t[int64_t(blockIdx.x) * p.ldst + blockIdx.y] = scale;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int c = 0; c < 8; ++c) x[r][c] *= inverse;
  }
  if (p.q != nullptr) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      float inverse = 1.0f;
      const int row = row0 + r;
      if constexpr (!kTiles) {
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) top = max(top, magnitude(x[r][c]));
#pragma unroll
        for (int step = 8; step > 0; step >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, step));
        const float scale = scale_of(top, inverse);
        if (lane16 == 0 && row < p.rows) p.scales[int64_t(blockIdx.x) * p.lds + row] = scale;
      }
      codes[r].x = to_codes(x[r][0] * inverse, x[r][1] * inverse, x[r][2] * inverse, x[r][3] * inverse);
      codes[r].y = to_codes(x[r][4] * inverse, x[r][5] * inverse, x[r][6] * inverse, x[r][7] * inverse);
      // rows have room up to a multiple of 16 elements: codes behind the last column are zero
      if (row < p.rows && col0 < p.cols) *reinterpret_cast<uint2*>(p.q + int64_t(row) * p.ldq + col0) = codes[r];
    }
  }
  if (p.qt == nullptr) return;
  float inverse[8];
  if constexpr (!kTiles) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint32_t top = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) top = max(top, magnitude(x[r][c]));
      column_part[group][lane16 * 8 + c] = top;
    }
    __syncthreads();
    if (threadIdx.x < kBlock) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max(top, column_part[i][threadIdx.x]);
      float inv;
      const float scale = scale_of(top, inv);
      const int col = tile_col + int(threadIdx.x);
      if (col < p.cols) p.scales_t[int64_t(blockIdx.y) * p.ldst + col] = scale;
      column_part[0][threadIdx.x] = __float_as_uint(inv);   // nobody else reads or writes this column
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 8; ++c) inverse[c] = __uint_as_float(column_part[0][lane16 * 8 + c]);
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c) inverse[c] = 1.0f;
  }
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint2 column;
    column.x = to_codes(x[0][c] * inverse[c], x[1][c] * inverse[c], x[2][c] * inverse[c], x[3][c] * inverse[c]);
    column.y = to_codes(x[4][c] * inverse[c], x[5][c] * inverse[c], x[6][c] * inverse[c], x[7][c] * inverse[c]);
    turned[lane16 * 8 + c][group ^ lane16] = column;
  }
  __syncthreads();
  const int out_col = tile_row + lane16 * 8;   // of the transposed matrix
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = group + 16 * i, row = tile_col + c;
    if (row < p.cols && out_col < p.rows)
      *reinterpret_cast<uint2*>(p.qt + int64_t(row) * p.ldqt + out_col) = turned[c][lane16 ^ (c >> 3)];
  }
}

template <bool kTiles>
int launch(const QuantizeParams& p, int dtype, cudaStream_t stream) {
  const dim3 grid(unsigned((p.cols + kBlock - 1) / kBlock), unsigned((p.rows + kBlock - 1) / kBlock));
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
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
                                     float* scales_t, int64_t ldst, void* stream_ptr) {
  DIONW_REQUIRE(dtype >= DIONW_F32 && dtype <= DIONW_BF16, "float8_quantize: bad dtype");
  DIONW_REQUIRE(rows >= 0 && cols >= 0 && rows <= 0x7FFFFF80ll && cols <= 0x7FFFFF80ll, "float8_quantize: bad shape %lld x %lld",
                (long long)rows, (long long)cols);
  const int64_t row_blocks = (rows + kBlock - 1) / kBlock, col_blocks = (cols + kBlock - 1) / kBlock;
  DIONW_REQUIRE(row_blocks <= 65535, "float8_quantize: at most %d rows", 65535 * kBlock);
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
  p.rows = int(rows);
  p.cols = int(cols);
  const int64_t size = dtype == DIONW_F32 ? 4 : 2;
  p.vec = aligned16(x) && (rows == 1 || (ldx * size) % 16 == 0);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  return tiles ? launch<true>(p, dtype, stream) : launch<false>(p, dtype, stream);
}
