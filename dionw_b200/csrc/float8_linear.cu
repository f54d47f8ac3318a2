// A linear layer on the 8-bit operators: what its forward and its backward pass launch, in one call each, on matrices packed
// with their scales.  (Three calls from Python instead of one cost a layer 10 us of host time in each direction.)
#include <algorithm>

#include "cluster.cuh"
#include "common.cuh"

namespace dionw {
namespace {

constexpr int64_t kBlock = 128;

int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Codes, scales and exponents of a [rows, cols] matrix in one buffer.
struct Packed {
  int64_t rows, cols, ld, lds, scales_at, exponents_at, bytes;
  int tiles;
  Packed(int64_t rows_, int64_t cols_, int tiles_) : rows(rows_), cols(cols_), tiles(tiles_) {
    ld = up(cols, 16);
    lds = tiles ? blocks_of(cols) : rows;   // tile row after tile row, or block after block of single rows
    scales_at = up(rows * ld, 256);
    exponents_at = scales_at + up(4 * lds * (tiles ? blocks_of(rows) : blocks_of(cols)), 256);
    bytes = std::max<int64_t>(256, exponents_at + 4 * kBlock * blocks_of(rows) * blocks_of(cols));   // (never a null buffer)
  }
  void* codes(const void* base) const { return const_cast<void*>(base); }
  float* scales(const void* base) const { return reinterpret_cast<float*>(static_cast<char*>(const_cast<void*>(base)) + scales_at); }
  uint32_t* exponents(const void* base) const { return reinterpret_cast<uint32_t*>(static_cast<char*>(const_cast<void*>(base)) + exponents_at); }
};

// `x` into `straight` at `a` and its transpose into `turned` at `b`, each where there is room for it.
int quantize(const void* x, int dtype, int64_t ldx, const Packed& straight, void* a, const Packed& turned, void* b, void* stream) {
  if (a == nullptr && b == nullptr) return DIONW_OK;
  return dionw_float8_quantize(x, dtype, straight.rows, straight.cols, ldx, straight.tiles, a, straight.ld,
                               a ? straight.scales(a) : nullptr, straight.lds, b, turned.ld, b ? turned.scales(b) : nullptr,
                               turned.lds, a ? straight.exponents(a) : nullptr, b ? turned.exponents(b) : nullptr, stream);
}

int multiply(const Packed& x, const void* a, const Packed& y, const void* b, const void* bias, int bias_dtype, void* out,
             int out_dtype, void* stream) {
  return dionw_float8_product(x.codes(a), x.ld, x.scales(a), x.tiles ? x.lds : 1, x.tiles ? 1 : x.lds, x.tiles, y.codes(b), y.ld,
                              y.scales(b), y.tiles ? y.lds : 1, y.tiles ? 1 : y.lds, y.tiles, bias, bias_dtype, out, y.rows,
                              out_dtype, 0, x.rows, y.rows, x.cols, x.exponents(a), y.exponents(b), nullptr, 0, stream);
}

// ---------------------------------------------------------------------------
// sums of a matrix's columns, in fp32
// ---------------------------------------------------------------------------
// A CTA takes 32 columns: eight lanes of a warp four columns each, four rows at a time, 64 rows with its 16 warps; the 64
// partial sums of a column are added in a fixed order.  Eight rows are under way for each thread: with four, and half the
// warps, 1000 x 2304 took 12.6 us.  Bound by the few CTAs where a matrix is narrow and long: 768 columns of bf16 are 24 of them, and
// take 11.4 us for 8192 rows, 217 us (0.5 TB/s) for 65536.
constexpr int kSumColumns = 32, kSumThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kSumThreads)
column_sums_kernel(const T* __restrict__ x, int64_t ldx, int rows, int cols, int vec, float* __restrict__ out) {
  __shared__ float part[kSumThreads / 8][kSumColumns + 1];
  after_previous();
  const int group = threadIdx.x >> 3, col0 = int(blockIdx.x) * kSumColumns + (threadIdx.x & 7) * 4;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (vec && col0 + 4 <= cols) {
#pragma unroll 8
    for (int row = group; row < rows; row += kSumThreads / 8) {
      const T* at = x + int64_t(row) * ldx + col0;
      if constexpr (sizeof(T) == 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(at));
        sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
      } else {
        const uint2 raw = __ldg(reinterpret_cast<const uint2*>(at));
        const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += to_float<T>(h[i]);
      }
    }
  } else {
    for (int row = group; row < rows; row += kSumThreads / 8)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col0 + i < cols) sum[i] += to_float<T>(x[int64_t(row) * ldx + col0 + i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[group][(threadIdx.x & 7) * 4 + i] = sum[i];
  __syncthreads();
  if (threadIdx.x < kSumColumns) {
    float total = 0.0f;
#pragma unroll
    for (int g = 0; g < kSumThreads / 8; ++g) total += part[g][threadIdx.x];
    const int col = int(blockIdx.x) * kSumColumns + int(threadIdx.x);
    if (col < cols) out[col] = total;
  }
}

template <typename T>
int column_sums(const void* x, int64_t ldx, int64_t rows, int64_t cols, float* out, cudaStream_t stream) {
  const int vec = (reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T))) == 0 && ldx % 4 == 0;
  launch_dependent(column_sums_kernel<T>, unsigned((cols + kSumColumns - 1) / kSumColumns), kSumThreads, stream,
                   static_cast<const T*>(x), ldx, int(rows), int(cols), vec, out);
  return launch_status("column_sums_kernel");
}

int check_shape(const char* what, int64_t tokens, int64_t inputs, int64_t outputs) {
  DIONW_REQUIRE(tokens >= 0 && inputs >= 0 && outputs >= 0 && std::max({tokens, inputs, outputs}) <= 0x7FFFFF00ll,
                "%s: bad shape %lld x %lld x %lld", what, (long long)tokens, (long long)inputs, (long long)outputs);
  return DIONW_OK;
}

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" size_t dionw_float8_packed_bytes(int64_t rows, int64_t cols, int tiles) {
  if (rows < 0 || cols < 0) return 0;
  return size_t(Packed(rows, cols, tiles).bytes);
}

extern "C" int dionw_column_sums(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, float* out, void* stream_ptr) {
  DIONW_REQUIRE(dtype >= DIONW_F32 && dtype <= DIONW_BF16, "column_sums: bad dtype");
  DIONW_REQUIRE(rows >= 0 && cols >= 0 && rows <= 0x7FFFFF00ll && cols <= 0x7FFFFF00ll, "column_sums: bad shape %lld x %lld",
                (long long)rows, (long long)cols);
  if (cols == 0) return DIONW_OK;
  DIONW_REQUIRE(out != nullptr && (rows == 0 || (x != nullptr && ldx >= cols)), "column_sums: null operand or leading dimension %lld of %lld columns",
                (long long)ldx, (long long)cols);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  return dtype == DIONW_F32   ? column_sums<float>(x, ldx, rows, cols, out, stream)
         : dtype == DIONW_F16 ? column_sums<__half>(x, ldx, rows, cols, out, stream)
                              : column_sums<__nv_bfloat16>(x, ldx, rows, cols, out, stream);
}

extern "C" int dionw_float8_linear_forward(const void* x, int x_dtype, int64_t ldx, const void* weight, int weight_dtype,
                                           int64_t ldw, const void* bias, int bias_dtype, void* y, int64_t tokens,
                                           int64_t inputs, int64_t outputs, void* work, void* x_kept, void* weight_kept,
                                           void* stream) {
  int st = check_shape("float8_linear_forward", tokens, inputs, outputs);
  if (st != DIONW_OK) return st;
  DIONW_REQUIRE(work != nullptr && aligned16(work) && aligned16(x_kept) && aligned16(weight_kept),
                "float8_linear_forward: packed matrices need 16-byte aligned room");
  const Packed x_rows(tokens, inputs, 0), x_columns(inputs, tokens, 0);
  const Packed w_tiles(outputs, inputs, 1), w_turned(inputs, outputs, 1);
  char* w_at = static_cast<char*>(work) + x_rows.bytes;
  st = quantize(x, x_dtype, ldx, x_rows, work, x_columns, x_kept, stream);
  if (st == DIONW_OK) st = quantize(weight, weight_dtype, ldw, w_tiles, w_at, w_turned, weight_kept, stream);
  if (st == DIONW_OK) st = multiply(x_rows, work, w_tiles, w_at, bias, bias_dtype, y, x_dtype, stream);
  return st;
}

extern "C" int dionw_float8_linear_backward(const void* dy, int dy_dtype, int64_t ldy, void* dx, int dx_dtype, void* dw,
                                            int dw_dtype, float* db, int64_t tokens, int64_t inputs, int64_t outputs,
                                            void* work, const void* x_kept, const void* weight_kept, void* stream) {
  int st = check_shape("float8_linear_backward", tokens, inputs, outputs);
  if (st != DIONW_OK) return st;
  DIONW_REQUIRE((dx == nullptr || weight_kept != nullptr) && (dw == nullptr || x_kept != nullptr),
                "float8_linear_backward: a gradient without what the forward pass keeps for it");
  DIONW_REQUIRE(((dx == nullptr && dw == nullptr) || work != nullptr) && aligned16(work) && aligned16(x_kept) && aligned16(weight_kept),
                "float8_linear_backward: packed matrices need 16-byte aligned room");
  const Packed rows(tokens, outputs, 0), columns(outputs, tokens, 0);
  const Packed x_columns(inputs, tokens, 0), w_turned(inputs, outputs, 1);
  void* rows_at = dx != nullptr ? work : nullptr;
  void* columns_at = dw != nullptr ? static_cast<char*>(work) + (dx != nullptr ? rows.bytes : 0) : nullptr;
  st = quantize(dy, dy_dtype, ldy, rows, rows_at, columns, columns_at, stream);
  if (st == DIONW_OK && dx != nullptr) st = multiply(rows, rows_at, w_turned, weight_kept, nullptr, 0, dx, dx_dtype, stream);
  if (st == DIONW_OK && dw != nullptr) st = multiply(columns, columns_at, x_columns, x_kept, nullptr, 0, dw, dw_dtype, stream);
  if (st == DIONW_OK && db != nullptr) st = dionw_column_sums(dy, dy_dtype, tokens, outputs, ldy, db, stream);
  return st;
}
