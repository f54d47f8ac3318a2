// Host side of the 8-bit products (float8_sm100.cuh): tensor maps, tile shapes, launches.
#include <atomic>

#include "float8_pair_sm100.cuh"
#include "float8_scaled_sm100.cuh"
#include "float8_sm100.cuh"
#include "float8_tokens_sm100.cuh"
#include "products.cuh"

namespace dionw {
namespace {

constexpr int kMaxDevices = 64;

// Sets a kernel's shared memory once for each device.
template <typename Kernel>
int allow_shared(Kernel kernel, size_t smem, std::atomic<bool> (&configured)[kMaxDevices]) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) device = 0;
  if (configured[device].load(std::memory_order_acquire)) return DIONW_OK;
  DIONW_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  configured[device].store(true, std::memory_order_release);
  return DIONW_OK;
}

// In clusters of `cluster` CTAs.
template <typename Kernel, typename... Args>
int launch_in_clusters(Kernel kernel, unsigned ctas, unsigned cluster, size_t smem, int threads, const float8::Params& p,
                       cudaStream_t stream, const Args&... maps) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = cluster;
  attributes[1].val.clusterDim.y = 1;
  attributes[1].val.clusterDim.z = 1;
  // the attributes that are wanted lie together
  config.attrs = use_dependent_launch() ? attributes : attributes + 1;
  config.numAttrs = (use_dependent_launch() ? 1 : 0) + (cluster > 1 ? 1 : 0);
  count_launch();
  return check_cuda(cudaLaunchKernelEx(&config, kernel, maps..., p), "product_kernel launch");
}

// Tensor maps of the codes, where there are any.
int code_maps(CUtensorMap& map_a, CUtensorMap& map_b, const void* a, int64_t lda, uint32_t a_rows, const void* b, int64_t ldb,
              uint32_t b_rows, const float8::Params& p) {
  if (p.k == 0) return DIONW_OK;
  const int st = make_byte_map(&map_a, a, p.k, p.m, lda, float8::kBK, a_rows);
  return st != DIONW_OK ? st : make_byte_map(&map_b, b, p.k, p.n, ldb, float8::kBK, b_rows);
}

// Clusters of so many CTAs, one to an SM, that run at once.  (Of 148 SMs the driver counts 74 of two, 33 of four and 15 of eight.)
long long cluster_slots(unsigned parts) {
  return parts == 8 ? sm_count() / 8 - 3 : parts == 4 ? sm_count() / 4 - 4 : sm_count() / parts;
}

// How many CTAs share a tile: what costs least, `round` for a block that SMs go through one after the other and `join` for adding
// the parts.
struct Split {
  unsigned parts;
  long long cost;
  Split(long long tiles, long long blocks, int round, int join) : parts(1), cost(0) {
    for (unsigned p = 1; p <= unsigned(float8::kMaxParts); p *= 2) {
      const long long slots = cluster_slots(p);
      if (slots < 1) break;
      const long long c = (tiles + slots - 1) / slots * ((blocks + p - 1) / p) * round + (p > 1 ? join : 0);
      if (p == 1 || c < cost) {
        parts = p;
        cost = c;
      }
    }
  }
};

// A product of more than 64 rows whose 256 x 256 tiles would not fill the SM pairs: 128 x 128 tiles, or 256 x 128 ones of pairs where
// the tensor cores apply the scales.  Costs in 0.14 us: a block takes 0.7 us and 0.28, adding the parts 2.8.  Measured, one CTA to a
// tile and parts (us): 200 x 200 x 8192 42.7 and 11.4 (eight), 128 x 4096 x 4096 22.5 and 10.2 (four), 1000 x 768 x 2304 14.5 and 10.1
// (two), 1024^3 6.8 and 8.2 (two: it stays with one).
struct Shapes {
  Split own;
  long long scaled;
  Shapes(long long m, long long n, long long k)
      : own(((m + 127) / 128) * ((n + 127) / 128), (k + 127) / 128, 5, 20) {
    const long long pairs = sm_count() / 2, tiles = ((m + 255) / 256) * ((n + 127) / 128);
    scaled = (tiles + pairs - 1) / pairs * ((k + 127) / 128) * 2;
  }
};

// 128 x 128 tiles, each shared by `parts` CTAs.
template <typename T, bool kRowScales, bool kSplit>
int launch_single(const void* a, int64_t lda, const void* b, int64_t ldb, float8::Params p, unsigned parts, cudaStream_t stream) {
  using S = float8::Shape<kRowScales>;
  static_assert(S::kSmemBytes <= 227 * 1024, "shared memory of a CTA");
  auto kernel = float8::product_kernel<T, kRowScales, kSplit>;
  static std::atomic<bool> configured[kMaxDevices];
  int st = allow_shared(kernel, S::kSmemBytes, configured);
  CUtensorMap map_a{}, map_b{};
  if (st == DIONW_OK) st = code_maps(map_a, map_b, a, lda, float8::kBM, b, ldb, float8::kTileN, p);
  if (st != DIONW_OK) return st;
  p.tiles_m = (p.m + float8::kBM - 1) / float8::kBM;
  p.tiles_n = (p.n + float8::kTileN - 1) / float8::kTileN;
  const long long total = (long long)p.tiles_m * p.tiles_n;
  DIONW_REQUIRE(total <= 0x7FFFFFFFll, "float8_product: too many tiles");
  return launch_in_clusters(kernel, kSplit ? parts * unsigned(total) : unsigned(total < sm_count() ? total : sm_count()), parts,
                            S::kSmemBytes, float8::kThreads, p, stream, map_a, map_b);
}

// Up to kTokens rows of B, tiles of 128 rows of A.
template <typename T, int kTokens, bool kRowScales>
int launch_tokens(const void* a, int64_t lda, const void* b, int64_t ldb, float8::Params p, cudaStream_t stream) {
  using S = float8::tokens::Shape<kTokens, kRowScales>;
  static_assert(S::kSmemBytes <= 227 * 1024, "shared memory of a CTA");
  auto kernel = float8::tokens::product_kernel<T, kTokens, kRowScales>;
  static std::atomic<bool> configured[kMaxDevices];
  int st = allow_shared(kernel, S::kSmemBytes, configured);
  CUtensorMap map_a{}, map_b{};
  if (st == DIONW_OK) st = code_maps(map_a, map_b, a, lda, float8::kBM, b, ldb, kTokens, p);
  if (st != DIONW_OK) return st;
  p.tiles_m = (p.m + float8::kBM - 1) / float8::kBM;
  p.tiles_n = 1;
  // A tile's blocks are shared out by groups; adding the parts costs about as much as a group.
  const unsigned parts = Split(p.tiles_m, ((p.k + 127) / 128 + float8::tokens::kGroup - 1) / float8::tokens::kGroup, 1, 1).parts;
  const unsigned ctas = parts > 1 || p.tiles_m < sm_count() ? parts * p.tiles_m : sm_count();
  return launch_in_clusters(kernel, ctas, parts, S::kSmemBytes, float8::kThreads, p, stream, map_a, map_b);
}

// As clusters of two CTAs, one to each SM pair that has a tile.
template <typename Kernel, typename... Args>
int launch_clusters_of_two(Kernel kernel, size_t smem, int threads, const float8::Params& p, cudaStream_t stream,
                           const Args&... maps) {
  const long long total = (long long)p.tiles_m * p.tiles_n, pairs_max = sm_count() / 2;
  return launch_in_clusters(kernel, unsigned(2 * (total < pairs_max ? total : pairs_max)), 2, smem, threads, p, stream, maps...);
}

int count_pair_tiles(float8::Params& p, int tile_n) {
  p.tiles_m = (p.m + float8::pair::kPairM - 1) / float8::pair::kPairM;
  p.tiles_n = (p.n + tile_n - 1) / tile_n;
  DIONW_REQUIRE((long long)p.tiles_m * p.tiles_n <= 0x7FFFFFFFll, "float8_product: too many tiles");
  return DIONW_OK;
}

// 256 x 256 tiles on SM pairs.
template <typename T, bool kRowScales>
int launch_pairs(const void* a, int64_t lda, const void* b, int64_t ldb, float8::Params p, cudaStream_t stream) {
  namespace pair = float8::pair;
  static_assert(pair::kSmemBytes<kRowScales> <= 227 * 1024, "shared memory of a CTA");
  auto kernel = pair::product_kernel<T, kRowScales>;
  static std::atomic<bool> configured[kMaxDevices];
  int st = allow_shared(kernel, pair::kSmemBytes<kRowScales>, configured);
  if (st != DIONW_OK) return st;
  CUtensorMap map_a{}, map_b{};
  st = code_maps(map_a, map_b, a, lda, float8::kBM, b, ldb, pair::kPairN / 2, p);
  if (st != DIONW_OK) return st;
  st = count_pair_tiles(p, pair::kPairN);
  if (st != DIONW_OK) return st;
  return launch_clusters_of_two(kernel, pair::kSmemBytes<kRowScales>, pair::kThreads, p, stream, map_a, map_b);
}

// The same with exponents that the tensor cores apply.
template <typename T, int kTileN>
int launch_scaled(const void* a, int64_t lda, const void* a_exponents, const void* b, int64_t ldb, const void* b_exponents,
                  float8::Params p, cudaStream_t stream) {
  namespace scaled = float8::scaled;
  static_assert(scaled::Shape<kTileN>::kSmemBytes <= 227 * 1024, "shared memory of a CTA");
  auto kernel = scaled::product_kernel<T, kTileN>;
  static std::atomic<bool> configured[kMaxDevices];
  int st = allow_shared(kernel, scaled::Shape<kTileN>::kSmemBytes, configured);
  if (st != DIONW_OK) return st;
  scaled::Maps maps;
  const int64_t blocks = (p.k + 127) / 128;
  st = make_byte_map(&maps.a, a, p.k, p.m, lda, float8::kBK, float8::kBM);
  if (st == DIONW_OK) st = make_byte_map(&maps.b, b, p.k, p.n, ldb, float8::kBK, kTileN / 2);
  if (st == DIONW_OK) st = make_word_map(&maps.a_scales, a_exponents, blocks * ((p.m + 127) / 128), 1);
  if (st == DIONW_OK) st = make_word_map(&maps.b_scales, b_exponents, blocks * ((p.n + 127) / 128), kTileN / 128);
  if (st == DIONW_OK) st = count_pair_tiles(p, kTileN);
  if (st != DIONW_OK) return st;
  return launch_clusters_of_two(kernel, scaled::Shape<kTileN>::kSmemBytes, scaled::kThreads, p, stream, maps);
}

// ---------------------------------------------------------------------------
// exponents of scales of any strides
// ---------------------------------------------------------------------------
constexpr int kExponentThreads = 256, kExponentCtas = 296;

struct ExponentJob {
  float8::Scales scales;
  uint32_t* out;
  int rows, atoms;         // 128 rows of a block are an atom
  long long all;           // blocks * atoms
};

// The exponents of both operands' scales, and one word a CTA that says whether one of its scales is neither a power of two nor
// NaN.  A warp takes an atom: lane l reads the scales of rows l, 32 + l, 64 + l and 96 + l and writes them as words 4 l .. 4 l + 3;
// rows behind the matrix get 1.
__global__ void __launch_bounds__(kExponentThreads)
exponents_kernel(const ExponentJob a, const ExponentJob b, int* odd) {
  after_previous();
  const int lane = threadIdx.x & 31;
  bool mine = false;
  for (long long i = ((long long)blockIdx.x * kExponentThreads + threadIdx.x) >> 5; i < a.all + b.all;
       i += ((long long)gridDim.x * kExponentThreads) >> 5) {
    const bool second = i >= a.all;
    const ExponentJob& job = second ? b : a;
    const long long atom = second ? i - a.all : i, block = atom / job.atoms;
    const long long row0 = (atom - block * job.atoms) * 128 + lane;
    const float* base = job.scales.base + block * job.scales.block_stride;
    uint32_t bits[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const long long row = row0 + 32 * c;
      bits[c] = row < job.rows ? __float_as_uint(base[(row >> job.scales.shift) * job.scales.row_stride]) : 0x3F800000u;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bool nan = (bits[c] & 0x7FFFFFFFu) > 0x7F800000u;
      const uint32_t exponent = (bits[c] >> 23) & 0xFFu;
      mine = mine || (!nan && ((bits[c] & 0x807FFFFFu) != 0 || exponent == 0 || exponent == 255));
      bits[c] = exponent;
    }
    reinterpret_cast<uint4*>(job.out)[atom * 32 + lane] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
  }
  const int any = __syncthreads_or(mine);
  if (threadIdx.x == 0) odd[blockIdx.x] = any;
}

long long pair_tiles(long long m, long long n) { return ((m + 255) / 256) * ((n + 255) / 256); }

bool wide(long long m, long long n) { return pair_tiles(m, n) >= sm_count() / 2; }

// Whether a product looks at its scales, to leave them to the tensor cores where they are powers of two; the two launches more cost 5
// us.  Measured, own sums against looking first (us): 1000 x 2304 x 768 7.2 and 10.7, 1000 x 768 x 2304 10.1 and 12.8, 1024 x 1024 x 4096
// 14.0 and 16.2, 1531 x 1100 x 2927 25.3 and 18.1, 2048^3 20.3 and 17.8, 512 x 4096 x 14336 54 and 40.  256 x 256 tiles: from 18 blocks
// of 128 x 128 on that SMs would go through one after the other.
bool takes_exponents(long long m, long long n, long long k) {
  if (m <= 64) return false;
  if (wide(m, n)) return (((m + 127) / 128) * ((n + 127) / 128) + sm_count() - 1) / sm_count() * ((k + 127) / 128) >= 18;
  const Shapes shapes(m, n, k);
  return shapes.scaled + 36 < shapes.own.cost;
}

// Whether a product that is given its exponents uses them: unless it has so few tiles that parts of them, with sums of its own, are
// faster.  Measured, own sums against tensor cores (us): 65 x 256 x 4096 8.2 and 12.3, 200 x 200 x 8192 11.4 and 21.2, 128 x 4096 x 4096
// 12.5 and 13.1, 256 x 2048 x 2048 9.7 and 7.9, 512 x 2048 x 4096 17.2 and 12.8, 128 x 1024 x 1024 7.7 and 6.3.
bool prefers_exponents(long long m, long long n, long long k) {
  if (m <= 64) return false;
  if (wide(m, n)) return true;
  const Shapes shapes(m, n, k);
  return shapes.scaled <= shapes.own.cost;
}

// Scratch of a product whose scales are looked at: a word a CTA, and both operands' exponents.
struct ExponentRoom {
  size_t a_at, b_at, bytes;
  ExponentRoom(long long m, long long n, long long k) {
    const long long blocks = (k + 127) / 128;
    a_at = (4 * kExponentCtas + 511) / 512 * 512;
    b_at = a_at + 512 * size_t(blocks * ((m + 127) / 128));
    bytes = b_at + 512 * size_t(blocks * ((n + 127) / 128));
  }
};

template <typename T>
int run_scaled(const void* a, int64_t lda, const void* ea, const void* b, int64_t ldb, const void* eb, const float8::Params& p,
               cudaStream_t stream) {
  if (wide(p.m, p.n)) return launch_scaled<T, 256>(a, lda, ea, b, ldb, eb, p, stream);
  return launch_scaled<T, 128>(a, lda, ea, b, ldb, eb, p, stream);
}

// The kernel for a product of this shape.
template <typename T>
int run(const void* a, int64_t lda, const void* b, int64_t ldb, float8::Params p, cudaStream_t stream) {
  const int m = p.m;
  if (m <= 64) {
    // A few tokens: the weights are the 128 rows of a tile.
    std::swap(p.a, p.b);
    std::swap(p.m, p.n);
    auto launch = [&](auto row_scales) {
      constexpr bool kRowScales = decltype(row_scales)::value;
      if (m <= 16) return launch_tokens<T, 16, kRowScales>(b, ldb, a, lda, p, stream);
      if (m <= 32) return launch_tokens<T, 32, kRowScales>(b, ldb, a, lda, p, stream);
      return launch_tokens<T, 64, kRowScales>(b, ldb, a, lda, p, stream);
    };
    return p.b.shift == 0 ? launch(std::true_type()) : launch(std::false_type());
  }
  if (wide(p.m, p.n))
    return p.b.shift != 0 ? launch_pairs<T, false>(a, lda, b, ldb, p, stream) : launch_pairs<T, true>(a, lda, b, ldb, p, stream);
  const unsigned parts = Shapes(p.m, p.n, p.k).own.parts;
  if (parts > 1)
    return p.b.shift != 0 ? launch_single<T, false, true>(a, lda, b, ldb, p, parts, stream)
                          : launch_single<T, true, true>(a, lda, b, ldb, p, parts, stream);
  return p.b.shift != 0 ? launch_single<T, false, false>(a, lda, b, ldb, p, 1, stream)
                        : launch_single<T, true, false>(a, lda, b, ldb, p, 1, stream);
}

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" size_t dionw_float8_product_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || !takes_exponents(m, n, k)) return 0;
  return ExponentRoom(m, n, k).bytes;
}

extern "C" int dionw_float8_product(const void* a, int64_t lda, const float* a_scales, int64_t a_row_stride,
                                    int64_t a_block_stride, int a_tiles, const void* b, int64_t ldb,
                                    const float* b_scales, int64_t b_row_stride, int64_t b_block_stride, int b_tiles,
                                    const void* bias, int bias_dtype, void* out, int64_t ldo, int out_dtype,
                                    int accumulate, int64_t m, int64_t n, int64_t k, const uint32_t* a_exponents,
                                    const uint32_t* b_exponents, void* workspace, size_t workspace_bytes,
                                    void* stream_ptr) {
  DIONW_REQUIRE(m >= 0 && n >= 0 && k >= 0 && m <= 0x7FFFFF00ll && n <= 0x7FFFFF00ll && k <= 0x7FFFFF00ll,
                "float8_product: bad shape %lld x %lld x %lld", (long long)m, (long long)n, (long long)k);
  DIONW_REQUIRE(out_dtype >= DIONW_F32 && out_dtype <= DIONW_BF16, "float8_product: bad output dtype");
  DIONW_REQUIRE(bias == nullptr || (bias_dtype >= DIONW_F32 && bias_dtype <= DIONW_BF16), "float8_product: bad bias dtype");
  DIONW_REQUIRE((a_exponents == nullptr) == (b_exponents == nullptr), "float8_product: exponents of one operand only");
  if (m == 0 || n == 0) return DIONW_OK;
  DIONW_REQUIRE(out != nullptr && ldo >= n, "float8_product: leading dimension %lld of %lld columns", (long long)ldo,
                (long long)n);
  if (k > 0) {
    DIONW_REQUIRE(a != nullptr && b != nullptr && a_scales != nullptr && b_scales != nullptr, "float8_product: null operand");
    DIONW_REQUIRE(aligned16(a) && aligned16(b) && (lda % 16 == 0 || m == 1) && (ldb % 16 == 0 || n == 1) && lda >= k && ldb >= k,
                  "float8_product: rows of codes must start on 16-byte boundaries (leading dimensions %lld, %lld)",
                  (long long)lda, (long long)ldb);
  }
  float8::Params p{};
  p.a = {a_scales, a_row_stride, a_block_stride, a_tiles ? 7 : 0};
  p.b = {b_scales, b_row_stride, b_block_stride, b_tiles ? 7 : 0};
  p.out = out;
  p.ldo = ldo;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.accumulate = accumulate;
  p.m = int(m);
  p.n = int(n);
  p.k = int(k);
  p.status = device_status_word();
  p.wait_ns = gemm::kWaitLimitNs;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  auto scaled = [&](const uint32_t* ea, const uint32_t* eb) {
    if (out_dtype == DIONW_F32) return run_scaled<float>(a, lda, ea, b, ldb, eb, p, stream);
    if (out_dtype == DIONW_F16) return run_scaled<__half>(a, lda, ea, b, ldb, eb, p, stream);
    return run_scaled<__nv_bfloat16>(a, lda, ea, b, ldb, eb, p, stream);
  };
  if (a_exponents != nullptr && b_exponents != nullptr) {
    DIONW_REQUIRE(aligned16(a_exponents) && aligned16(b_exponents), "float8_product: exponents must be 16-byte aligned");
    if (k > 0 && prefers_exponents(m, n, k)) return scaled(a_exponents, b_exponents);
  } else if (takes_exponents(m, n, k)) {
    const ExponentRoom room(m, n, k);
    if (workspace != nullptr) {
      DIONW_REQUIRE(aligned16(workspace), "float8_product: the workspace must be 16-byte aligned");
      if (workspace_bytes < room.bytes) {
        set_error("float8_product: workspace of %zu bytes, %zu needed", workspace_bytes, room.bytes);
        return DIONW_ERR_WORKSPACE;
      }
      // Three launches: what the scales are, the product if they are powers of two, the product if they are not.  The one that has
      // nothing to do costs 2 to 3 us of some hundred.
      char* base = static_cast<char*>(workspace);
      const long long blocks = (k + 127) / 128;
      ExponentJob ja{p.a, reinterpret_cast<uint32_t*>(base + room.a_at), int(m), int((m + 127) / 128), 0};
      ExponentJob jb{p.b, reinterpret_cast<uint32_t*>(base + room.b_at), int(n), int((n + 127) / 128), 0};
      ja.all = blocks * ja.atoms;
      jb.all = blocks * jb.atoms;
      const long long ctas = (32 * (ja.all + jb.all) + kExponentThreads - 1) / kExponentThreads;
      p.odd_scales = static_cast<const int*>(workspace);
      p.odd_parts = int(ctas < kExponentCtas ? ctas : kExponentCtas);
      launch_dependent(exponents_kernel, unsigned(p.odd_parts), kExponentThreads, stream, ja, jb, static_cast<int*>(workspace));
      int st = launch_status("exponents_kernel");
      if (st == DIONW_OK) st = scaled(ja.out, jb.out);
      if (st != DIONW_OK) return st;
    }
  }
  if (out_dtype == DIONW_F32) return run<float>(a, lda, b, ldb, p, stream);
  if (out_dtype == DIONW_F16) return run<__half>(a, lda, b, ldb, p, stream);
  return run<__nv_bfloat16>(a, lda, b, ldb, p, stream);
}
