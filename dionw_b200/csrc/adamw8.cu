// AdamW with moments held in 8 bits: one step over many tensors.
//
// Every 128 consecutive elements of a tensor are a block.  The first moment is e4m3 times the block's fp32 scale
// max|m| / 448, the second e5m2 times max(v) / 57344: the largest value of a block has the largest code.  e5m2 for
// the second because it is a square: 57344 / 2^-16 = 2^32 between the largest and the smallest code of a block are
// 2^16 between gradients.  Moments are updated in fp32 from what the codes stand for, the weight from those fp32
// moments; only what is kept for the next step is rounded.
//
// That rounding is stochastic: to the code below or above, with the probability of the distance to the other.  An
// average moves by (1 - beta) of its distance per step; where that is less than half a step of the format (6 to 12 % of
// the value in e4m3, 12 to 25 % in e5m2), rounding to nearest would keep it where it is for ever.  Its noise is a hash of the
// seed, the step and the element's index in its tensor: the same on every replay and whatever the launch looks
// like.  A second moment that is not zero is not rounded to zero: the weight's step divides by its root.
#include <cmath>
#include <type_traits>

#include "cluster.cuh"
#include "common.cuh"

namespace dionw {
namespace {

constexpr int kBlock = 128;          // elements of a scale: four for each lane of a warp
constexpr int kTable = 96;
constexpr int kThreads = 256;
constexpr int kUnroll = 2;           // blocks of a warp
constexpr int kChunk = kThreads / 32 * kUnroll * kBlock;   // elements per CTA
constexpr float kMeanMax = 448.0f, kSquareMax = 57344.0f;
constexpr float kSmallestScale = 1.17549435e-38f;          // 2^-126: its reciprocal is finite

struct Table {
  float* p[kTable];
  const void* g[kTable];
  uint8_t* m[kTable];
  uint8_t* v[kTable];
  float* m_scale[kTable];
  float* v_scale[kTable];
  float* step[kTable];
  long long numel[kTable];
  unsigned block_end[kTable];
  int n;
};

struct Hyper {
  float lr, weight_decay, eps;
  float beta1, one_minus_beta1, log_beta1;
  float beta2, one_minus_beta2, log_beta2;
  uint32_t seed;
  const float* device;   // nullable: {lr, weight decay} in device memory instead
};

__global__ void adamw8_bump_steps_kernel(const Table tab) {
  after_previous();
  const int i = threadIdx.x;
  if (i < tab.n) *tab.step[i] += 1.0f;
}

// What all elements of a tensor share in this step.
__device__ __forceinline__ uint32_t step_key(float step, uint32_t seed) {
  uint32_t key = uint32_t(step) * 0x9E3779B9u + seed;
  key = (key ^ (key >> 16)) * 0x85EBCA6Bu;
  return key ^ (key >> 13);
}
__device__ __forceinline__ uint32_t mix(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x7FEB352Du;
  return h ^ (h >> 15);
}

// The 8-bit code, without its sign, of x >= 0: rounded down after `noise` / 2^16 of a step is added.  Codes of normal
// numbers are the top bits of the fp32 ones.  Below the smallest normal number they are evenly spaced; adding that
// number turns them into its mantissa.
template <int kMantissa, int kBias, int kMost>
__device__ __forceinline__ uint32_t encode(float x, uint32_t noise) {
  constexpr int kDrop = 23 - kMantissa, kFirst = (127 - kBias) << kMantissa;
  const float normal = __uint_as_float(uint32_t(128 - kBias) << 23);
  const bool low = x < normal;
  const uint32_t bits = __float_as_uint(low ? x + normal : x) + (noise << (kDrop - 16));
  return uint32_t(min(int(bits >> kDrop) - (low ? kFirst + (1 << kMantissa) : kFirst), kMost));
}

__device__ __forceinline__ float2 halves(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Four e4m3 codes, and four e5m2 codes (the top byte of the fp16 number of the same value).
__device__ __forceinline__ void decode_mean(uint32_t codes, float (&out)[4]) {
  uint32_t lo, hi;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi) : "r"(codes));
  const float2 a = halves(lo), b = halves(hi);
  out[0] = a.x; out[1] = a.y; out[2] = b.x; out[3] = b.y;
}
__device__ __forceinline__ void decode_square(uint32_t codes, float (&out)[4]) {
  const float2 a = halves(__byte_perm(codes, 0, 0x1404)), b = halves(__byte_perm(codes, 0, 0x3424));
  out[0] = a.x; out[1] = a.y; out[2] = b.x; out[3] = b.y;
}

template <typename G>
__device__ __forceinline__ void load_gradient(const G* g, float (&out)[4]) {
  if constexpr (std::is_same<G, float>::value) {
    Span<4>::load(g, out);
  } else {
    const uint2 raw = __ldcs(reinterpret_cast<const uint2*>(g));
    const G* h = reinterpret_cast<const G*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = to_float<G>(h[i]);
  }
}

// One block of 128 elements: four for each lane.
struct Piece {
  float p[4], g[4];
  uint32_t m, v;
  float m_scale, v_scale;
};

struct Factors {
  float keep;         // 1 - lr * weight decay, as the factor that is subtracted: lr * weight decay
  float rate;         // lr / (1 - beta1^t)
  float inv_root2;    // 1 / sqrt(1 - beta2^t)
  float eps, beta1, omb1, beta2, omb2;
};

// Updates a piece; `words` are the four elements' noise.
__device__ __forceinline__ void update(Piece& x, const Factors& f, const uint32_t (&words)[4]) {
  float m[4], v[4];
  decode_mean(x.m, m);
  decode_square(x.v, v);
  uint32_t m_top = 0, v_top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float g = x.g[i];
    // every operation rounded by itself: two evaluations of the moments in fp32 are the same bit for bit, and a
    // difference in the last bit, rounded to the next code, would be one of a tenth in the steps to come
    m[i] = __fadd_rn(__fmul_rn(f.beta1, __fmul_rn(m[i], x.m_scale)), __fmul_rn(f.omb1, g));
    v[i] = __fadd_rn(__fmul_rn(f.beta2, __fmul_rn(v[i], x.v_scale)), __fmul_rn(f.omb2, __fmul_rn(g, g)));
    float root;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v[i]));
    x.p[i] = fmaf(-f.keep, x.p[i], x.p[i]) - __fdividef(f.rate * m[i], fmaf(root, f.inv_root2, f.eps));
    // as integers, magnitudes are in order, infinity and NaN above all numbers
    m_top = max(m_top, __float_as_uint(m[i]) & 0x7FFFFFFFu);
    v_top = max(v_top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  }
  const float m_largest = __uint_as_float(__reduce_max_sync(0xffffffffu, m_top));
  const float v_largest = __uint_as_float(__reduce_max_sync(0xffffffffu, v_top));
  const float nan = __uint_as_float(0x7FFFFFFFu);
  x.m_scale = m_largest < INFINITY ? fmaxf(m_largest * (1.0f / kMeanMax), kSmallestScale) : nan;
  x.v_scale = v_largest < INFINITY ? fmaxf(v_largest * (1.0f / kSquareMax), kSmallestScale) : nan;
  const float m_inv = __frcp_rn(x.m_scale), v_inv = __frcp_rn(x.v_scale);
  x.m = x.v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t mean = encode<3, 7, 0x7E>(fabsf(m[i]) * m_inv, words[i] & 0xFFFFu) | ((__float_as_uint(m[i]) >> 24) & 0x80u);
    uint32_t square = encode<2, 15, 0x7B>(v[i] * v_inv, words[i] >> 16);
    if (v[i] > 0.0f) square = max(square, 1u);
    x.m |= mean << (8 * i);
    x.v |= square << (8 * i);
  }
}

template <typename G>
__global__ void __launch_bounds__(kThreads, 4)
adamw8_kernel(const Table tab, const Hyper hyper) {
  after_previous();
  const float lr = hyper.device != nullptr ? hyper.device[0] : hyper.lr;
  const float weight_decay = hyper.device != nullptr ? hyper.device[1] : hyper.weight_decay;
  int lo = 0, hi = tab.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (blockIdx.x < tab.block_end[mid]) hi = mid; else lo = mid + 1;
  }
  const unsigned first_cta = lo == 0 ? 0u : tab.block_end[lo - 1];
  const int lane = threadIdx.x & 31;
  const long long first = ((long long)(blockIdx.x - first_cta) * (kThreads / 32) + (threadIdx.x >> 5)) * kUnroll;
  const long long n = tab.numel[lo];
  if (first * kBlock >= n) return;
  float* p = tab.p[lo];
  const G* g = static_cast<const G*>(tab.g[lo]);
  uint8_t* m = tab.m[lo];
  uint8_t* v = tab.v[lo];
  float* m_scale = tab.m_scale[lo];
  float* v_scale = tab.v_scale[lo];
  const float step = *tab.step[lo];
  // 1 - beta^t without the cancellation of its first steps
  Factors f;
  f.keep = lr * weight_decay;
  f.rate = lr / -expm1f(step * hyper.log_beta1);
  f.inv_root2 = rsqrtf(-expm1f(step * hyper.log_beta2));
  f.eps = hyper.eps;
  f.beta1 = hyper.beta1;
  f.omb1 = hyper.one_minus_beta1;
  f.beta2 = hyper.beta2;
  f.omb2 = hyper.one_minus_beta2;
  const uint32_t key = step_key(step, hyper.seed);
  const bool vec = ((reinterpret_cast<uintptr_t>(p) | (reinterpret_cast<uintptr_t>(g) * (4 / sizeof(G)))) & 15u) == 0 &&
                   ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 3u) == 0;
  auto words_of = [&](long long e, uint32_t (&words)[4]) {
    uint32_t h = uint32_t(e) * 0x9E3779B1u + (key + uint32_t(e >> 32) * 0xC2B2AE35u);
#pragma unroll
    for (int i = 0; i < 4; ++i, h += 0x9E3779B1u) words[i] = mix(h);   // four elements never straddle 2^32
  };
  Piece x[kUnroll];
  if (vec && (first + kUnroll) * kBlock <= n) {
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const long long e = (first + j) * kBlock + 4 * lane;
      Span<4>::load(p + e, x[j].p);
      load_gradient<G>(g + e, x[j].g);
      x[j].m = __ldcs(reinterpret_cast<const unsigned int*>(m + e));
      x[j].v = __ldcs(reinterpret_cast<const unsigned int*>(v + e));
      x[j].m_scale = m_scale[first + j];
      x[j].v_scale = v_scale[first + j];
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const long long e = (first + j) * kBlock + 4 * lane;
      uint32_t words[4];
      words_of(e, words);
      update(x[j], f, words);
      Span<4>::store(p + e, x[j].p);
      __stcs(reinterpret_cast<unsigned int*>(m + e), x[j].m);
      __stcs(reinterpret_cast<unsigned int*>(v + e), x[j].v);
      if (lane == 0) {
        m_scale[first + j] = x[j].m_scale;
        v_scale[first + j] = x[j].v_scale;
      }
    }
    return;
  }
  // Tensors between 16-byte boundaries, and the last blocks: element by element.
  for (int j = 0; j < kUnroll && (first + j) * kBlock < n; ++j) {
    Piece y{};
    const long long at = (first + j) * kBlock;
    // lane l holds elements l, l + 32, l + 64, l + 96, so that neighbours read neighbours
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long e = at + lane + 32 * i;
      if (e >= n) continue;
      y.p[i] = p[e];
      y.g[i] = to_float<G>(g[e]);
      y.m |= uint32_t(m[e]) << (8 * i);
      y.v |= uint32_t(v[e]) << (8 * i);
    }
    y.m_scale = m_scale[first + j];
    y.v_scale = v_scale[first + j];
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long e = at + lane + 32 * i;
      words[i] = mix(uint32_t(e) * 0x9E3779B1u + (key + uint32_t(e >> 32) * 0xC2B2AE35u));
    }
    update(y, f, words);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long e = at + lane + 32 * i;
      if (e >= n) continue;
      p[e] = y.p[i];
      m[e] = uint8_t(y.m >> (8 * i));
      v[e] = uint8_t(y.v >> (8 * i));
    }
    if (lane == 0) {
      m_scale[first + j] = y.m_scale;
      v_scale[first + j] = y.v_scale;
    }
  }
}

template <typename G>
int launch(const Table& tab, unsigned ctas, const Hyper& hyper, cudaStream_t stream) {
  launch_dependent(adamw8_bump_steps_kernel, 1, kTable, stream, tab);
  const int st = launch_status("adamw8_bump_steps_kernel");
  if (st != DIONW_OK) return st;
  launch_dependent(adamw8_kernel<G>, ctas, kThreads, stream, tab, hyper);
  return launch_status("adamw8_kernel");
}

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" int dionw_adamw8_multi(void* const* params, const void* const* grads, int grad_dtype, void* const* exp_avg,
                                  void* const* exp_avg_sq, void* const* exp_avg_scale, void* const* exp_avg_sq_scale,
                                  void* const* steps, const int64_t* numels, int n_tensors, float lr, double beta1,
                                  double beta2, float weight_decay, float eps, uint32_t seed,
                                  const float* hyper_device, void* stream_ptr) {
  DIONW_REQUIRE(n_tensors >= 0, "adamw8_multi: negative tensor count");
  DIONW_REQUIRE(grad_dtype >= DIONW_F32 && grad_dtype <= DIONW_BF16, "adamw8_multi: bad gradient dtype");
  DIONW_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw8_multi: betas must be in [0, 1)");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  Hyper hyper;
  hyper.lr = lr;
  hyper.weight_decay = weight_decay;
  hyper.eps = eps;
  hyper.beta1 = float(beta1);
  hyper.one_minus_beta1 = float(1.0 - beta1);
  hyper.log_beta1 = float(std::log(beta1));
  hyper.beta2 = float(beta2);
  hyper.one_minus_beta2 = float(1.0 - beta2);
  hyper.log_beta2 = float(std::log(beta2));
  hyper.seed = seed;
  hyper.device = hyper_device;
  for (int start = 0; start < n_tensors;) {
    Table tab;
    int count = 0;
    unsigned long long ctas = 0;
    for (; start + count < n_tensors && count < kTable; ++count) {
      const int i = start + count;
      DIONW_REQUIRE(numels[i] >= 0, "adamw8_multi: tensor %d has %lld elements", i, (long long)numels[i]);
      const unsigned long long need = (unsigned long long)((numels[i] + kChunk - 1) / kChunk);
      if (ctas + need > 0x7FFFFFFFull) break;
      ctas += need;
      tab.p[count] = static_cast<float*>(params[i]);
      tab.g[count] = grads[i];
      tab.m[count] = static_cast<uint8_t*>(exp_avg[i]);
      tab.v[count] = static_cast<uint8_t*>(exp_avg_sq[i]);
      tab.m_scale[count] = static_cast<float*>(exp_avg_scale[i]);
      tab.v_scale[count] = static_cast<float*>(exp_avg_sq_scale[i]);
      tab.step[count] = static_cast<float*>(steps[i]);
      tab.numel[count] = numels[i];
      tab.block_end[count] = unsigned(ctas);
    }
    if (count == 0) {
      set_error("adamw8_multi: a tensor of %lld elements is too large for one launch", (long long)numels[start]);
      return DIONW_ERR_UNSUPPORTED;
    }
    tab.n = count;
    start += count;
    if (ctas == 0) {   // empty tensors still count the step
      launch_dependent(adamw8_bump_steps_kernel, 1, kTable, stream, tab);
      const int st = launch_status("adamw8_bump_steps_kernel");
      if (st != DIONW_OK) return st;
      continue;
    }
    const int st = grad_dtype == DIONW_F32   ? launch<float>(tab, unsigned(ctas), hyper, stream)
                   : grad_dtype == DIONW_F16 ? launch<__half>(tab, unsigned(ctas), hyper, stream)
                                             : launch<__nv_bfloat16>(tab, unsigned(ctas), hyper, stream);
    if (st != DIONW_OK) return st;
  }
  return DIONW_OK;
}
