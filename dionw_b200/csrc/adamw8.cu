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
// seed, the step and the element's index in its tensor: the same on every replay and whatever the launch looks like, and the same
// for element i of every tensor of a call.  It has 16 bits: the probability is that of the distance, to 2^-16 below it, which leaves a
// slow average low by at most 2^-16 / (1 - beta) of a step of the format (0.015 of one for beta = 0.999).
// A second moment that is not zero is not rounded to zero: the weight's step divides by its root.
#include <cmath>
#include <type_traits>

#include "cluster.cuh"
#include "common.cuh"

namespace dionw {
namespace {

constexpr int kBlock = 128;          // elements of a scale: four for each lane of a warp
constexpr int kTable = 96;
// Threads of a CTA, CTAs of an SM and blocks of a warp, in three forms.
// Aligned: whole accesses throughout, and at least eight rounds of CTAs.  A warp with four blocks works out what a tensor's elements
//   share half as often as one with two: 39.4 M elements with fp32 gradients take 103.7 us against 105.1, 39.0 M with bf16 ones 94
//   against 98, 1051 M 2.76 ms against 2.92.  (Three blocks 110 us, five 117, four with seven CTAs 118.)
// Any: everything else.  Two blocks against four: 4.8 M elements between 16-byte boundaries 21.7 us and 23.5, 5 M aligned ones 16.2
//   and 17.1, 1 M 4.8 and 6.0, 5000 3.6 and 6.3.
// Vectors: no tensor above 4096 elements.  512 threads take a whole one and count its step themselves, which saves a launch.
struct Aligned { static constexpr int kThreads = 128, kCtas = 6, kUnroll = 4; static constexpr bool kWhole = false; };
struct Any { static constexpr int kThreads = 128, kCtas = 8, kUnroll = 2; static constexpr bool kWhole = false; };
struct Vectors { static constexpr int kThreads = 512, kCtas = 2, kUnroll = 2; static constexpr bool kWhole = true; };
template <typename Form>
constexpr int elements_of = Form::kThreads / 32 * Form::kUnroll * kBlock;
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

// The 8-bit code of x >= 0, in the top byte and without its sign: rounded down after the noise, in 2^-16 of a step, is added.
// Codes of normal numbers are the top bits of the fp32 ones; a shift brings them into the byte, and the difference of the
// exponents' biases is 0x40000000 there in both formats.  The largest value of a block may come out a little above the format's:
// the noise leaves room for 15 units in the last place below the next code.
// `noise` holds its 16 bits in the two middle bytes and 0x40 in the top one.
template <int kMantissa, int kBias>
__device__ __forceinline__ uint32_t encode_normal(float x, uint32_t noise) {
  constexpr int kUp = kMantissa + 1;   // what brings 8 bits, and the sign before them, to the top
  static_assert(((uint64_t(127 - kBias) << 23) << kUp) % (1ull << 32) == 0xC0000000u, "difference of the biases");
  return (__float_as_uint(x) << kUp) + noise;
}
// Of any x: below the smallest normal number codes are evenly spaced, and adding that number turns them into its
// mantissa.
template <int kMantissa, int kBias>
__device__ __forceinline__ uint32_t encode(float x, uint32_t noise) {
  const float normal = __uint_as_float(uint32_t(128 - kBias) << 23);
  const bool low = x < normal;
  return encode_normal<kMantissa, kBias>(low ? x + normal : x, noise) - (low ? 1u << (24 + kMantissa) : 0u);
}
// The low and the high 16 bits of a word as such noise.
__device__ __forceinline__ uint32_t low_noise(uint32_t word) { return __byte_perm(word, 0x40u, 0x4105u); }
__device__ __forceinline__ uint32_t high_noise(uint32_t word) { return __byte_perm(word, 0x40u, 0x4325u); }
// The top bytes of four words.
__device__ __forceinline__ uint32_t top_bytes(const uint32_t (&w)[4]) {
  return __byte_perm(__byte_perm(w[0], w[1], 0x0073), __byte_perm(w[2], w[3], 0x0073), 0x5410);
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

// Four gradients in the type they have: turned into floats only when all loads are under way.
template <typename G>
struct Raw {
  uint32_t w[2];
  __device__ __forceinline__ void load(const G* g) {
    const uint2 raw = __ldcs(reinterpret_cast<const uint2*>(g));
    w[0] = raw.x; w[1] = raw.y;
  }
  __device__ __forceinline__ void set(int i, G v) { w[i >> 1] |= uint32_t(*reinterpret_cast<const uint16_t*>(&v)) << (16 * (i & 1)); }
  __device__ __forceinline__ float value(int i) const {
    const uint16_t h = uint16_t(w[i >> 1] >> (16 * (i & 1)));
    return to_float<G>(*reinterpret_cast<const G*>(&h));
  }
};
template <>
struct Raw<float> {
  float f[4];
  __device__ __forceinline__ void load(const float* g) { Span<4>::load(g, f); }
  __device__ __forceinline__ void set(int i, float v) { f[i] = v; }
  __device__ __forceinline__ float value(int i) const { return f[i]; }
};

// One block of 128 elements: four for each lane.
template <typename G>
struct Piece {
  Raw<float> p;
  Raw<G> g;
  uint32_t m, v;
  float m_scale, v_scale;
};

struct Factors {
  float decay;        // lr * weight decay
  float rate;         // lr / (1 - beta1^t)
  float inv_root2;    // 1 / sqrt(1 - beta2^t)
  float eps, beta1, omb1, beta2, omb2;
};

// Updates a warp's pieces.  words(j, w) gives the noise of piece j's four elements.  Lane 2j of the warp is left with the
// scale of piece j's first moment, lane 2j + 1 with that of the second.
//
// What bounds it: the memory, as long as an element takes clearly fewer than the 85 instructions that an SM has time for at 16 bytes
// an element and 6.5 TB/s.  It takes 58 (71 with two blocks a warp), and 39.4 M elements with fp32 gradients 104 us, 6.1 TB/s.  The
// first version took 100 and 141 us: each lane worked out each scale and its reciprocal, and each code went through the form that holds for the smallest
// numbers too.  Those are now left to the pieces that have any (1 of 100 where gradients are normal), and the scales to a
// lane each.  Noise that a byte permutation puts where the code wants it, instead of a shift and a mask, was 3 us.
template <int kUnroll, typename G, typename Words>
__device__ __forceinline__ float update(Piece<G> (&x)[kUnroll], const Factors& f, int lane, Words&& words) {
  float m[kUnroll][4], v[kUnroll][4];
  float largest = 0.0f;
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    decode_mean(x[j].m, m[j]);
    decode_square(x[j].v, v[j]);
    uint32_t m_top = 0, v_top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float g = x[j].g.value(i);
      // every operation rounded by itself: two evaluations of the moments in fp32 are the same bit for bit, and a
      // difference in the last bit, rounded to the next code, would be one of a tenth in the steps to come
      m[j][i] = __fadd_rn(__fmul_rn(f.beta1, __fmul_rn(m[j][i], x[j].m_scale)), __fmul_rn(f.omb1, g));
      v[j][i] = __fadd_rn(__fmul_rn(f.beta2, __fmul_rn(v[j][i], x[j].v_scale)), __fmul_rn(f.omb2, __fmul_rn(g, g)));
      float root, inverse;
      asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(v[j][i]));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(fmaf(root, f.inv_root2, f.eps)));
      x[j].p.f[i] = fmaf(-f.rate * m[j][i], inverse, fmaf(-f.decay, x[j].p.f[i], x[j].p.f[i]));
      // as integers, magnitudes are in order, infinity and NaN above all numbers
      m_top = max(m_top, __float_as_uint(m[j][i]) & 0x7FFFFFFFu);
      v_top = max(v_top, __float_as_uint(v[j][i]));
    }
    const float m_largest = __uint_as_float(__reduce_max_sync(0xffffffffu, m_top));
    const float v_largest = __uint_as_float(__reduce_max_sync(0xffffffffu, v_top));
    if ((lane >> 1) == j) largest = (lane & 1) != 0 ? v_largest : m_largest;
  }
  const float scaled = largest * ((lane & 1) != 0 ? 1.0f / kSquareMax : 1.0f / kMeanMax);
  const float scale = scaled < INFINITY ? fmaxf(scaled, kSmallestScale) : __uint_as_float(0x7FFFFFFFu);
  const float inverse = __frcp_rn(scale);
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    const float m_inv = __shfl_sync(0xffffffffu, inverse, 2 * j), v_inv = __shfl_sync(0xffffffffu, inverse, 2 * j + 1);
    uint32_t w[4], mean[4], square[4];
    words(j, w);
    float a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = fabsf(m[j][i]) * m_inv;
      b[i] = v[j][i] * v_inv;
    }
    const bool low = fminf(fminf(a[0], a[1]), fminf(a[2], a[3])) < 0x1p-6f || fminf(fminf(b[0], b[1]), fminf(b[2], b[3])) < 0x1p-14f;
    if (!__any_sync(0xffffffffu, low)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mean[i] = encode_normal<3, 7>(a[i], low_noise(w[i]));
        square[i] = encode_normal<2, 15>(b[i], high_noise(w[i]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mean[i] = encode<3, 7>(a[i], low_noise(w[i]));
        square[i] = encode<2, 15>(b[i], high_noise(w[i]));
        if (v[j][i] > 0.0f) square[i] = max(square[i], 1u << 24);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) mean[i] = (mean[i] & 0x7FFFFFFFu) | (__float_as_uint(m[j][i]) & 0x80000000u);
    x[j].m = top_bytes(mean);
    x[j].v = top_bytes(square);
  }
  return scale;
}

// 1 - e^x for x < 0: without the cancellation near zero, and in a few instructions away from it, where the exponential's 2^-21
// at most is one of a third and less.
__device__ __forceinline__ float correction(float x) { return x < -1.0f ? 1.0f - __expf(x) : -expm1f(x); }

// Form::kWhole: a CTA takes all of a tensor, and its step has not been counted yet.
template <typename G, typename Form>
__global__ void __launch_bounds__(Form::kThreads, Form::kCtas)
adamw8_kernel(const Table tab, const Hyper hyper) {
  constexpr int kUnroll = Form::kUnroll;
  constexpr bool kWhole = Form::kWhole;
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
  const long long first = ((long long)(blockIdx.x - first_cta) * (Form::kThreads / 32) + (threadIdx.x >> 5)) * kUnroll;
  const long long n = tab.numel[lo];
  const float step = kWhole ? *tab.step[lo] + 1.0f : *tab.step[lo];
  if constexpr (kWhole) {
    __syncthreads();   // everyone has read it
    if (threadIdx.x == 0) *tab.step[lo] = step;
  }
  if (first * kBlock >= n) return;
  float* p = tab.p[lo];
  const G* g = static_cast<const G*>(tab.g[lo]);
  uint8_t* m = tab.m[lo];
  uint8_t* v = tab.v[lo];
  float* m_scale = tab.m_scale[lo];
  float* v_scale = tab.v_scale[lo];
  Factors f;
  f.decay = lr * weight_decay;
  f.rate = __fdividef(lr, correction(step * hyper.log_beta1));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(f.inv_root2) : "f"(correction(step * hyper.log_beta2)));
  f.eps = hyper.eps;
  f.beta1 = hyper.beta1;
  f.omb1 = hyper.one_minus_beta1;
  f.beta2 = hyper.beta2;
  f.omb2 = hyper.one_minus_beta2;
  const uint32_t key = step_key(step, hyper.seed);
  const bool codes_fours = ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 3u) == 0 && (first + kUnroll) * kBlock <= n;
  const bool all_fours = codes_fours && (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (reinterpret_cast<uintptr_t>(g) & (4 * sizeof(G) - 1)) == 0;
  Piece<G> x[kUnroll];
  // Whole blocks go four neighbours to a lane: in one access to each array, or, where weights or gradients lie between its
  // boundaries, codes alone so.  The last blocks of a tensor, and codes between 4-byte boundaries, go element by element: lane l
  // holds elements l, l + 32, l + 64 and l + 96 of a block, and what lies behind the tensor is zero.  The first way has a copy of
  // update() to itself: with one for all three the 39.4 M elements took 117 us instead of 105.
  // Noise of four elements, `apart` times the hash's factor from one to the next.
  auto words = [&](long long e, uint32_t apart, uint32_t (&w)[4]) {   // (a block never straddles 2^32)
    uint32_t h = uint32_t(e) * 0x9E3779B1u + (key + uint32_t(e >> 32) * 0xC2B2AE35u);
#pragma unroll
    for (int i = 0; i < 4; ++i, h += apart) w[i] = mix(h);
  };
  // lanes 2j, 2j + 1 of the warp: the scales of block first + j
  float* const scale_at = ((lane & 1) != 0 ? v_scale : m_scale) + first + (lane >> 1);
  if (all_fours) {
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const long long e = (first + j) * kBlock + 4 * lane;
      x[j].p.load(p + e);
      x[j].g.load(g + e);
      x[j].m = __ldcs(reinterpret_cast<const unsigned int*>(m + e));
      x[j].v = __ldcs(reinterpret_cast<const unsigned int*>(v + e));
      x[j].m_scale = m_scale[first + j];
      x[j].v_scale = v_scale[first + j];
    }
    const float scale = update<kUnroll>(x, f, lane, [&](int j, uint32_t (&w)[4]) { words((first + j) * kBlock + 4 * lane, 0x9E3779B1u, w); });
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const long long e = (first + j) * kBlock + 4 * lane;
      Span<4>::store(p + e, x[j].p.f);
      __stcs(reinterpret_cast<unsigned int*>(m + e), x[j].m);
      __stcs(reinterpret_cast<unsigned int*>(v + e), x[j].v);
    }
    if (lane < 2 * kUnroll) *scale_at = scale;
    return;
  }
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    x[j] = Piece<G>{};
    const long long at = (first + j) * kBlock;
    if (at >= n) continue;
    x[j].m_scale = m_scale[first + j];
    x[j].v_scale = v_scale[first + j];
    if (codes_fours) {
      const long long e = at + 4 * lane;
      x[j].m = __ldcs(reinterpret_cast<const unsigned int*>(m + e));
      x[j].v = __ldcs(reinterpret_cast<const unsigned int*>(v + e));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[j].p.set(i, p[e + i]);
        x[j].g.set(i, g[e + i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long e = at + lane + 32 * i;
        if (e >= n) continue;
        x[j].p.set(i, p[e]);
        x[j].g.set(i, g[e]);
        x[j].m |= uint32_t(m[e]) << (8 * i);
        x[j].v |= uint32_t(v[e]) << (8 * i);
      }
    }
  }
  const float scale = update<kUnroll>(x, f, lane, [&](int j, uint32_t (&w)[4]) {
    words((first + j) * kBlock + (codes_fours ? 4 * lane : lane), codes_fours ? 0x9E3779B1u : 32u * 0x9E3779B1u, w);
  });
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    const long long at = (first + j) * kBlock;
    if (codes_fours) {
      const long long e = at + 4 * lane;
#pragma unroll
      for (int i = 0; i < 4; ++i) p[e + i] = x[j].p.f[i];
      __stcs(reinterpret_cast<unsigned int*>(m + e), x[j].m);
      __stcs(reinterpret_cast<unsigned int*>(v + e), x[j].v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long e = at + lane + 32 * i;
        if (e >= n) continue;
        p[e] = x[j].p.f[i];
        m[e] = uint8_t(x[j].m >> (8 * i));
        v[e] = uint8_t(x[j].v >> (8 * i));
      }
    }
  }
  if (lane < 2 * kUnroll && (first + (lane >> 1)) * kBlock < n) *scale_at = scale;
}

// Launches one form of the kernel over the first `count` tensors of the table, or as many as a grid takes: -> `count`.
template <typename G, typename Form>
int launch(Table& tab, int& count, const Hyper& hyper, cudaStream_t stream) {
  unsigned long long ctas = 0;
  for (int i = 0; i < count; ++i) {
    const unsigned long long need =
        Form::kWhole ? 1 : (unsigned long long)((tab.numel[i] + elements_of<Form> - 1) / elements_of<Form>);
    if (ctas + need > 0x7FFFFFFFull) {
      if (i == 0) {
        set_error("adamw8_multi: a tensor of %lld elements is too large for one launch", (long long)tab.numel[i]);
        return DIONW_ERR_UNSUPPORTED;
      }
      count = i;
      break;
    }
    ctas += need;
    tab.block_end[i] = unsigned(ctas);
  }
  tab.n = count;
  if (!Form::kWhole) {
    launch_dependent(adamw8_bump_steps_kernel, 1, kTable, stream, tab);
    const int st = launch_status("adamw8_bump_steps_kernel");
    if (st != DIONW_OK || ctas == 0) return st;   // empty tensors still count the step
  }
  launch_dependent(adamw8_kernel<G, Form>, unsigned(ctas), Form::kThreads, stream, tab, hyper);
  return launch_status("adamw8_kernel");
}

template <typename G>
int launch(Table& tab, int& count, const Hyper& hyper, cudaStream_t stream) {
  bool vectors = true, aligned = true;
  long long all = 0;
  for (int i = 0; i < count; ++i) {
    all += tab.numel[i];
    vectors = vectors && tab.numel[i] <= elements_of<Vectors>;
    aligned = aligned && aligned16(tab.p[i]) && reinterpret_cast<uintptr_t>(tab.g[i]) % (4 * sizeof(G)) == 0 &&
              (reinterpret_cast<uintptr_t>(tab.m[i]) | reinterpret_cast<uintptr_t>(tab.v[i])) % 4 == 0;
  }
  if (vectors) return launch<G, Vectors>(tab, count, hyper, stream);
  aligned = aligned && all >= 8ll * sm_count() * Aligned::kCtas * elements_of<Aligned>;
  return aligned ? launch<G, Aligned>(tab, count, hyper, stream) : launch<G, Any>(tab, count, hyper, stream);
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
  DIONW_REQUIRE(n_tensors == 0 || (params && grads && exp_avg && exp_avg_sq && exp_avg_scale && exp_avg_sq_scale && steps && numels),
                "adamw8_multi: null list");
  DIONW_REQUIRE(grad_dtype >= DIONW_F32 && grad_dtype <= DIONW_BF16, "adamw8_multi: bad gradient dtype");
  DIONW_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw8_multi: betas must be in [0, 1)");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  Hyper hyper;
  hyper.lr = lr;
  hyper.weight_decay = weight_decay;
  hyper.eps = std::fmax(eps, kSmallestScale);   // of a normal number the approximate reciprocal is finite
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
    for (; start + count < n_tensors && count < kTable; ++count) {
      const int i = start + count;
      DIONW_REQUIRE(numels[i] >= 0, "adamw8_multi: tensor %d has %lld elements", i, (long long)numels[i]);
      tab.p[count] = static_cast<float*>(params[i]);
      tab.g[count] = grads[i];
      tab.m[count] = static_cast<uint8_t*>(exp_avg[i]);
      tab.v[count] = static_cast<uint8_t*>(exp_avg_sq[i]);
      tab.m_scale[count] = static_cast<float*>(exp_avg_scale[i]);
      tab.v_scale[count] = static_cast<float*>(exp_avg_sq_scale[i]);
      tab.step[count] = static_cast<float*>(steps[i]);
      tab.numel[count] = numels[i];
    }
    const int st = grad_dtype == DIONW_F32   ? launch<float>(tab, count, hyper, stream)
                   : grad_dtype == DIONW_F16 ? launch<__half>(tab, count, hyper, stream)
                                             : launch<__nv_bfloat16>(tab, count, hyper, stream);
    if (st != DIONW_OK) return st;
    start += count;
  }
  return DIONW_OK;
}
