// The AdamW step over a list of tensors, with moments in 32 or in 8 bits.
//
//   g' = g min(1, max_norm / (norm + 1e-6)),  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - rate decay) - rate / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8 bits: a block of 256 values of a tensor shares a power of two, twice the largest value's, and a
// value over it is 3 bits behind the point with a sign and 4 bits of exponent (m) or 5 bits of
// exponent (v, never negative); below 2^-14 or 2^-30 the steps stay as they are.  A step is 6 to 12 %
// of a value, while v moves by 0.1 % a call: rounded to the nearest it would never move.  So a value
// is rounded up with the probability of what is cut off, by 16 bits of a word made from the seed, the
// step's number and the value's place in the list; and since scales are powers of two, a value
// that keeps its place in the grid is not rounded anew when its block's largest changes.  A v above
// zero stays above zero: it is divided by.
//
// Bound by memory: 26 to 28 bytes a value with moments in 32 bits, 14 to 16 in 8, where the vector units have
// nearly as much to do: a code's bits are shifted into a float's, subnormal where its exponent is 0, so that
// one product decodes and one scaling rounds as the code's grid does.  One launch for up to kMost tensors,
// whose table travels in its arguments.
//   Measured with bf16 gradients: 0.6 billion float32 parameters with moments in 32 bits 3.03 ms, 5.1 TB/s; 0.2 billion
// with moments in 8 bits 0.60 ms, 4.8 TB/s (14 bytes a value).  30 tensors of up to 147456 values 8.6 us.
#include <algorithm>
#include <cmath>

#include "mcx_mfma_common.h"

namespace mcx {
namespace {

constexpr int kThreads = 256;
constexpr int kMost = 52;        // tensors of a launch: 3.6 kB of arguments
constexpr int kBlocks = 4096;    // workgroups of a launch
constexpr int kBlock = 256;      // values that share a scale: those of a wave
constexpr int64_t kLeast = 1024;     // values of a chunk
constexpr int64_t kLargest = 16384;
// Of the last-level cache: parameters, gradients and moments of 32 bits pass it by where there is more (0.6
// billion values 3.27 -> 3.04 ms).  Bytes do not: words of 4 a lane are slower past it.
constexpr int64_t kCacheBytes = 256 << 20;

struct AdamTensors {
  void *p[kMost];
  const void *g[kMost];
  void *m[kMost], *v[kMost];
  float *ms[kMost], *vs[kMost];
  int64_t size[kMost];
  int64_t base[kMost];       // blocks before it in the whole list
  int32_t first[kMost + 1];  // chunks before it in this launch
  uint64_t p_bf16, g_bf16, wide;  // a bit a tensor
  int32_t count, chunk;
};
static_assert(sizeof(AdamTensors) <= 3600, "the launch's arguments hold the table");

struct AdamNumbers {
  double rate, beta1, beta2, decay, max_norm;
  const int64_t *device_step;
  const float *device_rate, *norm;
  int64_t step;
  float eps;
  uint32_t seed;
};

// What every value is computed with.
struct AdamFactors {
  float b1, c1, b2, c2, keep, rate, root, eps, clip;
  uint32_t key;
};

typedef float float4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

__device__ inline uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}

__device__ inline AdamFactors factors_of(const AdamNumbers &n) {
  const int64_t step = n.device_step ? *n.device_step : n.step;
  const double rate = n.device_rate ? (double)*n.device_rate : n.rate;
  AdamFactors f;
  f.b1 = (float)n.beta1, f.c1 = (float)(1. - n.beta1);
  f.b2 = (float)n.beta2, f.c2 = (float)(1. - n.beta2);
  f.keep = (float)(1. - rate * n.decay);
  f.rate = (float)(rate / (1. - pow(n.beta1, (double)step)));
  f.root = (float)(1. / sqrt(1. - pow(n.beta2, (double)step)));
  f.eps = n.eps;
  f.clip = 1.f;
  if (n.norm) {
    const double ratio = n.max_norm / ((double)*n.norm + 1e-6);
    f.clip = ratio > 1. ? 1.f : (float)ratio;  // (no number stays none)
  }
  f.key = mix(mix((uint32_t)step) ^ n.seed);
  return f;
}

// Four values from i on, those below n.
template <typename T, bool Whole, bool Passing = false>
__device__ inline float4v four(const T *x, int64_t i, int64_t n) {
  float4v r = {0.f, 0.f, 0.f, 0.f};
  if (Whole) {
    typedef T Vec __attribute__((ext_vector_type(4)));
    const Vec w = Passing ? __builtin_nontemporal_load((const Vec *)(x + i)) : *(const Vec *)(x + i);
#pragma unroll
    for (int e = 0; e < 4; e++) r[e] = (float)w[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (i + e < n) r[e] = (float)x[i + e];
  }
  return r;
}
template <typename T, bool Whole, bool Passing = false>
__device__ inline void put_four(T *x, int64_t i, int64_t n, const float4v &r) {
  if (Whole) {
    typedef T Vec __attribute__((ext_vector_type(4)));
    Vec w;
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = (T)r[e];
    if (Passing) __builtin_nontemporal_store(w, (Vec *)(x + i));
    else *(Vec *)(x + i) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (i + e < n) x[i + e] = (T)r[e];
  }
}
template <bool Whole>
__device__ inline uint32_t four_codes(const uint8_t *x, int64_t i, int64_t n) {
  if (Whole) return *(const uint32_t *)(x + i);
  uint32_t r = 0;
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (i + e < n) r |= (uint32_t)x[i + e] << (8 * e);
  return r;
}
template <bool Whole>
__device__ inline void put_four_codes(uint8_t *x, int64_t i, int64_t n, uint32_t r) {
  if (Whole) {
    *(uint32_t *)(x + i) = r;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (i + e < n) x[i + e] = (uint8_t)(r >> (8 * e));
}

// Low: the exponent from which down the steps stay; a sign in the uppermost bit.
constexpr float power(int e) {
  float x = 1.f;
  for (; e > 0; e--) x *= 2.f;
  return x;
}
template <int Low, bool Signed>
__device__ inline float value_of(uint32_t code) {
  const uint32_t bits = Signed ? (code & 127) << 20 | (code & 128) << 24 : code << 20;
  constexpr float up = power(126 + Low);
  return __uint_as_float(bits) * up;
}
// A value of a block whose power of two has this exponent; 20 bits of chance.
template <int Low, bool Signed>
__device__ inline uint32_t code_of(float x, int exponent, uint32_t chance) {
  const float y = __builtin_amdgcn_ldexpf(fabsf(x), -exponent - 126 - Low);
  const uint32_t c = (__float_as_uint(y) + chance) >> 20;
  if (Signed) return min(c, 127u) | (x < 0.f ? 128u : 0u);
  return x > 0.f ? min(max(c, 1u), 255u) : 0u;
}

// The largest of a wave's values: lanes of four, eight and sixteen exchange, then rows go on to rows.
template <int Ctrl> __device__ inline uint32_t max_of(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, Ctrl, 0xf, 0xf, false));
}
__device__ inline uint32_t wave_max(uint32_t x) {
  x = max_of<0xb1>(x);   // quad_perm 1, 0, 3, 2
  x = max_of<0x4e>(x);   // quad_perm 2, 3, 0, 1
  x = max_of<0x141>(x);  // row_half_mirror
  x = max_of<0x140>(x);  // row_mirror
  x = max_of<0x142>(x);  // row_bcast 15
  x = max_of<0x143>(x);  // row_bcast 31
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
// The exponent of a block's power of two from its largest value's bits.
__device__ inline int exponent_of(uint32_t top) {
  return min(max((int)(top >> 23) - 126, -125), 127);
}
__device__ inline float scale_of(uint32_t top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);  // not a number
  return top ? __builtin_amdgcn_ldexpf(1.f, exponent_of(top)) : 0.f;
}

template <int Bits, typename P, typename G, bool Whole, bool Passing>
__device__ inline void adam_four(const AdamFactors &f, const AdamTensors &l, int t, int64_t i,
                                 int64_t n) {
  float4v p = four<P, Whole, Passing>((const P *)l.p[t], i, n), g = four<G, Whole, Passing>((const G *)l.g[t], i, n);
  float4v m, v;
  const int64_t block = i / kBlock;
  const bool here = i < n;
  if (Bits == 32) {
    m = four<float, Whole, Passing>((const float *)l.m[t], i, n);
    v = four<float, Whole, Passing>((const float *)l.v[t], i, n);
  } else {
    const uint32_t mc = four_codes<Whole>((const uint8_t *)l.m[t], i, n);
    const uint32_t vc = four_codes<Whole>((const uint8_t *)l.v[t], i, n);
    const float ms = Whole || here ? l.ms[t][block] : 0.f, vs = Whole || here ? l.vs[t][block] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      m[e] = value_of<-14, true>((mc >> (8 * e)) & 255) * ms;
      v[e] = value_of<-30, false>((vc >> (8 * e)) & 255) * vs;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float x = g[e] * f.clip;
    m[e] = m[e] * f.b1 + x * f.c1;
    v[e] = v[e] * f.b2 + (x * x) * f.c2;
    // (in 8 bits, where the vector units count, root and quotient to a unit in the last place)
    const float root = Bits == 32 ? sqrtf(v[e]) : __builtin_amdgcn_sqrtf(v[e]);
    const float below = root * f.root + f.eps;
    const float ratio = Bits == 32 ? m[e] / below : m[e] * __builtin_amdgcn_rcpf(below);
    p[e] = p[e] * f.keep - f.rate * ratio;
  }
  put_four<P, Whole, Passing>((P *)l.p[t], i, n, p);
  if (Bits == 32) {
    put_four<float, Whole, Passing>((float *)l.m[t], i, n, m);
    put_four<float, Whole, Passing>((float *)l.v[t], i, n, v);
    return;
  }
  uint32_t mt = 0, vt = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (!Whole && i + e >= n) continue;  // (what is not there may be no number by now)
    mt = max(mt, __float_as_uint(m[e]) & 0x7fffffffu);
    vt = max(vt, __float_as_uint(v[e]) & 0x7fffffffu);
  }
  mt = wave_max(mt), vt = wave_max(vt);
  const int me = exponent_of(mt), ve = exponent_of(vt);
  // (i is a multiple of 4: the upper half of the place is that of all four)
  const uint64_t at = (uint64_t)(l.base[t] * kBlock + i);
  const uint32_t upper = (uint32_t)(at >> 32) * 0x9E3779B1u;
  uint32_t mc = 0, vc = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const uint32_t word = mix((((uint32_t)at + e) ^ upper) + f.key);
    mc |= code_of<-14, true>(m[e], me, ((word & 0xffff) << 4) | 8) << (8 * e);
    vc |= code_of<-30, false>(v[e], ve, ((word >> 16) << 4) | 8) << (8 * e);
  }
  put_four_codes<Whole>((uint8_t *)l.m[t], i, n, mc);
  put_four_codes<Whole>((uint8_t *)l.v[t], i, n, vc);
  if ((threadIdx.x & 63) == 0 && here) l.ms[t][block] = scale_of(mt), l.vs[t][block] = scale_of(vt);
}

// Values [lo, hi) of a tensor, lo a multiple of kBlock; every wave walks whole blocks, so that the
// lanes behind the end are there for its sums.
template <int Bits, typename P, typename G, bool Passing>
__device__ inline void adam_chunk(const AdamFactors &f, const AdamTensors &l, int t, int64_t lo,
                                  int64_t hi) {
  const bool wide = (l.wide >> t) & 1;
  const int64_t last = lo + (hi - lo + kBlock - 1) / kBlock * kBlock;
  for (int64_t i = lo + 4 * threadIdx.x; i < last; i += 4 * kThreads) {
    const int64_t block = i / kBlock * kBlock;
    if (wide && block + kBlock <= hi) adam_four<Bits, P, G, true, Passing>(f, l, t, i, hi);
    else adam_four<Bits, P, G, false, Passing>(f, l, t, i, hi);
  }
}

template <int Bits, bool Passing>
__global__ __launch_bounds__(kThreads) void adamw_kernel(AdamTensors l, AdamNumbers n) {
  const AdamFactors f = factors_of(n);
  const int chunks = l.first[l.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (l.first[mid] <= c) lo = mid;
      else hi = mid - 1;
    }
    const int t = lo;
    const int64_t a = (int64_t)(c - l.first[t]) * l.chunk, z = min(l.size[t], a + l.chunk);
    const bool pb = (l.p_bf16 >> t) & 1, gb = (l.g_bf16 >> t) & 1;
    if (pb && gb) adam_chunk<Bits, __bf16, __bf16, Passing>(f, l, t, a, z);
    else if (pb) adam_chunk<Bits, __bf16, float, Passing>(f, l, t, a, z);
    else if (gb) adam_chunk<Bits, float, __bf16, Passing>(f, l, t, a, z);
    else adam_chunk<Bits, float, float, Passing>(f, l, t, a, z);
  }
}

template <typename T, int Low, bool Signed>
__global__ __launch_bounds__(kThreads) void adamw_moment_kernel(const uint8_t *codes, const float *scales,
                                                                T *out, int64_t n, bool wide) {
  const int64_t step = (int64_t)gridDim.x * kThreads * 4;
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4; i < n; i += step) {
    const bool whole = wide && i + 4 <= n;
    const uint32_t c = whole ? four_codes<true>(codes, i, n) : four_codes<false>(codes, i, n);
    const float scale = scales[i / kBlock];
    float4v r;
#pragma unroll
    for (int e = 0; e < 4; e++) r[e] = value_of<Low, Signed>((c >> (8 * e)) & 255) * scale;
    if (whole) put_four<T, true>(out, i, n, r);
    else put_four<T, false>(out, i, n, r);
  }
}

bool aligned(const void *x, int bytes) { return ((uintptr_t)x & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace
}  // namespace mcx

extern "C" {

int mcx_adamw_step(void *const *params, const void *const *grads, void *const *first,
                   void *const *second, float *const *first_scales, float *const *second_scales,
                   const int64_t *sizes, const int32_t *param_dtypes, const int32_t *grad_dtypes,
                   int64_t count, const mcx_adamw_options *o, void *stream) {
  using namespace mcx;
  if (!o) return MCX_E_NULL;
  if (count < 0 || !(o->beta1 >= 0 && o->beta1 < 1) || !(o->beta2 >= 0 && o->beta2 < 1) ||
      !(o->eps >= 0) || !(o->weight_decay >= 0) || (o->bits != 32 && o->bits != 8) ||
      (!o->device_step && o->step < 1) || (!o->device_rate && !std::isfinite(o->rate)) ||
      (o->grad_norm && !(o->max_norm >= 0)))
    return MCX_E_SHAPE;
  if (!count) return MCX_OK;
  if (!params || !grads || !first || !second || !sizes || !param_dtypes || !grad_dtypes ||
      (o->bits == 8 && (!first_scales || !second_scales)))
    return MCX_E_NULL;
  int64_t total = 0, bytes = 0;
  for (int64_t t = 0; t < count; t++) {
    if ((param_dtypes[t] != MCX_F32 && param_dtypes[t] != MCX_BF16) ||
        (grad_dtypes[t] != MCX_F32 && grad_dtypes[t] != MCX_BF16))
      return MCX_E_DTYPE;
    if (sizes[t] < 0 || sizes[t] > (1LL << 40)) return MCX_E_SHAPE;
    if (sizes[t] && (!params[t] || !grads[t] || !first[t] || !second[t] ||
                     (o->bits == 8 && (!first_scales[t] || !second_scales[t]))))
      return MCX_E_NULL;
    total += sizes[t];
    bytes += sizes[t] * ((param_dtypes[t] == MCX_BF16 ? 2 : 4) + (grad_dtypes[t] == MCX_BF16 ? 2 : 4) + o->bits / 4);
  }
  const bool passing = bytes > kCacheBytes;
  // two chunks a workgroup
  const int64_t even = ((total + 2 * kBlocks - 1) / (2 * kBlocks) + 1023) / 1024 * 1024;
  const int64_t chunk = std::max(kLeast, std::min(kLargest, even));
  if (total / chunk + count > 0x7fffffffLL) return MCX_E_SHAPE;
  AdamNumbers n;
  n.rate = o->rate, n.beta1 = o->beta1, n.beta2 = o->beta2, n.decay = o->weight_decay;
  n.max_norm = o->max_norm, n.device_step = o->device_step, n.device_rate = o->device_rate;
  n.norm = o->grad_norm, n.step = o->step, n.eps = (float)o->eps, n.seed = o->seed;
  int64_t base = 0;
  for (int64_t t0 = 0; t0 < count;) {
    AdamTensors l;
    l.count = 0, l.chunk = (int)chunk, l.first[0] = 0;
    l.p_bf16 = l.g_bf16 = l.wide = 0;
    for (; t0 < count && l.count < kMost; t0++) {
      if (!sizes[t0]) continue;
      const int k = l.count++;
      const bool pb = param_dtypes[t0] == MCX_BF16, gb = grad_dtypes[t0] == MCX_BF16;
      l.p[k] = params[t0], l.g[k] = grads[t0], l.m[k] = first[t0], l.v[k] = second[t0];
      l.ms[k] = o->bits == 8 ? first_scales[t0] : nullptr;
      l.vs[k] = o->bits == 8 ? second_scales[t0] : nullptr;
      l.size[k] = sizes[t0], l.base[k] = base;
      l.first[k + 1] = l.first[k] + (int)((sizes[t0] + chunk - 1) / chunk);
      base += (sizes[t0] + kBlock - 1) / kBlock;
      const int state = o->bits == 8 ? 4 : 16;
      if (aligned(params[t0], pb ? 8 : 16) && aligned(grads[t0], gb ? 8 : 16) &&
          aligned(first[t0], state) && aligned(second[t0], state))
        l.wide |= 1ull << k;
      l.p_bf16 |= (uint64_t)pb << k, l.g_bf16 |= (uint64_t)gb << k;
    }
    if (!l.count) break;
    const int blocks = std::min(l.first[l.count], kBlocks);
    const auto kernel = o->bits == 8 ? (passing ? adamw_kernel<8, true> : adamw_kernel<8, false>)
                                     : (passing ? adamw_kernel<32, true> : adamw_kernel<32, false>);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, l, n);
    MCX_HIP_CHECK_LAUNCH();
  }
  return MCX_OK;
}

int mcx_adamw_moment(const void *codes, const float *scales, void *out, int64_t size, int second,
                     int dtype, void *stream) {
  using namespace mcx;
  if (dtype != MCX_F32 && dtype != MCX_BF16) return MCX_E_DTYPE;
  if (size < 0 || size > (1LL << 40)) return MCX_E_SHAPE;
  if (!size) return MCX_OK;
  if (!codes || !scales || !out) return MCX_E_NULL;
  const bool wide = aligned(codes, 4) && aligned(out, dtype == MCX_BF16 ? 8 : 16);
  const dim3 grid((unsigned)std::min<int64_t>((size + 1023) / 1024, 8192)), threads(kThreads);
  const uint8_t *c = (const uint8_t *)codes;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MCX_F32 && second)
    hipLaunchKernelGGL((adamw_moment_kernel<float, -30, false>), grid, threads, 0, s, c, scales, (float *)out, size, wide);
  else if (dtype == MCX_F32)
    hipLaunchKernelGGL((adamw_moment_kernel<float, -14, true>), grid, threads, 0, s, c, scales, (float *)out, size, wide);
  else if (second)
    hipLaunchKernelGGL((adamw_moment_kernel<__bf16, -30, false>), grid, threads, 0, s, c, scales, (__bf16 *)out, size, wide);
  else
    hipLaunchKernelGGL((adamw_moment_kernel<__bf16, -14, true>), grid, threads, 0, s, c, scales, (__bf16 *)out, size, wide);
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}

}  // extern "C"
