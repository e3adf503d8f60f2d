// Clipping of a list of tensors by their global norm.
//
// Bound by memory: the squares need every value once, the products read and write every value
// once more, and nothing can be multiplied before all is summed.  Two launches for up to kMost
// tensors: their table travels in the launch's arguments (no copy to the device), a workgroup
// takes chunks of them in turn, and the second launch's workgroups each add up the first's sums,
// in the same order, instead of waiting for a third.
//   300 tensors of 0.6 billion bf16 values: 68 us for the squares of 0.4 GB (5.9 TB/s), 664 us in
// all for 3.6 GB (5.4 TB/s; a large copy reaches 4.9): 708 us with the products in the squares'
// order and 696 us with results written through the cache.  30 small tensors take 10 us.
#include <algorithm>
#include <cmath>

#include "mcx_mfma_common.h"

namespace mcx {
namespace {

constexpr int kThreads = 256;
constexpr int kMost = 128;         // tensors of a launch: 3.6 kB of arguments
constexpr int kBlocks = 1024;      // workgroups of a launch
constexpr int64_t kLeast = 2048;   // values of a chunk
constexpr int64_t kLargest = 32768;
constexpr int64_t kCacheBytes = 256 << 20;  // of the last-level cache

struct List {
  const void *in[kMost];
  void *out[kMost];
  int64_t size[kMost];
  int32_t first[kMost + 1];  // chunks before each tensor
  uint32_t bf16[kMost / 32];
  int32_t count, chunk;
};

template <typename T> __device__ inline float value(T x) { return (float)x; }

// What a workgroup does to values [lo, hi) of a tensor, in 16-byte words where the address allows it.
template <typename T> struct Chunk {
  static constexpr int E = 16 / (int)sizeof(T);
  typedef __attribute__((ext_vector_type(E))) T Vec;

  // This thread's part of the sum of squares, in A; the bits that any of its values has go to `bits`.
  template <typename A>
  static __device__ inline A squares(const T *x, int64_t lo, int64_t hi, unsigned &bits) {
    typedef __attribute__((ext_vector_type(4))) unsigned Words;
    const int tid = threadIdx.x;
    // values before the first whole word, and behind the last
    const int64_t skew = (int64_t)(((uintptr_t)(x + lo) & 15) / sizeof(T));
    const int64_t a = min(hi, lo + (skew ? E - skew : 0)), z = a + (hi - a) / E * E;
    A s = 0, t[4] = {0, 0, 0, 0};
    const auto one = [&](T v) {
      s = fma((A)value(v), (A)value(v), s);
      bits |= __float_as_uint(value(v));
    };
    const auto word = [&](const Vec &v, A &sum) {
#pragma unroll
      for (int e = 0; e < E; e++) sum = fma((A)value(v[e]), (A)value(v[e]), sum);
      const Words w = __builtin_bit_cast(Words, v);
      bits |= w[0] | w[1] | w[2] | w[3];
    };
    for (int64_t i = lo + tid; i < a; i += kThreads) one(x[i]);
    for (int64_t i = z + tid; i < hi; i += kThreads) one(x[i]);
    int64_t i = a + tid * E;
    for (; i + 3 * kThreads * E < z; i += 4 * kThreads * E) {
      Vec v[4];
#pragma unroll
      for (int n = 0; n < 4; n++) v[n] = *(const Vec *)(x + i + n * kThreads * E);
#pragma unroll
      for (int n = 0; n < 4; n++) word(v[n], t[n]);
    }
    for (; i < z; i += kThreads * E) word(*(const Vec *)(x + i), s);
    return s + (t[0] + t[1]) + (t[2] + t[3]);
  }
  // In fp32 (a few hundred squares at most), and again in fp64 where that overflows (a value beyond
  // 10^19) or is so small that squares may be lost below it.
  static __device__ inline double squares(const T *x, int64_t lo, int64_t hi) {
    unsigned bits = 0;
    const float s = squares<float>(x, lo, hi, bits);
    if ((s >= 0x1p-90f && s < __builtin_inff()) || !bits) return s;
    return squares<double>(x, lo, hi, bits);
  }

  template <bool Passing>
  static __device__ inline void scale(const T *x, T *y, int64_t lo, int64_t hi, float factor) {
    const int tid = threadIdx.x;
    const int64_t skew = (int64_t)(((uintptr_t)(x + lo) & 15) / sizeof(T));
    // words only where both sides start alike
    const bool alike = (((uintptr_t)x ^ (uintptr_t)y) & 15) == 0;
    const int64_t a = alike ? min(hi, lo + (skew ? E - skew : 0)) : hi, z = a + (hi - a) / E * E;
    for (int64_t i = lo + tid; i < a; i += kThreads) y[i] = (T)(value(x[i]) * factor);
    for (int64_t i = z + tid; i < hi; i += kThreads) y[i] = (T)(value(x[i]) * factor);
    int64_t i = a + tid * E;
    for (; i + 3 * kThreads * E < z; i += 4 * kThreads * E) {
      Vec v[4];
#pragma unroll
      for (int n = 0; n < 4; n++) v[n] = *(const Vec *)(x + i + n * kThreads * E);
#pragma unroll
      for (int n = 0; n < 4; n++) {
#pragma unroll
        for (int e = 0; e < E; e++) v[n][e] = (T)(value(v[n][e]) * factor);
        if (Passing) __builtin_nontemporal_store(v[n], (Vec *)(y + i + n * kThreads * E));
        else *(Vec *)(y + i + n * kThreads * E) = v[n];
      }
    }
    for (; i < z; i += kThreads * E) {
      Vec v = *(const Vec *)(x + i);
#pragma unroll
      for (int e = 0; e < E; e++) v[e] = (T)(value(v[e]) * factor);
      *(Vec *)(y + i) = v;
    }
  }
};

// The tensor that chunk c belongs to.
__device__ inline int tensor_of(const List &l, int c) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ inline double block_sum(double x) {
  __shared__ double part[kThreads / 64];
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0.;
  for (int w = 0; w < kThreads / 64; w++) x += part[w];
  __syncthreads();
  return x;
}

// A thread's squares of a chunk are summed in fp32 where it holds them, everything else in fp64.
__global__ __launch_bounds__(kThreads) void grad_squares_kernel(List l, double *sums) {
  double s = 0.;
  const int chunks = l.first[l.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(l, c);
    const int64_t lo = (int64_t)(c - l.first[t]) * l.chunk, hi = min(l.size[t], lo + l.chunk);
    s += (l.bf16[t >> 5] >> (t & 31)) & 1 ? Chunk<__bf16>::squares((const __bf16 *)l.in[t], lo, hi)
                                          : Chunk<float>::squares((const float *)l.in[t], lo, hi);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// Passing: the results are more than the cache holds, and are written past it.
template <bool Passing>
__global__ __launch_bounds__(kThreads) void grad_scale_kernel(List l, const double *sums, int n,
                                                              double max_norm, double eps,
                                                              float *norm) {
  double s = 0.;
  for (int i = threadIdx.x; i < n; i += kThreads) s += sums[i];
  const double total = sqrt(block_sum(s));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)total;
  const double ratio = max_norm / (total + eps);
  const float factor = ratio > 1. ? 1.f : (float)ratio;  // (no number stays none)
  const int chunks = l.first[l.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(l, c);
    if (factor == 1.f && l.in[t] == l.out[t]) continue;  // in place, nothing changes
    const int64_t lo = (int64_t)(c - l.first[t]) * l.chunk, hi = min(l.size[t], lo + l.chunk);
    if ((l.bf16[t >> 5] >> (t & 31)) & 1)
      Chunk<__bf16>::template scale<Passing>((const __bf16 *)l.in[t], (__bf16 *)l.out[t], lo, hi, factor);
    else
      Chunk<float>::template scale<Passing>((const float *)l.in[t], (float *)l.out[t], lo, hi, factor);
  }
}

int64_t chunk_of(int64_t total) {
  const int64_t even = (total + 2 * kBlocks - 1) / (2 * kBlocks);  // two chunks a workgroup
  return std::max(kLeast, std::min(kLargest, (even + 2047) / 2048 * 2048));
}

}  // namespace
}  // namespace mcx

extern "C" {

size_t mcx_clip_grad_norm_workspace(const int64_t *sizes, int64_t count) {
  if (count < 0 || (count && !sizes)) return 0;
  return sizeof(double) * mcx::kBlocks * (size_t)((count + mcx::kMost - 1) / mcx::kMost + 1);
}

int mcx_clip_grad_norm(const void *const *in, void *const *out, const int64_t *sizes,
                       const int32_t *dtypes, int64_t count, double max_norm, double eps,
                       float *norm, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace mcx;
  if (count < 0 || !(max_norm >= 0) || !(eps >= 0)) return MCX_E_SHAPE;
  if (!norm || (count && (!in || !sizes || !dtypes))) return MCX_E_NULL;
  if (!workspace || workspace_bytes < mcx_clip_grad_norm_workspace(sizes, count))
    return MCX_E_WORKSPACE;
  int64_t total = 0, bytes = 0;
  for (int64_t t = 0; t < count; t++) {
    if (dtypes[t] != MCX_F32 && dtypes[t] != MCX_BF16) return MCX_E_DTYPE;
    if (sizes[t] < 0 || sizes[t] > (1LL << 40)) return MCX_E_SHAPE;
    if (sizes[t] && (!in[t] || (out && !out[t]))) return MCX_E_NULL;
    total += sizes[t];
    bytes += sizes[t] * (dtypes[t] == MCX_BF16 ? 2 : 4);
  }
  const int64_t chunk = chunk_of(total);
  if (total / chunk + count > 0x7fffffffLL) return MCX_E_SHAPE;
  double *sums = (double *)workspace;
  hipStream_t s = (hipStream_t)stream;
  int used = 0;
  for (int pass = 0; pass < 2; pass++) {
    // pass 0: the squares of every kMost tensors; pass 1: the products, and the norm
    bool norm_done = false;
    for (int64_t t0 = 0; t0 < count || (pass == 1 && !norm_done);) {
      List l;
      l.count = 0, l.chunk = (int)chunk, l.first[0] = 0;
      for (int w = 0; w < kMost / 32; w++) l.bf16[w] = 0;
      for (; t0 < count && l.count < kMost; t0++) {
        // the products begin with what the squares read last, which may still be cached
        const int64_t t = pass == 0 ? t0 : count - 1 - t0;
        if (!sizes[t]) continue;
        const int n = l.count++;
        l.in[n] = in[t], l.out[n] = out ? out[t] : nullptr, l.size[n] = sizes[t];
        l.first[n + 1] = l.first[n] + (int)((sizes[t] + chunk - 1) / chunk);
        if (dtypes[t] == MCX_BF16) l.bf16[n >> 5] |= 1u << (n & 31);
      }
      const int chunks = l.first[l.count];
      if (pass == 0) {
        if (!l.count) continue;
        const int blocks = std::min(chunks, kBlocks);
        hipLaunchKernelGGL(grad_squares_kernel, dim3(blocks), dim3(kThreads), 0, s, l, sums + used);
        used += blocks;
      } else {
        if (!out) l.count = 0;
        if (!l.count) l.first[0] = 0;
        const int blocks = l.count ? std::min(chunks, 2 * kBlocks) : 1;
        if (l.count || !norm_done)
          hipLaunchKernelGGL(bytes > kCacheBytes ? grad_scale_kernel<true> : grad_scale_kernel<false>,
                             dim3(blocks), dim3(kThreads), 0, s, l, sums, used, max_norm, eps,
                             norm_done ? nullptr : norm);
        norm_done = true;
        if (!out) break;
      }
      MCX_HIP_CHECK_LAUNCH();
    }
  }
  return MCX_OK;
}

}  // extern "C"
