// Group norm with an activation over tokens whose channels lie last, and its gradients.
//
//   n = (x - mean) r,  r = (var + eps)^(-1/2) over the tokens and a group's channels of a sample
//   u = n w + b,  y = act(u)
//   g = gy act'(u),  S1 = sum g, S2 = sum g n of a channel over the tokens of a sample
//   gx = r (w g - mean(w g) - n mean(w g n)),  gw = sum S2, gb = sum S1 over the samples
//
// Bound by memory.  A workgroup has a slab of whole groups, as wide as its threads reach in words, and a
// part of a sample's tokens; a thread walks down a word of channels.  Means and squares are formed in blocks
// of kRows tokens about each block's own mean and merged (counts, means and squared deviations), so a
// mean far from zero costs nothing.  Statistics of the parts, then products: two launches forward, and
// a third between them backward that joins the parts' sums.  No atomics: the same bits from call to call.
// Samples that a workgroup's threads hold a slab of take one launch and are read once; every sample has a work-
// group of its own at least, most of whose threads are idle where samples are a token or a few (65536 samples of a
// token of 128 channels 576 us).
//   Measured in bf16: 8 x 131072 tokens of 64 channels with silu statistics 33 us, products 50, sums 52, their join
// 5, gradients 68 (4.1, 5.4, 5.2 and 5.9 TB/s; a large copy 4.8: what was read last is read first from the cache).  32 x
// 2048 tokens of 512 channels with gelu 14, 31, 35, 5 and 42 us: there the vector units are busy 74 to 85 %
// of the time.  512 tokens of 128 channels 8.3 us.
#include <algorithm>
#include <type_traits>

#include "mcx_mfma_common.h"

namespace mcx {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 8;        // tokens of a block
constexpr int kBlocks = 1024;   // workgroups aimed at (2048: 32 x 2048 tokens of 512 channels 142 -> 157 us)
constexpr int kMostParts = 256;
constexpr int kAtOnce = 4;      // tokens whose loads are under way together
// Tensors of which two do not fit half the last-level cache: results that stay in it push out the input
// that is read a second time (8 x 131072 tokens of 64 channels, forward and gradients 230 -> 211 us).
constexpr int64_t kPassingBytes = 64 << 20;
constexpr int kJoin = 16;       // channels, or whole groups, of a workgroup that joins parts

enum { kNone = 0, kSilu = 1, kGelu = 2 };

struct GroupParams {
  const void *x, *w, *b, *gy;
  void *y, *gx, *gw, *gb;
  float *stats;    // [B, G, 2]: mean, r
  float *partial;  // forward [B, G, parts, 2]: mean, squares; backward [B, parts, C, 2]: S1, S2
  float *sums;     // backward [B, C, 2]: S1, S2
  float *means;    // backward [B, G, 2]: the means of w g and w g n
  int64_t xs[2];   // strides of sample and token
  int64_t N;
  int B, C, G, per;    // per: channels of a group
  int slab, slabs;     // groups of a slab
  int parts, rows;     // parts of a sample's tokens, tokens of a part
  float eps;
};

template <typename T, int E> struct Word {
  typedef T Vec __attribute__((ext_vector_type(E)));
  static __device__ inline void load(const T *p, float *v) {
    const Vec w = *(const Vec *)p;
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = (float)w[e];
  }
  // Passing: past the cache
  template <bool Passing> static __device__ inline void store(T *p, const float *v) {
    Vec w;
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = (T)v[e];
    if (Passing) __builtin_nontemporal_store(w, (Vec *)p);
    else *(Vec *)p = w;
  }
};
template <typename T> struct Word<T, 1> {
  static __device__ inline void load(const T *p, float *v) { v[0] = (float)*p; }
  template <bool> static __device__ inline void store(T *p, const float *v) { *p = (T)v[0]; }
};

// e^x and 1 / (1 + e^-x), to a few units in the last place: the hardware's powers of two and reciprocals,
// in single precision with what the product's rounding takes put back.
template <bool Fine> __device__ inline float exponential(float x) {
  constexpr float kLog2e = 1.44269504f, kRest = 1.92596299e-8f;
  const float t = x * kLog2e;
  const float e = __builtin_amdgcn_exp2f(t);
  return Fine ? fmaf(e, 0.69314718f * fmaf(x, kRest, fmaf(x, kLog2e, -t)), e) : e;
}
template <bool Fine> __device__ inline float logistic(float x) {
  if (!Fine) return __builtin_amdgcn_rcpf(1.f + exponential<false>(-x));
  // (an infinite power has no rounding to put back: 0 where e^-x leaves the range, since u is multiplied by it;
  // what is no number stays none)
  const float y = __builtin_elementwise_minimum(__builtin_elementwise_maximum(x, -87.f), 80.f);
  return x < -87.f ? 0.f : __builtin_amdgcn_rcpf(1.f + exponential<true>(-y));
}
// (1 + erf(u / sqrt 2)) / 2 by formula 7.1.26 of Abramowitz and Stegun, off by 7.5e-8 at most (in all: far below zero
// few digits are right); `bell` is e^(-u^2 / 2), down to 0: the slope multiplies it by u.  It costs a third of the
// library's erf, which the vector units took longer for than memory.
template <bool Fine> __device__ inline float normal(float u, float &bell) {
  // (an infinite power has no rounding to put back)
  const float q = Fine ? fminf(u * u, 1000.f) : u * u;
  bell = Fine ? exponential<true>(-0.5f * q) : __builtin_amdgcn_exp2f(-0.72134752f * q);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.23164190f, fabsf(u), 1.f));
  float s = fmaf(0.5307027145f, t, -0.7265760135f);
  s = fmaf(s, t, 0.7107068705f);
  s = fmaf(s, t, -0.142248368f);
  s = fmaf(s, t, 0.127414796f);
  s = s * t * bell;
  return u < 0.f ? s : 1.f - s;
}

template <int Act, bool Fine> __device__ inline float act(float u) {
  float bell;
  if (Act == kSilu) return u * logistic<Fine>(u);
  if (Act == kGelu) return u * normal<Fine>(u, bell);
  return u;
}
template <int Act, bool Fine> __device__ inline float act_slope(float u) {
  if (Act == kSilu) {
    const float s = logistic<Fine>(u);
    return s * fmaf(u, 1.f - s, 1.f);
  }
  if (Act == kGelu) {
    float bell;
    const float n = normal<Fine>(u, bell);
    return fmaf(u * bell, 0.39894228f, n);
  }
  return 1.f;
}
template <typename T> constexpr bool kFine = sizeof(T) == 4;

// Where a workgroup and its threads stand.
struct Place {
  int b, part, g0, groups, c0, channels;  // groups and channels of the slab
  int words, across, lanes, lane, col;    // words of the slab; threads a row, rows a pass
  int64_t row, end;
};
template <int E> __device__ inline Place place_of(const GroupParams &p, int64_t index) {
  Place a;
  a.part = (int)(index % p.parts);
  index /= p.parts;
  const int s = (int)(index % p.slabs);
  a.b = (int)(index / p.slabs);
  a.g0 = s * p.slab, a.groups = min(p.slab, p.G - a.g0);
  a.c0 = a.g0 * p.per, a.channels = a.groups * p.per;
  a.words = a.channels / E;
  a.across = min(a.words, kThreads);
  a.lanes = kThreads / a.across;
  a.lane = threadIdx.x / a.across, a.col = threadIdx.x % a.across;
  a.row = (int64_t)a.part * p.rows, a.end = min(p.N, a.row + p.rows);
  return a;
}

// A thread's tokens of the part: f(count, first) for `Count` of them at a time, then one by one.
template <int Count, typename F> __device__ inline void walk(const Place &a, F f) {
  int64_t r = a.row + a.lane;
  for (; r + (int64_t)(Count - 1) * a.lanes < a.end; r += (int64_t)Count * a.lanes)
    f(std::integral_constant<int, Count>(), r);
  for (; r < a.end; r += a.lanes) f(std::integral_constant<int, 1>(), r);
}

// Count, mean and squared deviations, and those of a block merged into them.
struct Moments {
  float n, mean, squares;
  __device__ inline void merge(float count, float m, float q) {
    const float all = n + count, d = m - mean, f = count / all;
    mean += d * f;
    squares += q + d * d * n * f;
    n = all;
  }
};

// Threads a group's entries are summed by: `team` of them, a power of two, for each of `groups`.
__device__ inline int team_of(int groups) {
  int team = 64;
  while (team > 1 && team * groups > kThreads) team >>= 1;
  return team;
}
__device__ inline float team_sum(float x, int team) {
  for (int m = team >> 1; m; m >>= 1) x += __shfl_xor(x, m);
  return x;
}

// Own: every channel of a word has moments of its own (a word may lie in two groups).
template <typename T, int E, bool Own>
__global__ __launch_bounds__(kThreads) void group_stats_kernel(GroupParams p) {
  constexpr int M = Own ? E : 1;  // moments of a thread
  __shared__ float count[kThreads], mean[kThreads * M], squares[kThreads * M];
  const Place a = place_of<E>(p, blockIdx.x);
  Moments s[M];
#pragma unroll
  for (int e = 0; e < M; e++) s[e] = {0.f, 0.f, 0.f};
  if (a.lane < a.lanes) {
    // (more than one round only where the slab is one group, whose moments are one)
    for (int col = a.col; col < a.words; col += a.across) {
      const T *x = (const T *)p.x + a.b * p.xs[0] + a.c0 + col * E;
      int64_t r = a.row + a.lane;
      for (; r + (int64_t)(kRows - 1) * a.lanes < a.end; r += (int64_t)kRows * a.lanes) {
        float v[kRows][E];
#pragma unroll
        for (int k = 0; k < kRows; k++) Word<T, E>::load(x + (r + (int64_t)k * a.lanes) * p.xs[1], v[k]);
#pragma unroll
        for (int m = 0; m < M; m++) {
          float sum = 0.f, q = 0.f;
#pragma unroll
          for (int k = 0; k < kRows; k++)
#pragma unroll
            for (int e = 0; e < E; e++)
              if (!Own || e == m) sum += v[k][e];
          const int n = Own ? kRows : kRows * E;
          sum *= 1.f / n;
#pragma unroll
          for (int k = 0; k < kRows; k++)
#pragma unroll
            for (int e = 0; e < E; e++)
              if (!Own || e == m) q += (v[k][e] - sum) * (v[k][e] - sum);
          s[m].merge((float)n, sum, q);
        }
      }
      for (; r < a.end; r += a.lanes) {
        float v[E];
        Word<T, E>::load(x + r * p.xs[1], v);
#pragma unroll
        for (int m = 0; m < M; m++) {
          float sum = 0.f, q = 0.f;
          const int n = Own ? 1 : E;
#pragma unroll
          for (int e = 0; e < E; e++)
            if (!Own || e == m) sum += v[e];
          sum *= 1.f / n;
#pragma unroll
          for (int e = 0; e < E; e++)
            if (!Own || e == m) q += (v[e] - sum) * (v[e] - sum);
          s[m].merge((float)n, sum, q);
        }
      }
    }
  }
  count[threadIdx.x] = s[0].n;
#pragma unroll
  for (int m = 0; m < M; m++) {
    mean[threadIdx.x * M + m] = s[m].mean;
    squares[threadIdx.x * M + m] = s[m].squares;
  }
  __syncthreads();
  // a group's entries: `wide` neighbours of each row of threads
  const int wide = a.words > a.across ? a.across : p.per * M / E, entries = wide * a.lanes;
  const int team = team_of(a.groups), lane = threadIdx.x & (team - 1);
  for (int g = threadIdx.x / team; g < a.groups; g += kThreads / team) {
    float n = 0.f, sum = 0.f, q = 0.f;
    for (int i = lane; i < entries; i += team) {
      const int at = i / wide * a.across * M + g * wide + i % wide;
      n += count[at / M], sum += count[at / M] * mean[at];
    }
    n = team_sum(n, team), sum = team_sum(sum, team);
    const float centre = n > 0.f ? sum / n : 0.f;
    for (int i = lane; i < entries; i += team) {
      const int at = i / wide * a.across * M + g * wide + i % wide;
      const float d = mean[at] - centre;
      q += squares[at] + count[at / M] * d * d;
    }
    q = team_sum(q, team);
    if (lane == 0) {
      float *to = p.partial + (((int64_t)a.b * p.G + a.g0 + g) * p.parts + a.part) * 2;
      to[0] = centre, to[1] = q;
    }
  }
}

// Mean and r of a slab's groups from the parts', into LDS [groups][2]; a lane's reads are under way four at a
// time (60000 tokens of 64 bf16 channels in 32 groups, forward, 27 -> 20 us).
__device__ inline void join_stats(const GroupParams &p, const Place &a, float *stats) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  const int team = team_of(a.groups), lane = threadIdx.x & (team - 1);
  // (all parts have the tokens of the first but the last)
  const float all = (float)p.N, n = (float)p.rows, last = (float)(p.N - (int64_t)(p.parts - 1) * p.rows);
  for (int g = threadIdx.x / team; g < a.groups; g += kThreads / team) {
    const float2v *from = (const float2v *)p.partial + ((int64_t)a.b * p.G + a.g0 + g) * p.parts;
    float sum = 0.f, q = 0.f;
#pragma unroll 4
    for (int i = lane; i < p.parts; i += team) sum += from[i].x * ((i == p.parts - 1 ? last : n) / all);
    const float mean = team_sum(sum, team);
#pragma unroll 4
    for (int i = lane; i < p.parts; i += team) {
      const float2v part = from[i];
      const float d = part.x - mean;
      q += part.y + (i == p.parts - 1 ? last : n) * p.per * d * d;
    }
    q = team_sum(q, team);
    if (lane == 0) {
      stats[2 * g] = mean;
      stats[2 * g + 1] = 1.f / sqrtf(q / (all * p.per) + p.eps);
    }
  }
}

// A thread's channels (Own: of several groups).  n = x r - mean r in one step where x has few bits itself (its
// own are lost before the product's rounding is); in single precision the difference first.
template <typename T, int E, bool Own = true> struct Channels {
  static constexpr int M = Own ? E : 1;
  float mean[M], r[M], w[E], b[E];
  __device__ inline float norm(float x, int e) const {
    const int m = Own ? e : 0;
    return kFine<T> ? (x - mean[m]) * r[m] : fmaf(x, r[m], mean[m]);
  }
  __device__ inline float scaled(float x, int e) const { return fmaf(norm(x, e), w[e], b[e]); }
  __device__ inline Channels(const GroupParams &p, const Place &a, int col) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      w[e] = p.w ? (float)((const T *)p.w)[a.c0 + col * E + e] : 1.f;
      b[e] = p.b ? (float)((const T *)p.b)[a.c0 + col * E + e] : 0.f;
    }
  }
  __device__ inline Channels(const GroupParams &p, const Place &a, const float *stats, int col)
      : Channels(p, a, col) {
    take(p, stats, col);
  }
  __device__ inline void take(const GroupParams &p, const float *stats, int col) {
    int g = col * E / p.per, rest = col * E - g * p.per;
#pragma unroll
    for (int m = 0; m < M; m++) {
      mean[m] = stats[2 * g], r[m] = stats[2 * g + 1];
      if (!kFine<T>) mean[m] *= -r[m];
      if (++rest == p.per) rest = 0, g++;
    }
  }
};

// gx from n and g, for a thread's channels.
template <typename T, int E, bool Own = true> struct Slope {
  static constexpr int M = Own ? E : 1;
  float m1[M], m2[M], wr[E];  // (times r in bf16)
  __device__ inline Slope(const GroupParams &p, const Channels<T, E, Own> &ch, const float *means, int col) {
    int g = col * E / p.per, rest = col * E - g * p.per;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float r = kFine<T> ? 1.f : ch.r[Own ? e : 0];
      if (e < M) {
        m1[e] = -means[2 * g] * r, m2[e] = -means[2 * g + 1] * r;
        if (++rest == p.per) rest = 0, g++;
      }
      wr[e] = ch.w[e] * r;
    }
  }
  __device__ inline float value(const Channels<T, E, Own> &ch, float n, float d, int e) const {
    const int m = Own ? e : 0;
    return kFine<T> ? ch.r[m] * ((d * ch.w[e] + m1[m]) + n * m2[m]) : fmaf(d, wr[e], fmaf(n, m2[m], m1[m]));
  }
};

extern __shared__ float dynamic[];

template <typename T, int E, int Act, bool Passing>
__global__ __launch_bounds__(kThreads) void group_apply_kernel(GroupParams p) {
  const Place a = place_of<E>(p, gridDim.x - 1 - (int64_t)blockIdx.x);
  float *stats = dynamic;  // [slab][2]
  join_stats(p, a, stats);
  __syncthreads();
  if (p.stats && a.part == 0)
    for (int i = threadIdx.x; i < 2 * a.groups; i += kThreads)
      p.stats[((int64_t)a.b * p.G + a.g0) * 2 + i] = stats[i];
  if (a.lane >= a.lanes) return;
  for (int col = a.col; col < a.words; col += a.across) {
    const Channels<T, E> ch(p, a, stats, col);
    const T *x = (const T *)p.x + a.b * p.xs[0] + a.c0 + col * E;
    T *y = (T *)p.y + (int64_t)a.b * p.N * p.C + a.c0 + col * E;
    walk<kAtOnce>(a, [&](auto count, int64_t r) {
      constexpr int K = decltype(count)::value;
      float v[K][E];
#pragma unroll
      for (int k = 0; k < K; k++) Word<T, E>::load(x + (r + (int64_t)k * a.lanes) * p.xs[1], v[k]);
#pragma unroll
      for (int k = 0; k < K; k++) {
#pragma unroll
        for (int e = 0; e < E; e++)
          v[k][e] = act<Act, kFine<T>>(ch.scaled(v[k][e], e));
        Word<T, E>::template store<Passing>(y + (r + (int64_t)k * a.lanes) * p.C, v[k]);
      }
    });
  }
}

// S1 and S2 of the channels of a slab over a part.
template <typename T, int E, int Act>
__global__ __launch_bounds__(kThreads) void group_sums_kernel(GroupParams p) {
  __shared__ float part[kThreads * E * 2];
  const Place a = place_of<E>(p, blockIdx.x);
  const float *stats = p.stats + ((int64_t)a.b * p.G + a.g0) * 2;
  for (int first = 0; first < a.words; first += a.across) {
    const int col = first + a.col;
    float s1[E], s2[E];
#pragma unroll
    for (int e = 0; e < E; e++) s1[e] = s2[e] = 0.f;
    if (a.lane < a.lanes && col < a.words) {
      const Channels<T, E> ch(p, a, stats, col);
      const T *x = (const T *)p.x + a.b * p.xs[0] + a.c0 + col * E;
      const T *gy = (const T *)p.gy + (int64_t)a.b * p.N * p.C + a.c0 + col * E;
      walk<kAtOnce>(a, [&](auto count, int64_t r) {
        constexpr int K = decltype(count)::value;
        float v[K][E], g[K][E];
#pragma unroll
        for (int k = 0; k < K; k++) {
          Word<T, E>::load(x + (r + (int64_t)k * a.lanes) * p.xs[1], v[k]);
          Word<T, E>::load(gy + (r + (int64_t)k * a.lanes) * p.C, g[k]);
        }
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
          for (int e = 0; e < E; e++) {
            const float n = ch.norm(v[k][e], e);
            const float d = g[k][e] * act_slope<Act, kFine<T>>(fmaf(n, ch.w[e], ch.b[e]));
            s1[e] += d, s2[e] = fmaf(d, n, s2[e]);
          }
      });
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++) {
      part[(threadIdx.x * E + e) * 2] = s1[e];
      part[(threadIdx.x * E + e) * 2 + 1] = s2[e];
    }
    __syncthreads();
    const int n = min(a.across, a.words - first) * E * 2;
    float *to = p.partial + (((int64_t)a.b * p.parts + a.part) * p.C + a.c0 + first * E) * 2;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      float s = 0.f;
      for (int l = 0; l < a.lanes; l++) s += part[l * a.across * E * 2 + i];
      to[i] = s;
    }
  }
}

// The sums over the parts of a sample's groups (kJoin channels of them, or one), and the means of w g and
// w g n.
template <typename T>
__global__ __launch_bounds__(kThreads) void group_join_kernel(GroupParams p, int several, int jobs) {
  __shared__ float part[kThreads];
  const int b = blockIdx.x / jobs, g0 = blockIdx.x % jobs * several, groups = min(several, p.G - g0);
  const int c0 = g0 * p.per, all = groups * p.per * 2;  // sums
  const int across = min(all, kThreads), lanes = kThreads / across;
  const int lane = threadIdx.x / across, col = threadIdx.x % across;
  float *sums = p.sums + ((int64_t)b * p.C + c0) * 2;
  for (int first = 0; first < all; first += across) {
    float x = 0.f;
    if (lane < lanes && first + col < all) {
      const float *from = p.partial + ((int64_t)b * p.parts * p.C + c0) * 2 + first + col;
      int i = lane;
      for (; i + 7 * lanes < p.parts; i += 8 * lanes) {
        float y[8];
#pragma unroll
        for (int k = 0; k < 8; k++) y[k] = from[(int64_t)(i + k * lanes) * p.C * 2];
#pragma unroll
        for (int k = 0; k < 8; k++) x += y[k];
      }
      for (; i < p.parts; i += lanes) x += from[(int64_t)i * p.C * 2];
    }
    __syncthreads();
    part[threadIdx.x] = x;
    __syncthreads();
    if (lane == 0 && first + col < all) {
      for (int l = 1; l < lanes; l++) x += part[l * across + col];
      sums[first + col] = x;
    }
  }
  __syncthreads();  // (the workgroup's own writes)
  const int team = team_of(groups);
  for (int g = threadIdx.x / team; g < groups; g += kThreads / team) {
    float x1 = 0.f, x2 = 0.f;
    for (int i = threadIdx.x & (team - 1); i < p.per; i += team) {
      const float w = p.w ? (float)((const T *)p.w)[c0 + g * p.per + i] : 1.f;
      x1 = fmaf(w, sums[(g * p.per + i) * 2], x1);
      x2 = fmaf(w, sums[(g * p.per + i) * 2 + 1], x2);
    }
    x1 = team_sum(x1, team), x2 = team_sum(x2, team);
    if ((threadIdx.x & (team - 1)) == 0) {
      const float n = (float)p.N * p.per;
      float *to = p.means + ((int64_t)b * p.G + g0 + g) * 2;
      to[0] = x1 / n, to[1] = x2 / n;
    }
  }
}

// gw and gb of a slab's channels: the sums over the samples.
template <typename T, int Threads>
__device__ inline void sum_samples(const GroupParams &p, int c0, int channels, float *part) {
  if (!p.gw && !p.gb) return;
  const int across = min(channels, Threads), lanes = Threads / across;
  const int lane = threadIdx.x / across, col = threadIdx.x % across;
  for (int first = 0; first < channels; first += across) {
    const int c = first + col;
    float x1 = 0.f, x2 = 0.f;
    if (lane < lanes && c < channels) {
      const float *from = p.sums + (int64_t)(c0 + c) * 2;
#pragma unroll 4
      for (int b = lane; b < p.B; b += lanes) {
        x1 += from[(int64_t)b * p.C * 2];
        x2 += from[(int64_t)b * p.C * 2 + 1];
      }
    }
    __syncthreads();
    part[threadIdx.x] = x1, part[Threads + threadIdx.x] = x2;
    __syncthreads();
    if (lane == 0 && c < channels) {
      for (int l = 1; l < lanes; l++) {
        x1 += part[l * across + col];
        x2 += part[Threads + l * across + col];
      }
      if (p.gb) ((T *)p.gb)[c0 + c] = (T)x1;
      if (p.gw) ((T *)p.gw)[c0 + c] = (T)x2;
    }
  }
}

template <typename T, int E, int Act, bool Passing>
__global__ __launch_bounds__(kThreads) void group_gradient_kernel(GroupParams p) {
  __shared__ float part[kThreads * 2];
  const Place a = place_of<E>(p, gridDim.x - 1 - (int64_t)blockIdx.x);
  const float *stats = p.stats + ((int64_t)a.b * p.G + a.g0) * 2;
  const float *means = p.means + ((int64_t)a.b * p.G + a.g0) * 2;
  if (p.gx && a.lane < a.lanes)
    for (int col = a.col; col < a.words; col += a.across) {
      const Channels<T, E> ch(p, a, stats, col);
      const Slope<T, E> slope(p, ch, means, col);
      const T *x = (const T *)p.x + a.b * p.xs[0] + a.c0 + col * E;
      const int64_t from = (int64_t)a.b * p.N * p.C + a.c0 + col * E;
      const T *gy = (const T *)p.gy + from;
      T *gx = (T *)p.gx + from;
      walk<kAtOnce>(a, [&](auto count, int64_t r) {
        constexpr int K = decltype(count)::value;
        float v[K][E], g[K][E];
#pragma unroll
        for (int k = 0; k < K; k++) {
          Word<T, E>::load(x + (r + (int64_t)k * a.lanes) * p.xs[1], v[k]);
          Word<T, E>::load(gy + (r + (int64_t)k * a.lanes) * p.C, g[k]);
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
          for (int e = 0; e < E; e++) {
            const float n = ch.norm(v[k][e], e);
            const float d = g[k][e] * act_slope<Act, kFine<T>>(fmaf(n, ch.w[e], ch.b[e]));
            v[k][e] = slope.value(ch, n, d, e);
          }
          Word<T, E>::template store<Passing>(gx + (r + (int64_t)k * a.lanes) * p.C, v[k]);
        }
      });
    }
  // one workgroup of each slab
  if (a.b == 0 && a.part == 0) sum_samples<T, kThreads>(p, a.c0, a.channels, part);
}

// ---- samples whose slab a workgroup holds ----
//
// Up to kHeld words a thread stay there between the statistics and the products, so that everything is read
// once, by one launch (and a second small one for the sums over the samples).  They stay in registers but for some
// kernels of 1024 threads, which have 128 each, and words of 8 bf16 values: those whose words lie in several
// groups, and gradients with an activation, keep 12 to 132 bytes a lane in scratch memory.

constexpr int kHeld = 8;
constexpr int kHeldWords = 32;            // words of a slab at most
constexpr int kHeldSlots = kHeldWords * 8;

template <typename T, int E> struct Kept {
  typedef T Vec __attribute__((ext_vector_type(E)));
  Vec x;
  __device__ inline void load(const T *p) { x = *(const Vec *)p; }
  __device__ inline float operator[](int e) const { return (float)x[e]; }
};
template <typename T> struct Kept<T, 1> {
  T x;
  __device__ inline void load(const T *p) { x = *p; }
  __device__ inline float operator[](int) const { return (float)x; }
};

// The threads' values summed over the rows of threads into slots [across * M]: by lane exchange within a wave
// where rows are a power of two of lanes, through LDS otherwise.
template <int Threads, int M>
__device__ inline void sum_rows(const Place &a, float *values, float *all, float *some, float *slots) {
  const int n = a.across * M;
  __syncthreads();
  if ((a.across & (a.across - 1)) == 0) {
    for (int d = a.across; d < 64; d <<= 1)
#pragma unroll
      for (int m = 0; m < M; m++) values[m] += __shfl_xor(values[m], d);
    if ((threadIdx.x & 63) < a.across)
#pragma unroll
      for (int m = 0; m < M; m++) all[(threadIdx.x >> 6) * n + a.col * M + m] = values[m];
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += Threads) {
      float x = all[i];
#pragma unroll
      for (int w = 1; w < Threads / 64; w++) x += all[w * n + i];
      slots[i] = x;
    }
    __syncthreads();
    return;
  }
  // (two sums one after the other, of about as many values each)
  const int several = max(1, min(Threads / n, 8));
#pragma unroll
  for (int m = 0; m < M; m++) all[threadIdx.x * M + m] = values[m];
  __syncthreads();
  for (int i = threadIdx.x; i < n * several; i += Threads) {
    const int first = i / n, slot = i - first * n;
    float x = 0.f;
    for (int l = first; l < a.lanes; l += several) x += all[l * n + slot];
    some[i] = x;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += Threads) {
    float x = some[i];
    for (int k = 1; k < several; k++) x += some[k * n + i];
    slots[i] = x;
  }
  __syncthreads();
}

template <int Threads, int E> __device__ inline Place held_place(const GroupParams &p) {
  Place a;
  const int index = xcd_contiguous_tile(blockIdx.x, gridDim.x), s = index % p.slabs;
  a.b = index / p.slabs, a.part = 0;
  a.g0 = s * p.slab, a.groups = min(p.slab, p.G - a.g0);
  a.c0 = a.g0 * p.per, a.channels = a.groups * p.per;
  a.words = a.across = a.channels / E;
  a.lanes = Threads / a.across;
  a.lane = threadIdx.x / a.across, a.col = threadIdx.x % a.across;
  a.row = 0, a.end = p.N;
  return a;
}

template <int Threads, typename T, int E, int Act, bool Own>
__global__ __launch_bounds__(Threads) void group_held_kernel(GroupParams p) {
  constexpr int M = Own ? E : 1;
  __shared__ float all[Threads * M], some[Threads > kHeldSlots ? Threads : kHeldSlots], slots[kHeldSlots];
  __shared__ float stats[kHeldSlots * 2];
  const Place a = held_place<Threads, E>(p);
  const bool here = a.lane < a.lanes;
  const T *x = (const T *)p.x + a.b * p.xs[0] + a.c0 + a.col * E;
  Kept<T, E> v[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; k++) {
    const int64_t r = a.lane + (int64_t)k * a.lanes;
    if (here && r < p.N) v[k].load(x + r * p.xs[1]);
  }
  Channels<T, E, Own> ch(p, a, here ? a.col : 0);
  const float count = (float)p.N * p.per;
  const int each = p.per * M / E;  // slots of a group
  const int group = a.col * E / p.per, rest = a.col * E - group * p.per;
  // the means first, then the squares of what differs from them
  for (int pass = 0; pass < 2; pass++) {
    float sum[M], mean[M];
    int g = group, at = rest;
#pragma unroll
    for (int m = 0; m < M; m++) {
      sum[m] = 0.f;
      mean[m] = pass && here ? stats[2 * g] : 0.f;
      if (++at == p.per) at = 0, g++;
    }
#pragma unroll
    for (int k = 0; k < kHeld; k++)
      if (here && a.lane + (int64_t)k * a.lanes < p.N)
#pragma unroll
        for (int e = 0; e < E; e++) {
          const int m = Own ? e : 0;
          const float d = v[k][e] - mean[m];
          sum[m] = pass ? fmaf(d, d, sum[m]) : sum[m] + d;
        }
    sum_rows<Threads, M>(a, sum, all, some, slots);
    for (int g = threadIdx.x; g < a.groups; g += Threads) {
      float s = 0.f;
      for (int i = 0; i < each; i++) s += slots[g * each + i];
      stats[2 * g + pass] = pass ? 1.f / sqrtf(s / count + p.eps) : s / count;
    }
    __syncthreads();
  }
  if (p.stats)
    for (int i = threadIdx.x; i < 2 * a.groups; i += Threads)
      p.stats[((int64_t)a.b * p.G + a.g0) * 2 + i] = stats[i];
  if (!here) return;
  ch.take(p, stats, a.col);
  T *y = (T *)p.y + (int64_t)a.b * p.N * p.C + a.c0 + a.col * E;
#pragma unroll
  for (int k = 0; k < kHeld; k++) {
    const int64_t r = a.lane + (int64_t)k * a.lanes;
    if (r < p.N) {
      float o[E];
#pragma unroll
      for (int e = 0; e < E; e++) o[e] = act<Act, kFine<T>>(ch.scaled(v[k][e], e));
      Word<T, E>::template store<false>(y + r * p.C, o);
    }
  }
}

template <int Threads, typename T, int E, int Act, bool Own>
__global__ __launch_bounds__(Threads) void group_held_gradient_kernel(GroupParams p) {
  __shared__ float all[Threads * E], some[Threads > kHeldSlots ? Threads : kHeldSlots];
  __shared__ float sums[2][kHeldSlots], means[kHeldSlots * 2];
  const Place a = held_place<Threads, E>(p);
  const bool here = a.lane < a.lanes;
  const int64_t dense = (int64_t)a.b * p.N * p.C + a.c0 + a.col * E;
  const T *x = (const T *)p.x + a.b * p.xs[0] + a.c0 + a.col * E, *gy = (const T *)p.gy + dense;
  Kept<T, E> v[kHeld], g[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; k++) {
    const int64_t r = a.lane + (int64_t)k * a.lanes;
    if (here && r < p.N) v[k].load(x + r * p.xs[1]), g[k].load(gy + r * p.C);
  }
  const Channels<T, E, Own> ch(p, a, p.stats + ((int64_t)a.b * p.G + a.g0) * 2, here ? a.col : 0);
  float s1[E], s2[E];
#pragma unroll
  for (int e = 0; e < E; e++) s1[e] = s2[e] = 0.f;
#pragma unroll
  for (int k = 0; k < kHeld; k++)
    if (here && a.lane + (int64_t)k * a.lanes < p.N)
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float n = ch.norm(v[k][e], e);
        const float d = g[k][e] * act_slope<Act, kFine<T>>(fmaf(n, ch.w[e], ch.b[e]));
        s1[e] += d, s2[e] = fmaf(d, n, s2[e]);
      }
  sum_rows<Threads, E>(a, s1, all, some, sums[0]);
  sum_rows<Threads, E>(a, s2, all, some, sums[1]);
  for (int i = threadIdx.x; i < a.channels; i += Threads) {
    const int c = a.c0 + i;
    if (p.sums) {
      float *to = p.sums + ((int64_t)a.b * p.C + c) * 2;
      to[0] = sums[0][i], to[1] = sums[1][i];
    } else {  // the only sample
      if (p.gb) ((T *)p.gb)[c] = (T)sums[0][i];
      if (p.gw) ((T *)p.gw)[c] = (T)sums[1][i];
    }
  }
  if (!p.gx) return;
  const float count = (float)p.N * p.per;
  for (int k = threadIdx.x; k < 2 * a.groups; k += Threads) {
    const float *from = sums[k & 1] + (k >> 1) * p.per;
    float s = 0.f;
    for (int i = 0; i < p.per; i++)
      s = fmaf(p.w ? (float)((const T *)p.w)[a.c0 + (k >> 1) * p.per + i] : 1.f, from[i], s);
    means[k] = s / count;
  }
  __syncthreads();
  if (!here) return;
  T *gx = (T *)p.gx + dense;
  const Slope<T, E, Own> slope(p, ch, means, a.col);
#pragma unroll
  for (int k = 0; k < kHeld; k++) {
    const int64_t r = a.lane + (int64_t)k * a.lanes;
    if (r < p.N) {
      float o[E];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float n = ch.norm(v[k][e], e);
        const float d = g[k][e] * act_slope<Act, kFine<T>>(fmaf(n, ch.w[e], ch.b[e]));
        o[e] = slope.value(ch, n, d, e);
      }
      Word<T, E>::template store<false>(gx + r * p.C, o);
    }
  }
}

template <typename T> __global__ __launch_bounds__(kThreads) void group_samples_kernel(GroupParams p) {
  __shared__ float part[kThreads * 2];
  const int c0 = blockIdx.x * kJoin;
  sum_samples<T, kThreads>(p, c0, min(kJoin, p.C - c0), part);
}

// ---- host ----

int common(int a, int b) { return b ? common(b, a % b) : a; }

// (so that the parts' sums stay below 16 MB a sample)
int64_t most_parts(int64_t N, int64_t C) {
  return std::min<int64_t>({kMostParts, std::max<int64_t>(1, (1 << 21) / C), N});
}

// Values of a word that rows at this address, stride and width are read by, and the slab's groups.
struct Split {
  int word, slab, slabs, parts, rows;
};
Split split_of(int64_t B, int64_t N, int64_t C, int64_t G, int size, uint64_t bytes) {
  Split s;
  const int per = (int)(C / G);
  s.word = 1;
  for (int w : {16 / size, 2})
    if (s.word == 1 && C % w == 0 && bytes % (w * size) == 0) {
      // whole groups that are whole words
      const int least = w / common(per % w ? per : w, w);
      if (C / w <= kThreads || least == 1 || least * per <= kThreads * w) s.word = w;
    }
  const int w = s.word, least = w / common(per % w ? per : w, w);
  if (C / w <= kThreads) s.slab = (int)G;
  else s.slab = std::max(1, kThreads * w / (per * least)) * least;
  s.slab = (int)std::min<int64_t>(s.slab, G);
  s.slabs = (int)((G + s.slab - 1) / s.slab);
  const int64_t across = std::min<int64_t>((int64_t)s.slab * per / w, kThreads);
  const int64_t lanes = std::max<int64_t>(1, kThreads / std::max<int64_t>(1, across));
  int64_t parts = std::max<int64_t>(1, kBlocks / std::max<int64_t>(1, B * s.slabs));
  parts = std::min<int64_t>({parts, most_parts(N, C), (N + lanes * kRows - 1) / (lanes * kRows)});
  s.rows = (int)((N + parts - 1) / parts);
  s.parts = (int)((N + s.rows - 1) / s.rows);
  return s;
}

// The slab of the held form: as wide as a workgroup holds, but no wider than 128 bytes unless that leaves
// more than kHeldGroups workgroups; 0: a sample does not fit.  threads: of that workgroup.
// Workgroups of 1024 threads leave nothing to load beside those that compute: they are for calls that other-
// wise wait for launches (forward and gradients of 4096 tokens of 256 channels 36 -> 32 us; 16 of them 80 -> 96);
// others get a slab that 256 hold, 32 bytes of a row at least (219 x 606 tokens of 128 bf16 channels, which
// 1024 threads held 64 bytes of, 93 -> 74 us; 128 x 512 of 256 channels 83 -> 56).
constexpr int kHeldGroups = 512, kHeldAlone = 128, kHeldBytes = 32;
int held_slab(int64_t B, int64_t N, int64_t C, int64_t G, int word, int size, int *threads) {
  const int per = (int)(C / G), least = word / common(per % word ? per : word, word);
  const int64_t unit = (int64_t)least * per / word;  // words
  if (unit > kHeldWords || N > 1024 * kHeld || (int64_t)least > G) return 0;
  for (int most : {1024, 256}) {
    int64_t best = 0;
    for (int64_t k = 1; k * least < G + least && k * unit <= kHeldWords; k++) {
      const int64_t words = std::min(k * unit, C / word);
      if (N > most / words * kHeld) break;
      if (best && (words * word * size > 128 || B * ((G + k * least - 1) / (k * least)) < kHeldGroups)) break;
      best = k;
    }
    const int64_t slab = std::min(best * least, G), words = slab * per / word;
    if (!best || (most == 256 && slab < G && words * word * size < kHeldBytes)) return 0;
    *threads = N <= 256 / words * kHeld ? 256 : 1024;
    if (*threads == 256 || B * ((G + slab - 1) / slab) <= kHeldAlone) return (int)slab;
  }
  return 0;
}

int check_sizes(int64_t B, int64_t N, int64_t C, int64_t G, int dtype) {
  if (dtype != MCX_F32 && dtype != MCX_BF16) return MCX_E_DTYPE;
  if (B < 0 || N < 0 || C < 1 || G < 1 || C % G || C > (1 << 20) || N > 0x7fffffffLL ||
      B > (1 << 23) || B * G > (1 << 23) || (B && N > (1LL << 44) / B / C))
    return MCX_E_SHAPE;
  return MCX_OK;
}

uint64_t address_bits(const void *x, const int64_t *stride, int64_t B, int64_t N, int size) {
  return (uint64_t)(uintptr_t)x | (B > 1 ? (uint64_t)stride[0] * size : 0) |
         (N > 1 ? (uint64_t)stride[1] * size : 0);
}

template <int Threads, typename T, int E, int Act> int launch_held(const GroupParams &p, hipStream_t s) {
  const dim3 grid((unsigned)(p.B * p.slabs)), threads(Threads);
  if (p.per % E == 0) {
    hipLaunchKernelGGL((p.gy ? group_held_gradient_kernel<Threads, T, E, Act, false>
                             : group_held_kernel<Threads, T, E, Act, false>), grid, threads, 0, s, p);
  } else if constexpr (E > 1) {
    hipLaunchKernelGGL((p.gy ? group_held_gradient_kernel<Threads, T, E, Act, true>
                             : group_held_kernel<Threads, T, E, Act, true>), grid, threads, 0, s, p);
  }
  MCX_HIP_CHECK_LAUNCH();
  if (p.gy && p.sums && (p.gw || p.gb)) {
    hipLaunchKernelGGL((group_samples_kernel<T>), dim3((p.C + kJoin - 1) / kJoin), dim3(kThreads), 0, s, p);
    MCX_HIP_CHECK_LAUNCH();
  }
  return MCX_OK;
}
template <typename T, int E, int Act> int try_held(GroupParams p, hipStream_t s, bool *done) {
  int threads = 0;
  const int slab = held_slab(p.B, p.N, p.C, p.G, E, sizeof(T), &threads);
  *done = slab > 0;
  if (!slab) return MCX_OK;
  p.slab = slab, p.slabs = (p.G + slab - 1) / slab;
  if (p.gy && p.B == 1) p.sums = nullptr;
  return threads == 256 ? launch_held<256, T, E, Act>(p, s) : launch_held<1024, T, E, Act>(p, s);
}

template <typename T, int E> bool passing(const GroupParams &p) {
  return (int64_t)p.B * p.N * p.C * (int64_t)sizeof(T) >= kPassingBytes;
}

template <typename T, int E, int Act>
int launch_forward(const GroupParams &p, hipStream_t s) {
  bool done;
  if (int e = try_held<T, E, Act>(p, s, &done); e || done) return e;
  const dim3 grid((unsigned)((int64_t)p.B * p.slabs * p.parts)), threads(kThreads);
  if (p.per % E == 0) {
    hipLaunchKernelGGL((group_stats_kernel<T, E, false>), grid, threads, 0, s, p);
  } else if constexpr (E > 1) {
    hipLaunchKernelGGL((group_stats_kernel<T, E, true>), grid, threads, 0, s, p);
  }
  MCX_HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL((passing<T, E>(p) ? group_apply_kernel<T, E, Act, E * sizeof(T) == 16>
                                       : group_apply_kernel<T, E, Act, false>),
                     grid, threads, sizeof(float) * 2 * p.slab, s, p);
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}
template <typename T, int E, int Act>
int launch_backward(const GroupParams &p, hipStream_t s) {
  bool done;
  if (int e = try_held<T, E, Act>(p, s, &done); e || done) return e;
  const dim3 grid((unsigned)((int64_t)p.B * p.slabs * p.parts)), threads(kThreads);
  hipLaunchKernelGGL((group_sums_kernel<T, E, Act>), grid, threads, 0, s, p);
  MCX_HIP_CHECK_LAUNCH();
  const int several = std::min(p.G, std::max(1, kJoin / p.per)), jobs = (p.G + several - 1) / several;
  hipLaunchKernelGGL((group_join_kernel<T>), dim3((unsigned)(p.B * jobs)), threads, 0, s, p, several, jobs);
  MCX_HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL((passing<T, E>(p) ? group_gradient_kernel<T, E, Act, E * sizeof(T) == 16>
                                       : group_gradient_kernel<T, E, Act, false>),
                     grid, threads, 0, s, p);
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}
template <typename T, int E, bool Forward>
int launch_act(const GroupParams &p, int act, hipStream_t s) {
  if (Forward)
    return act == kSilu   ? launch_forward<T, E, kSilu>(p, s)
           : act == kGelu ? launch_forward<T, E, kGelu>(p, s)
                          : launch_forward<T, E, kNone>(p, s);
  return act == kSilu   ? launch_backward<T, E, kSilu>(p, s)
         : act == kGelu ? launch_backward<T, E, kGelu>(p, s)
                        : launch_backward<T, E, kNone>(p, s);
}
template <bool Forward>
int launch_word(const GroupParams &p, int word, int act, int dtype, hipStream_t s) {
  if (dtype == MCX_BF16)
    return word == 8   ? launch_act<__bf16, 8, Forward>(p, act, s)
           : word == 2 ? launch_act<__bf16, 2, Forward>(p, act, s)
                       : launch_act<__bf16, 1, Forward>(p, act, s);
  return word == 4   ? launch_act<float, 4, Forward>(p, act, s)
         : word == 2 ? launch_act<float, 2, Forward>(p, act, s)
                     : launch_act<float, 1, Forward>(p, act, s);
}

GroupParams params_of(const Split &f, const int64_t *stride, int64_t B, int64_t N, int64_t C, int64_t G) {
  GroupParams p = {};
  p.xs[0] = stride[0], p.xs[1] = stride[1], p.N = N;
  p.B = (int)B, p.C = (int)C, p.G = (int)G, p.per = (int)(C / G);
  p.slab = f.slab, p.slabs = f.slabs, p.parts = f.parts, p.rows = f.rows;
  return p;
}

}  // namespace
}  // namespace mcx

extern "C" {

size_t mcx_group_norm_workspace(int64_t B, int64_t N, int64_t C, int64_t G, int backward, int dtype) {
  using namespace mcx;
  if (check_sizes(B, N, C, G, dtype) != MCX_OK || !B || !N) return 0;
  // (as many parts as any alignment gives)
  const int64_t parts = std::min(most_parts(N, C), std::max<int64_t>(1, kBlocks / B));
  if (!backward) return (size_t)(B * G * parts * 2) * sizeof(float);
  return (size_t)(B * parts * C * 2 + B * C * 2 + B * G * 2) * sizeof(float);
}

int mcx_group_norm_forward(const void *x, const void *weight, const void *bias, void *y, float *stats,
                           void *workspace, size_t workspace_bytes, const int64_t *x_stride, int64_t B,
                           int64_t N, int64_t C, int64_t G, double eps, int activation, int dtype,
                           void *stream) {
  using namespace mcx;
  if (int e = check_sizes(B, N, C, G, dtype)) return e;
  if (!(eps >= 0) || activation < kNone || activation > kGelu) return MCX_E_SHAPE;
  if (!B || !N) return MCX_OK;
  if (!x || !y || !x_stride) return MCX_E_NULL;
  const size_t need = mcx_group_norm_workspace(B, N, C, G, 0, dtype);
  if (!workspace || workspace_bytes < need) return MCX_E_WORKSPACE;
  const int size = dtype == MCX_BF16 ? 2 : 4;
  const Split f = split_of(B, N, C, G, size, address_bits(x, x_stride, B, N, size) | (uint64_t)(uintptr_t)y);
  GroupParams p = params_of(f, x_stride, B, N, C, G);
  p.x = x, p.w = weight, p.b = bias, p.y = y, p.stats = stats, p.eps = (float)eps;
  p.partial = (float *)workspace;
  return launch_word<true>(p, f.word, activation, dtype, (hipStream_t)stream);
}

int mcx_group_norm_backward(const void *gy, const void *x, const float *stats, const void *weight,
                            const void *bias, void *gx, void *gweight, void *gbias, void *workspace,
                            size_t workspace_bytes, const int64_t *x_stride, int64_t B, int64_t N,
                            int64_t C, int64_t G, int activation, int dtype, void *stream) {
  using namespace mcx;
  if (int e = check_sizes(B, N, C, G, dtype)) return e;
  if (activation < kNone || activation > kGelu) return MCX_E_SHAPE;
  if (!B || !N || (!gx && !gweight && !gbias)) return MCX_OK;
  if (!gy || !x || !stats || !x_stride) return MCX_E_NULL;
  const size_t need = mcx_group_norm_workspace(B, N, C, G, 1, dtype);
  if (!workspace || workspace_bytes < need) return MCX_E_WORKSPACE;
  const int size = dtype == MCX_BF16 ? 2 : 4;
  const Split f = split_of(B, N, C, G, size, address_bits(x, x_stride, B, N, size) |
                                                 (uint64_t)(uintptr_t)gy | (uint64_t)(uintptr_t)gx);
  GroupParams p = params_of(f, x_stride, B, N, C, G);
  p.x = x, p.w = weight, p.b = bias, p.gy = gy, p.gx = gx, p.gw = gweight, p.gb = gbias;
  p.stats = const_cast<float *>(stats);
  p.partial = (float *)workspace;
  p.sums = p.partial + (int64_t)B * f.parts * C * 2;
  p.means = p.sums + B * C * 2;
  return launch_word<false>(p, f.word, activation, dtype, (hipStream_t)stream);
}

}  // extern "C"
