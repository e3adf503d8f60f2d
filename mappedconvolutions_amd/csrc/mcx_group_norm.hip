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
#include <algorithm>
#include <type_traits>

#include "mcx_mfma_common.h"

namespace mcx {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 8;        // tokens of a block
constexpr int kBlocks = 2048;   // workgroups aimed at
constexpr int kMostParts = 256;
constexpr int kAtOnce = 4;      // tokens whose loads are under way together
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
  static __device__ inline void store(T *p, const float *v) {
    Vec w;
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = (T)v[e];
    *(Vec *)p = w;
  }
};
template <typename T> struct Word<T, 1> {
  static __device__ inline void load(const T *p, float *v) { v[0] = (float)*p; }
  static __device__ inline void store(T *p, const float *v) { *p = (T)v[0]; }
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
  if (Fine) {  // (an infinite power has no rounding to put back; what is no number stays none)
    x = x < -80.f ? -80.f : x;
    x = x > 80.f ? 80.f : x;
  }
  return __builtin_amdgcn_rcpf(1.f + exponential<Fine>(-x));
}
// (1 + erf(u / sqrt 2)) / 2 by formula 7.1.26 of Abramowitz and Stegun, off by 7.5e-8 at most; `bell` is
// e^(-u^2 / 2).  It costs a third of the library's erf, which the vector units took longer for than memory.
template <bool Fine> __device__ inline float normal(float u, float &bell) {
  const float q = Fine ? fminf(u * u, 170.f) : u * u;
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

// Mean and r of a slab's groups from the parts', into LDS [groups][2].
__device__ inline void join_stats(const GroupParams &p, const Place &a, float *stats) {
  const int team = team_of(a.groups), lane = threadIdx.x & (team - 1);
  for (int g = threadIdx.x / team; g < a.groups; g += kThreads / team) {
    const float *from = p.partial + ((int64_t)a.b * p.G + a.g0 + g) * p.parts * 2;
    float sum = 0.f, q = 0.f;
    const float all = (float)p.N;
    for (int i = lane; i < p.parts; i += team)
      sum += from[2 * i] * ((float)min((int64_t)p.rows, p.N - (int64_t)i * p.rows) / all);
    const float mean = team_sum(sum, team);
    for (int i = lane; i < p.parts; i += team) {
      const float d = from[2 * i] - mean;
      const float n = (float)min((int64_t)p.rows, p.N - (int64_t)i * p.rows);
      q += from[2 * i + 1] + n * p.per * d * d;
    }
    q = team_sum(q, team);
    if (lane == 0) {
      stats[2 * g] = mean;
      stats[2 * g + 1] = 1.f / sqrtf(q / (all * p.per) + p.eps);
    }
  }
}

// A thread's channels.  n = x r - mean r in one step where x has few bits itself (its own are lost before
// the product's rounding is); in single precision the difference first.
template <typename T, int E> struct Channels {
  float mean[E], r[E], w[E], b[E];
  __device__ inline float norm(float x, int e) const {
    return kFine<T> ? (x - mean[e]) * r[e] : fmaf(x, r[e], mean[e]);
  }
  __device__ inline float scaled(float x, int e) const { return fmaf(norm(x, e), w[e], b[e]); }
  __device__ inline Channels(const GroupParams &p, const Place &a, const float *stats, int col) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int c = col * E + e, g = c / p.per;
      mean[e] = stats[2 * g], r[e] = stats[2 * g + 1];
      if (!kFine<T>) mean[e] *= -r[e];
      w[e] = p.w ? (float)((const T *)p.w)[a.c0 + c] : 1.f;
      b[e] = p.b ? (float)((const T *)p.b)[a.c0 + c] : 0.f;
    }
  }
};

extern __shared__ float dynamic[];

template <typename T, int E, int Act>
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
        Word<T, E>::store(y + (r + (int64_t)k * a.lanes) * p.C, v[k]);
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

template <typename T, int E, int Act>
__global__ __launch_bounds__(kThreads) void group_gradient_kernel(GroupParams p) {
  __shared__ float part[kThreads * 2];
  const Place a = place_of<E>(p, gridDim.x - 1 - (int64_t)blockIdx.x);
  const float *stats = p.stats + ((int64_t)a.b * p.G + a.g0) * 2;
  const float *means = p.means + ((int64_t)a.b * p.G + a.g0) * 2;
  if (p.gx && a.lane < a.lanes)
    for (int col = a.col; col < a.words; col += a.across) {
      const Channels<T, E> ch(p, a, stats, col);
      float m1[E], m2[E], wr[E];  // (times r in bf16)
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int g = (col * E + e) / p.per;
        const float r = kFine<T> ? 1.f : ch.r[e];
        m1[e] = -means[2 * g] * r, m2[e] = -means[2 * g + 1] * r, wr[e] = ch.w[e] * r;
      }
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
            v[k][e] = kFine<T> ? ch.r[e] * ((d * ch.w[e] + m1[e]) + n * m2[e])
                               : fmaf(d, wr[e], fmaf(n, m2[e], m1[e]));
          }
          Word<T, E>::store(gx + (r + (int64_t)k * a.lanes) * p.C, v[k]);
        }
      });
    }
  // one workgroup of each slab: the sums over the samples
  if (a.b || a.part || (!p.gw && !p.gb)) return;
  const int across = min(a.channels, kThreads), lanes = kThreads / across;
  const int lane = threadIdx.x / across, col = threadIdx.x % across;
  for (int first = 0; first < a.channels; first += across) {
    const int c = first + col;
    float x1 = 0.f, x2 = 0.f;
    if (lane < lanes && c < a.channels)
      for (int b = lane; b < p.B; b += lanes) {
        x1 += p.sums[((int64_t)b * p.C + a.c0 + c) * 2];
        x2 += p.sums[((int64_t)b * p.C + a.c0 + c) * 2 + 1];
      }
    __syncthreads();
    part[threadIdx.x] = x1, part[kThreads + threadIdx.x] = x2;
    __syncthreads();
    if (lane == 0 && c < a.channels) {
      for (int l = 1; l < lanes; l++) {
        x1 += part[l * across + col];
        x2 += part[kThreads + l * across + col];
      }
      if (p.gb) ((T *)p.gb)[a.c0 + c] = (T)x1;
      if (p.gw) ((T *)p.gw)[a.c0 + c] = (T)x2;
    }
  }
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

template <typename T, int E, int Act>
int launch_forward(const GroupParams &p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.B * p.slabs * p.parts)), threads(kThreads);
  if (p.per % E == 0 || p.slab == 1)
    hipLaunchKernelGGL((group_stats_kernel<T, E, false>), grid, threads, 0, s, p);
  else
    hipLaunchKernelGGL((group_stats_kernel<T, E, true>), grid, threads, 0, s, p);
  MCX_HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL((group_apply_kernel<T, E, Act>), grid, threads, sizeof(float) * 2 * p.slab, s, p);
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}
template <typename T, int E, int Act>
int launch_backward(const GroupParams &p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.B * p.slabs * p.parts)), threads(kThreads);
  hipLaunchKernelGGL((group_sums_kernel<T, E, Act>), grid, threads, 0, s, p);
  MCX_HIP_CHECK_LAUNCH();
  const int several = std::min(p.G, std::max(1, kJoin / p.per)), jobs = (p.G + several - 1) / several;
  hipLaunchKernelGGL((group_join_kernel<T>), dim3((unsigned)(p.B * jobs)), threads, 0, s, p, several, jobs);
  MCX_HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL((group_gradient_kernel<T, E, Act>), grid, threads, 0, s, p);
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
