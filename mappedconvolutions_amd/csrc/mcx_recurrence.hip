// A gated linear recurrence along a sequence, and its gradients.
//
//   a_t = sigmoid(f_t),  h_t = a_t h_{t-1} + (1 - a_t) v_t,  out_t = h_t g_t sigmoid(g_t)  (or h_t)
//   D_t = d_t + p_t,  d_t = go_t g_t sigmoid(g_t),  p_{t-1} = a_t D_t      (p_L: the final state's gradient)
//   gv = (1 - a) D,  gf = a (1 - a) (h_{t-1} - v) D,  gg = go h silu'(g),  gh_0 = p_0
//
// Bound by memory: 4 streams forward, 7 backward, and a few dozen operations a value.  Channels are
// independent; a workgroup has 16 lanes' words of them and walks the steps in tiles, each lane with T
// steps of its own.  h_t of a run of steps is A h + H of the state before it; the lanes' (A, H) are joined
// within a wave by lane exchange and between waves through LDS, so a tile costs one barrier forward and
// two backward.  States are kept for the gradients every kSpan steps and the others recomputed.  Where
// sequences and channels are too few to fill the card the steps are cut into segments, whose (A, H) a
// first launch sums up.
#include <algorithm>

#include "mcx_mfma_common.h"

namespace mcx {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kRowLanes = 16;           // lanes of a step's channels
constexpr int kRuns = kThreads / kRowLanes;  // runs of steps of a tile
constexpr int kForward = 8, kBackward = 4;   // steps of a run
constexpr int kTile = kRuns * kForward;      // 256 steps
constexpr int kSpan = kRuns * kBackward;     // steps from one kept state to the next
constexpr int kGroups = 512;            // workgroups aimed at
constexpr int kFew = 8;                 // steps that a thread walks alone

struct RecurParams {
  const void *v, *f, *g, *go;
  const float *initial, *gfinal;
  const int32_t *lengths;
  void *out, *gv, *gf, *gg;
  float *final, *ginitial, *states;  // states [B, ceil(L / kSpan), C]
  float *part;                       // [B, segments, 2, C]: A, H of a segment
  int64_t vs[2], fs[2], gs[2];       // strides of sequence and step
  int L, C, tiles, segments, segment;  // tiles of channels; steps of a segment
  int spans, reverse;
};

template <typename T, int E> struct Raw {
  typedef T Vec __attribute__((ext_vector_type(E)));
  Vec x;
  __device__ inline void load(const T *p) { x = *(const Vec *)p; }
  __device__ inline float operator[](int e) const { return (float)x[e]; }
};
template <typename T> struct Raw<T, 1> {
  T x;
  __device__ inline void load(const T *p) { x = *p; }
  __device__ inline float operator[](int) const { return (float)x; }
};
template <typename T, int E> __device__ inline void put(T *p, const float *v) {
  if constexpr (E == 1) {
    *p = (T)v[0];
  } else {
    typedef T Vec __attribute__((ext_vector_type(E)));
    Vec w;
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = (T)v[e];
    *(Vec *)p = w;
  }
}

// sigmoid(x), and in `away` 1 - sigmoid(x) without its cancellation.  Fine: what the roundings of the
// product and of the reciprocal took is put back; factors, whose errors add up over hundreds of steps,
// are always computed so (3 us of 330 on 134 million bf16 values), output gates in single precision.
template <bool Fine> __device__ inline float logistic(float x, float &away) {
  x = x < -80.f ? -80.f : x;  // (what is no number stays none)
  if (Fine) x = x > 200.f ? 200.f : x;
  constexpr float kLog2e = 1.44269504f, kRest = 1.92596299e-8f;
  const float t = -x * kLog2e;
  float e = __builtin_amdgcn_exp2f(t);
  if (Fine) e = fmaf(e, 0.69314718f * fmaf(-x, kRest, fmaf(-x, kLog2e, -t)), e);
  const float sum = 1.f + e;
  float a = __builtin_amdgcn_rcpf(sum);
  if (Fine) a = fmaf(fmaf(-sum, a, 1.f), a, a);
  away = e * a;
  return a;
}
template <typename T> constexpr bool kFine = sizeof(T) == 4;

struct Place {
  int b, c, segment, len;  // c: this lane's first channel; len: steps in use
  bool here;
  int wave, row, run;      // the run of a tile that the lane has, row of its wave
};
template <int E> __device__ inline Place place_of(const RecurParams &p, int segments) {
  Place a;
  int index = blockIdx.x;
  const int tile = index % p.tiles;
  index /= p.tiles;
  a.segment = index % segments;
  a.b = index / segments;
  a.c = (tile * kRowLanes + (threadIdx.x & (kRowLanes - 1))) * E;
  a.here = a.c < p.C;
  a.len = p.lengths ? min(max(p.lengths[a.b], 0), p.L) : p.L;
  a.wave = threadIdx.x >> 6, a.row = (threadIdx.x & 63) / kRowLanes;
  a.run = threadIdx.x / kRowLanes;
  return a;
}
// The token of step s (behind the last in use: the place of its zeros)
__device__ inline int64_t token_of(const RecurParams &p, const Place &a, int s) {
  return p.reverse && s < a.len ? a.len - 1 - s : s;
}

// (A, H) of the runs before (Up) or behind a lane's in its wave, and of the whole wave in its
// last (first) row.
template <int E, bool Up>
__device__ inline void wave_scan(int row, float *A, float *H, float *before_a, float *before_h) {
#pragma unroll
  for (int d = 1; d < 64 / kRowLanes; d *= 2) {
    const bool take = Up ? row >= d : row + d < 64 / kRowLanes;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float pa = Up ? __shfl_up(A[e], d * kRowLanes) : __shfl_down(A[e], d * kRowLanes);
      const float ph = Up ? __shfl_up(H[e], d * kRowLanes) : __shfl_down(H[e], d * kRowLanes);
      H[e] = take ? fmaf(A[e], ph, H[e]) : H[e];
      A[e] = take ? A[e] * pa : A[e];
    }
  }
  const bool first = Up ? row == 0 : row == 64 / kRowLanes - 1;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float pa = Up ? __shfl_up(A[e], kRowLanes) : __shfl_down(A[e], kRowLanes);
    const float ph = Up ? __shfl_up(H[e], kRowLanes) : __shfl_down(H[e], kRowLanes);
    before_a[e] = first ? 1.f : pa, before_h[e] = first ? 0.f : ph;
  }
}

// Whole waves' (A, H) of a tile.
template <int E> struct Exchange {
  float a[kWaves][kRowLanes][E], h[kWaves][kRowLanes][E];
};

template <typename T, int E, bool Gated>
__global__ __launch_bounds__(kThreads) void recurrence_forward_kernel(RecurParams p) {
  constexpr int N = kForward;
  __shared__ Exchange<E> both[2];
  const Place at = place_of<E>(p, p.segments);
  const int lane = threadIdx.x & (kRowLanes - 1);
  float carry[E];
#pragma unroll
  for (int e = 0; e < E; e++) carry[e] = 0.f;
  if (at.here) {
    if (p.segments == 1) {
      if (p.initial)
#pragma unroll
        for (int e = 0; e < E; e++) carry[e] = p.initial[(int64_t)at.b * p.C + at.c + e];
    } else {
      // the initial state lies in the last segment's place
      const float *part = p.part + (int64_t)at.b * p.segments * 2 * p.C + at.c;
#pragma unroll
      for (int e = 0; e < E; e++) carry[e] = part[(int64_t)(p.segments - 1) * 2 * p.C + e];
      for (int k = 0; k < at.segment; k++)
#pragma unroll
        for (int e = 0; e < E; e++)
          carry[e] = fmaf(part[(int64_t)k * 2 * p.C + e], carry[e], part[((int64_t)k * 2 + 1) * p.C + e]);
    }
  }
  const T *v = (const T *)p.v + at.b * p.vs[0] + at.c, *f = (const T *)p.f + at.b * p.fs[0] + at.c;
  const T *g = Gated ? (const T *)p.g + at.b * p.gs[0] + at.c : nullptr;
  T *out = (T *)p.out + (int64_t)at.b * p.L * p.C + at.c;
  const int begin = at.segment * p.segment, end = min(p.L, begin + p.segment);
  int turn = 0;
  for (int s0 = begin; s0 < end; s0 += kTile, turn ^= 1) {
    const int s = s0 + at.run * N;
    float a[N][E], u[N][E], A[E], H[E], before_a[E], before_h[E];
    Raw<T, E> z[N];
#pragma unroll
    for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
    Raw<T, E> rv[N], rf[N];
#pragma unroll
    for (int i = 0; i < N; i++)
      if (at.here && s + i < at.len) {
        const int64_t t = token_of(p, at, s + i);
        rv[i].load(v + t * p.vs[1]);
        rf[i].load(f + t * p.fs[1]);
        if (Gated) z[i].load(g + t * p.gs[1]);
      }
#pragma unroll
    for (int i = 0; i < N; i++) {
      const bool live = at.here && s + i < at.len;
#pragma unroll
      for (int e = 0; e < E; e++) {
        float away;
        a[i][e] = logistic<true>(rf[i][e], away);
        u[i][e] = away * rv[i][e];
        if (!live) a[i][e] = 1.f, u[i][e] = 0.f;
        A[e] *= a[i][e], H[e] = fmaf(a[i][e], H[e], u[i][e]);
      }
    }
    wave_scan<E, true>(at.row, A, H, before_a, before_h);
    Exchange<E> &x = both[turn];
    if (at.row == 64 / kRowLanes - 1)
#pragma unroll
      for (int e = 0; e < E; e++) x.a[at.wave][lane][e] = A[e], x.h[at.wave][lane][e] = H[e];
    __syncthreads();
    float h[E];
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (w == at.wave) h[e] = carry[e];
        carry[e] = fmaf(x.a[w][lane][e], carry[e], x.h[w][lane][e]);
      }
    }
#pragma unroll
    for (int e = 0; e < E; e++) h[e] = fmaf(before_a[e], h[e], before_h[e]);
    if (p.states && at.here && s < p.L && s % kSpan == 0)
#pragma unroll
      for (int e = 0; e < E; e++) p.states[((int64_t)at.b * p.spans + s / kSpan) * p.C + at.c + e] = h[e];
#pragma unroll
    for (int i = 0; i < N; i++) {
      float y[E];
#pragma unroll
      for (int e = 0; e < E; e++) {
        h[e] = fmaf(a[i][e], h[e], u[i][e]);
        y[e] = h[e];
        if (Gated) {
          float away;
          const float w = z[i][e];
          y[e] *= w * logistic<kFine<T>>(w, away);
        }
        if (s + i >= at.len) y[e] = 0.f;
      }
      if (at.here && s + i < p.L) put<T, E>(out + token_of(p, at, s + i) * p.C, y);
    }
  }
  if (at.here && at.segment == p.segments - 1 && threadIdx.x < kRowLanes)
#pragma unroll
    for (int e = 0; e < E; e++) p.final[(int64_t)at.b * p.C + at.c + e] = carry[e];
}

// (A, H) of all segments but the last, forward, and of all but the first, backward.
template <typename T, int E, bool Gated, bool Backward>
__global__ __launch_bounds__(kThreads) void recurrence_segments_kernel(RecurParams p) {
  __shared__ Exchange<E> x;
  const Place at = place_of<E>(p, p.segments - 1);
  const int segment = at.segment + (Backward ? 1 : 0), lane = threadIdx.x & (kRowLanes - 1);
  const T *v = (const T *)p.v + at.b * p.vs[0] + at.c, *f = (const T *)p.f + at.b * p.fs[0] + at.c;
  const T *g = Gated ? (const T *)p.g + at.b * p.gs[0] + at.c : nullptr;
  const T *go = (const T *)p.go + (int64_t)at.b * p.L * p.C + at.c;
  const int begin = segment * p.segment, end = min(at.len, begin + p.segment);
  const int each = p.segment / kRuns;  // steps of a run
  float A[E], H[E], before_a[E], before_h[E];
#pragma unroll
  for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
  const int lo = begin + at.run * each, hi = min(end, lo + each);
  if (at.here)
    for (int i = lo; i < hi; i++) {
      const int s = Backward ? hi - 1 - (i - lo) : i;
      const int64_t t = token_of(p, at, s);
      Raw<T, E> rf, rv, rg;
      rf.load(f + t * p.fs[1]);
      if (Backward) rv.load(go + t * p.C);
      else rv.load(v + t * p.vs[1]);
      if (Backward && Gated) rg.load(g + t * p.gs[1]);
#pragma unroll
      for (int e = 0; e < E; e++) {
        float away;
        const float a = logistic<true>(rf[e], away);
        if (Backward) {
          float d = rv[e], rest;
          if (Gated) d *= rg[e] * logistic<kFine<T>>(rg[e], rest);
          H[e] = a * (d + H[e]);
        } else {
          H[e] = fmaf(a, H[e], away * rv[e]);
        }
        A[e] *= a;
      }
    }
  wave_scan<E, !Backward>(at.row, A, H, before_a, before_h);
  if (at.row == (Backward ? 0 : 64 / kRowLanes - 1))
#pragma unroll
    for (int e = 0; e < E; e++) x.a[at.wave][lane][e] = A[e], x.h[at.wave][lane][e] = H[e];
  __syncthreads();
  if (threadIdx.x >= kRowLanes || !at.here) return;
#pragma unroll
  for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
  for (int k = 0; k < kWaves; k++) {
    const int w = Backward ? kWaves - 1 - k : k;
#pragma unroll
    for (int e = 0; e < E; e++) {
      H[e] = fmaf(x.a[w][lane][e], H[e], x.h[w][lane][e]);
      A[e] *= x.a[w][lane][e];
    }
  }
  float *part = p.part + (int64_t)at.b * p.segments * 2 * p.C + at.c;
#pragma unroll
  for (int e = 0; e < E; e++) {
    part[(int64_t)segment * 2 * p.C + e] = A[e], part[((int64_t)segment * 2 + 1) * p.C + e] = H[e];
    // the initial state, in the place of the last segment's A: `final` may be the same memory
    if (!Backward && segment == 0)
      part[(int64_t)(p.segments - 1) * 2 * p.C + e] = p.initial ? p.initial[(int64_t)at.b * p.C + at.c + e] : 0.f;
  }
}

template <typename T, int E, bool Gated>
__global__ __launch_bounds__(kThreads) void recurrence_backward_kernel(RecurParams p) {
  constexpr int N = kBackward;
  __shared__ Exchange<E> ahead[2], back[2];
  const Place at = place_of<E>(p, p.segments);
  const int lane = threadIdx.x & (kRowLanes - 1);
  float carry[E];
#pragma unroll
  for (int e = 0; e < E; e++) carry[e] = 0.f;
  if (at.here) {
    if (p.gfinal)
#pragma unroll
      for (int e = 0; e < E; e++) carry[e] = p.gfinal[(int64_t)at.b * p.C + at.c + e];
    const float *part = p.part + (int64_t)at.b * p.segments * 2 * p.C + at.c;
    for (int k = p.segments - 1; k > at.segment; k--)
#pragma unroll
      for (int e = 0; e < E; e++)
        carry[e] = fmaf(part[(int64_t)k * 2 * p.C + e], carry[e], part[((int64_t)k * 2 + 1) * p.C + e]);
  }
  const T *v = (const T *)p.v + at.b * p.vs[0] + at.c, *f = (const T *)p.f + at.b * p.fs[0] + at.c;
  const T *g = Gated ? (const T *)p.g + at.b * p.gs[0] + at.c : nullptr;
  const int64_t dense = (int64_t)at.b * p.L * p.C + at.c;
  const T *go = (const T *)p.go + dense;
  T *gv = (T *)p.gv, *gf = (T *)p.gf, *gg = (T *)p.gg;
  const int begin = at.segment * p.segment, end = min(p.L, begin + p.segment);
  int turn = 0;
  for (int s0 = begin + (end - begin - 1) / kSpan * kSpan; s0 >= begin; s0 -= kSpan, turn ^= 1) {
    const int s = s0 + at.run * N;
    float a[N][E], away[N][E], h[N][E], d[N][E], A[E], H[E], before_a[E], before_h[E];
    Raw<T, E> rv[N], rf[N], rg[N], ro[N];
    float state[E];
    if (at.here)
#pragma unroll
      for (int e = 0; e < E; e++) state[e] = p.states[((int64_t)at.b * p.spans + s0 / kSpan) * p.C + at.c + e];
#pragma unroll
    for (int i = 0; i < N; i++)
      if (at.here && s + i < at.len) {
        const int64_t t = token_of(p, at, s + i);
        rv[i].load(v + t * p.vs[1]);
        rf[i].load(f + t * p.fs[1]);
        if (Gated) rg[i].load(g + t * p.gs[1]);
        ro[i].load(go + t * p.C);
      }
#pragma unroll
    for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const bool live = at.here && s + i < at.len;
#pragma unroll
      for (int e = 0; e < E; e++) {
        a[i][e] = logistic<true>(rf[i][e], away[i][e]);
        float u = away[i][e] * rv[i][e];
        if (!live) a[i][e] = 1.f, u = 0.f;
        A[e] *= a[i][e], H[e] = fmaf(a[i][e], H[e], u);
      }
    }
    wave_scan<E, true>(at.row, A, H, before_a, before_h);
    Exchange<E> &x = ahead[turn];
    if (at.row == 64 / kRowLanes - 1)
#pragma unroll
      for (int e = 0; e < E; e++) x.a[at.wave][lane][e] = A[e], x.h[at.wave][lane][e] = H[e];
    __syncthreads();
    for (int w = 0; w < at.wave; w++)
#pragma unroll
      for (int e = 0; e < E; e++) state[e] = fmaf(x.a[w][lane][e], state[e], x.h[w][lane][e]);
#pragma unroll
    for (int e = 0; e < E; e++) state[e] = fmaf(before_a[e], state[e], before_h[e]);
    // from here on h: the state before a step
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < E; e++) {
        h[i][e] = state[e];
        state[e] = fmaf(a[i][e], state[e], away[i][e] * rv[i][e]);
        float rest;
        d[i][e] = ro[i][e];
        if (Gated) d[i][e] *= rg[i][e] * logistic<kFine<T>>(rg[i][e], rest);
        if (!(at.here && s + i < at.len)) d[i][e] = 0.f;
      }
#pragma unroll
    for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
#pragma unroll
    for (int i = N - 1; i >= 0; i--)
#pragma unroll
      for (int e = 0; e < E; e++) H[e] = a[i][e] * (d[i][e] + H[e]), A[e] *= a[i][e];
    wave_scan<E, false>(at.row, A, H, before_a, before_h);
    Exchange<E> &y = back[turn];
    if (at.row == 0)
#pragma unroll
      for (int e = 0; e < E; e++) y.a[at.wave][lane][e] = A[e], y.h[at.wave][lane][e] = H[e];
    __syncthreads();
    float push[E];
#pragma unroll
    for (int w = kWaves - 1; w >= 0; w--)
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (w == at.wave) push[e] = carry[e];
        carry[e] = fmaf(y.a[w][lane][e], carry[e], y.h[w][lane][e]);
      }
#pragma unroll
    for (int e = 0; e < E; e++) push[e] = fmaf(before_a[e], push[e], before_h[e]);
#pragma unroll
    for (int i = N - 1; i >= 0; i--) {
      const bool live = s + i < at.len;
      float y1[E], y2[E], y3[E];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float D = d[i][e] + push[e], x = rv[i][e];
        push[e] = a[i][e] * D;
        y1[e] = away[i][e] * D;
        y2[e] = D * (h[i][e] - x) * (a[i][e] * away[i][e]);
        if (Gated) {
          float rest;
          const float z = rg[i][e], sg = logistic<kFine<T>>(z, rest);
          y3[e] = ro[i][e] * fmaf(a[i][e], h[i][e], away[i][e] * x) * (sg * fmaf(z, rest, 1.f));
        }
        if (!live) y1[e] = y2[e] = y3[e] = 0.f;
      }
      if (at.here && s + i < p.L) {
        const int64_t to = dense + token_of(p, at, s + i) * p.C;
        if (gv) put<T, E>(gv + to, y1);
        if (gf) put<T, E>(gf + to, y2);
        if (Gated && gg) put<T, E>(gg + to, y3);
      }
    }
  }
  if (p.ginitial && at.here && at.segment == 0 && threadIdx.x < kRowLanes)
#pragma unroll
    for (int e = 0; e < E; e++) p.ginitial[(int64_t)at.b * p.C + at.c + e] = carry[e];
}

// Up to kFew steps: a thread walks them all.
template <typename T, int E, bool Gated>
__global__ __launch_bounds__(256) void recurrence_few_kernel(RecurParams p, int64_t words) {
  const int64_t index = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (index >= words) return;
  const int row = p.C / E;
  Place at;
  at.b = (int)(index / row), at.c = (int)(index % row) * E;
  at.len = p.lengths ? min(max(p.lengths[at.b], 0), p.L) : p.L;
  float h[E];
  const int64_t state = (int64_t)at.b * p.C + at.c;
#pragma unroll
  for (int e = 0; e < E; e++) h[e] = p.initial ? p.initial[state + e] : 0.f;
  if (p.states)
#pragma unroll
    for (int e = 0; e < E; e++) p.states[state + e] = h[e];
  for (int s = 0; s < p.L; s++) {
    const int64_t t = token_of(p, at, s);
    float y[E];
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = 0.f;
    if (s < at.len) {
      Raw<T, E> rv, rf, rg;
      rv.load((const T *)p.v + at.b * p.vs[0] + t * p.vs[1] + at.c);
      rf.load((const T *)p.f + at.b * p.fs[0] + t * p.fs[1] + at.c);
      if (Gated) rg.load((const T *)p.g + at.b * p.gs[0] + t * p.gs[1] + at.c);
#pragma unroll
      for (int e = 0; e < E; e++) {
        float away;
        const float a = logistic<true>(rf[e], away);
        h[e] = fmaf(a, h[e], away * rv[e]);
        y[e] = h[e];
        if (Gated) y[e] *= rg[e] * logistic<kFine<T>>(rg[e], away);
      }
    }
    put<T, E>((T *)p.out + ((int64_t)at.b * p.L + t) * p.C + at.c, y);
  }
#pragma unroll
  for (int e = 0; e < E; e++) p.final[state + e] = h[e];
}

// ---- host ----

int check_desc(const mcx_recurrence_desc *d, int dtype) {
  if (!d) return MCX_E_NULL;
  if (dtype != MCX_F32 && dtype != MCX_BF16) return MCX_E_DTYPE;
  if (d->B < 0 || d->L < 0 || d->C < 1 || d->L > 0x3fffffff || d->C > (1 << 24) || d->B > (1 << 24) ||
      d->B * ((d->C + 15) / 16) > (1 << 21))
    return MCX_E_SHAPE;
  return MCX_OK;
}
int word_of(const mcx_recurrence_desc *d, int size, bool gated, uint64_t addresses) {
  uint64_t bits = addresses;
  for (int k = 0; k < 2; k++) {
    if ((k ? d->L : d->B) <= 1) continue;
    bits |= (uint64_t)d->v_stride[k] * size | (uint64_t)d->f_stride[k] * size;
    if (gated) bits |= (uint64_t)d->g_stride[k] * size;
  }
  for (int w : {4, 2})
    if (d->C % w == 0 && bits % (w * size) == 0) return w;
  return 1;
}
// Segments of the steps: workgroups of `word` channels a lane are made kGroups, of two tiles at least.
int segment_of(const mcx_recurrence_desc *d, int word) {
  const int64_t tiles = (d->C + kRowLanes * word - 1) / (kRowLanes * word), groups = d->B * tiles;
  int64_t n = groups * 4 >= kGroups * 3 ? 1 : (kGroups + groups - 1) / std::max<int64_t>(1, groups);
  n = std::max<int64_t>(1, std::min(n, d->L / (2 * kTile)));
  const int64_t each = (d->L + n - 1) / n;
  return (int)((each + kTile - 1) / kTile * kTile);
}
size_t part_bytes(const mcx_recurrence_desc *d) {
  // (of the widest word, whose workgroups are the fewest)
  int64_t n = 1;
  for (int w : {1, 2, 4}) {
    const int each = segment_of(d, w);
    n = std::max<int64_t>(n, (d->L + each - 1) / each);
  }
  return n > 1 ? (size_t)(d->B * n * 2 * d->C) * sizeof(float) : 0;
}
RecurParams params_of(const mcx_recurrence_desc *d, int word) {
  RecurParams p = {};
  for (int k = 0; k < 2; k++) p.vs[k] = d->v_stride[k], p.fs[k] = d->f_stride[k], p.gs[k] = d->g_stride[k];
  p.L = (int)d->L, p.C = (int)d->C;
  p.tiles = (int)((d->C + kRowLanes * word - 1) / (kRowLanes * word));
  p.segment = segment_of(d, word);
  p.segments = (int)((d->L + p.segment - 1) / p.segment);
  p.spans = (int)((d->L + kSpan - 1) / kSpan);
  p.reverse = d->reverse != 0;
  return p;
}

template <typename T, int E, bool Gated>
int forward(const RecurParams &p, int64_t B, hipStream_t s) {
  if (p.L <= kFew) {
    const int64_t words = B * (p.C / E);
    hipLaunchKernelGGL((recurrence_few_kernel<T, E, Gated>), dim3((unsigned)((words + 255) / 256)), dim3(256),
                       0, s, p, words);
    MCX_HIP_CHECK_LAUNCH();
    return MCX_OK;
  }
  const unsigned groups = (unsigned)(B * p.tiles);
  if (p.segments > 1) {
    hipLaunchKernelGGL((recurrence_segments_kernel<T, E, false, false>), dim3(groups * (p.segments - 1)),
                       dim3(kThreads), 0, s, p);
    MCX_HIP_CHECK_LAUNCH();
  }
  hipLaunchKernelGGL((recurrence_forward_kernel<T, E, Gated>), dim3(groups * p.segments), dim3(kThreads), 0,
                     s, p);
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}
template <typename T, int E, bool Gated>
int backward(const RecurParams &p, int64_t B, hipStream_t s) {
  const unsigned groups = (unsigned)(B * p.tiles);
  if (p.segments > 1) {
    hipLaunchKernelGGL((recurrence_segments_kernel<T, E, Gated, true>), dim3(groups * (p.segments - 1)),
                       dim3(kThreads), 0, s, p);
    MCX_HIP_CHECK_LAUNCH();
  }
  hipLaunchKernelGGL((recurrence_backward_kernel<T, E, Gated>), dim3(groups * p.segments), dim3(kThreads), 0,
                     s, p);
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}
template <typename T, bool Forward>
int launch(const RecurParams &p, int64_t B, int word, hipStream_t s) {
#define MCX_RECUR(E)                                                                                 \
  (Forward ? (p.g ? forward<T, E, true>(p, B, s) : forward<T, E, false>(p, B, s))                    \
           : (p.g ? backward<T, E, true>(p, B, s) : backward<T, E, false>(p, B, s)))
  return word == 4 ? MCX_RECUR(4) : word == 2 ? MCX_RECUR(2) : MCX_RECUR(1);
#undef MCX_RECUR
}

}  // namespace
}  // namespace mcx

extern "C" {

int64_t mcx_gated_recurrence_spans(int64_t L) { return L < 0 ? 0 : (L + mcx::kSpan - 1) / mcx::kSpan; }

size_t mcx_gated_recurrence_workspace(const mcx_recurrence_desc *desc, int dtype) {
  using namespace mcx;
  if (check_desc(desc, dtype) != MCX_OK || !desc->B || !desc->L) return 0;
  return part_bytes(desc);
}

int mcx_gated_recurrence_forward(const void *value, const void *forget, const void *gate,
                                 const float *initial, const int32_t *lengths, void *out, float *final,
                                 float *states, void *workspace, size_t workspace_bytes,
                                 const mcx_recurrence_desc *desc, int dtype, void *stream) {
  using namespace mcx;
  if (int e = check_desc(desc, dtype)) return e;
  if (!desc->B || !desc->L) return MCX_OK;
  if (!value || !forget || !out || !final) return MCX_E_NULL;
  const size_t need = part_bytes(desc);
  if (need && (!workspace || workspace_bytes < need)) return MCX_E_WORKSPACE;
  const int word = word_of(desc, dtype == MCX_BF16 ? 2 : 4, gate != nullptr,
                           (uintptr_t)value | (uintptr_t)forget | (uintptr_t)gate | (uintptr_t)out);
  RecurParams p = params_of(desc, word);
  p.v = value, p.f = forget, p.g = gate, p.initial = initial, p.lengths = lengths;
  p.out = out, p.final = final, p.states = states, p.part = (float *)workspace;
  return dtype == MCX_BF16 ? launch<__bf16, true>(p, desc->B, word, (hipStream_t)stream)
                           : launch<float, true>(p, desc->B, word, (hipStream_t)stream);
}

int mcx_gated_recurrence_backward(const void *gout, const float *gfinal, const void *value,
                                  const void *forget, const void *gate, const float *states,
                                  const int32_t *lengths, void *gvalue, void *gforget, void *ggate,
                                  float *ginitial, void *workspace, size_t workspace_bytes,
                                  const mcx_recurrence_desc *desc, int dtype, void *stream) {
  using namespace mcx;
  if (int e = check_desc(desc, dtype)) return e;
  if (!desc->B || !desc->L) return MCX_OK;
  if (!gout || !value || !forget || !states) return MCX_E_NULL;
  const size_t need = part_bytes(desc);
  if (need && (!workspace || workspace_bytes < need)) return MCX_E_WORKSPACE;
  const int word = word_of(desc, dtype == MCX_BF16 ? 2 : 4, gate != nullptr,
                           (uintptr_t)value | (uintptr_t)forget | (uintptr_t)gate | (uintptr_t)gout |
                               (uintptr_t)gvalue | (uintptr_t)gforget | (uintptr_t)ggate);
  RecurParams p = params_of(desc, word);
  p.v = value, p.f = forget, p.g = gate, p.go = gout, p.gfinal = gfinal, p.lengths = lengths;
  p.gv = gvalue, p.gf = gforget, p.gg = ggate, p.ginitial = ginitial;
  p.states = const_cast<float *>(states), p.part = (float *)workspace;
  return dtype == MCX_BF16 ? launch<__bf16, false>(p, desc->B, word, (hipStream_t)stream)
                           : launch<float, false>(p, desc->B, word, (hipStream_t)stream);
}

}  // extern "C"
