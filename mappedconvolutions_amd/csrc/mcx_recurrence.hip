// A gated linear recurrence along a sequence, and its gradients.
//
//   a_t = sigmoid(f_t),  h_t = a_t h_{t-1} + (1 - a_t) v_t,  out_t = h_t g_t sigmoid(g_t)  (or h_t)
//   D_t = d_t + p_t,  d_t = go_t g_t sigmoid(g_t),  p_{t-1} = a_t D_t      (p_L: the final state's gradient)
//   gv = (1 - a) D,  gf = a (1 - a) (h_{t-1} - v) D,  gg = go h silu'(g),  gh_0 = p_0
//
// Bound by memory: 4 streams forward, 7 backward, and a few dozen operations a value.  Channels are
// independent; a workgroup has 16 lanes' words of them and walks the steps in tiles, each lane with a run
// of steps of its own and the next tile's values under way.  h_t of a run is A h + H of the state before
// it; the lanes' (A, H) are joined within a wave by lane exchange and between waves through LDS, so a tile
// costs one barrier forward and two backward.  States are kept for the gradients every kSpan steps and the
// others recomputed.
//   Where sequences and channels are too few to fill the card the steps are cut into segments, and a first
// launch sums up the (A, H) of each: it reads two streams of four, or three of seven, a second time.  (Tiles
// that wait for the state of the tile before them read everything once and took longer: 2 sequences of 32768
// steps of 1024 bf16 channels forward 165 us and backward 312.)  Few steps have a tile of as few or a thread to
// themselves, few channels four lanes a row instead of 16.
//   Measured in bf16 with an output gate, forward and gradients: 2048 sequences of 512 steps of 128 channels 214
// and 384 us, 5.0 and 4.9 TB/s; 2 of 32768 steps of 1024 channels 51 + 119 and 65 + 212 us, 4.7 and 4.8 TB/s
// with the second read (vector units 63 % of the time).  One step of 16 x 1024 channels 3.4 us.
#include <algorithm>
#include <type_traits>

#include "mcx_mfma_common.h"

namespace mcx {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kRowLanes = 16;           // lanes of a step's channels
constexpr int kNarrowLanes = 4;         // the same where channels are few
// Runs of steps of a tile
template <int Lanes> constexpr int kRuns = kThreads / Lanes;
// Steps of a run: 16 values a lane, 8 in single precision (whose words hold 2) and where no words can be read, so
// that all fits the registers.
constexpr int run_steps(int word, int size) { return word == 4 || size == 4 ? 4 : 8; }
constexpr int kSpan = kRuns<kRowLanes> * 4;  // steps from one kept state to the next, a part of every tile
// Steps that a thread walks alone, forward (8192 sequences of 16 steps of 256 bf16 channels 54 us, in a tile 74; 512 of
// 32 steps 20 and 13), and backward, which holds them all in registers (20000 of 8 steps of 66, forward and gradients,
// 64 and 154; 1500 of one step of 1661 35 and 350).
constexpr int kFew = 16, kFewBackward = 8;
// Workgroups aimed at by segments: as many as are resident at a time (forward, float32 backward, bf16 back-
// ward; 768 there: 2 sequences of 32768 steps of 1024 channels 440 -> 542 us), and by the parts of the first
// launch; workgroups from which on there are no segments (16 sequences of 4096 steps of 1024 bf16 channels, 256 of
// them, 388 us with and 403 without; 24 of 3000, 384 of them, 470 and 430).
constexpr int kGroups = 768, kGroupsBf16Backward = 512, kSums = 8192, kAlone = 257;
constexpr int kWideRow = 40;           // words of a row from which on the first launch reads rows of 64 lanes
// Tensors whose results would push out of the last-level cache what is read a second time (2 sequences of
// 32768 steps of 1024 channels 473 -> 440 us); only whole lines are written past it (rows of 360 bytes: 50 -> 66).
constexpr int64_t kPassingBytes = 64 << 20;
constexpr int kLine = 128;

struct RecurParams {
  const void *v, *f, *g, *go;
  const float *initial, *gfinal;
  const int32_t *lengths;
  void *out, *gv, *gf, *gg;
  float *final, *ginitial, *states;  // states [B, ceil(L / kSpan), C]
  float *part;                       // [B, parts + 1, 2, C]: A and H of a part; the initial state
  int64_t vs[2], fs[2], gs[2];       // strides of sequence and step
  int L, C, tiles;                   // tiles of channels
  int segments, segment;             // steps of a segment
  int parts, each, share;            // parts of all steps, their steps, parts of a segment
  int spans, reverse;
  int lanes;                         // of a row
  int together;                      // neighbours go to the same XCD
};

template <typename T, int E> struct Raw {
  typedef T Vec __attribute__((ext_vector_type(E)));
  Vec x;
  __device__ inline void load(const T *p) { x = *(const Vec *)p; }
  __device__ inline void fill(float v) { x = Vec((T)v); }
  __device__ inline float operator[](int e) const { return (float)x[e]; }
};
template <typename T> struct Raw<T, 1> {
  T x;
  __device__ inline void load(const T *p) { x = *p; }
  __device__ inline void fill(float v) { x = (T)v; }
  __device__ inline float operator[](int) const { return (float)x; }
};
// Passing: past the cache
template <typename T, int E, bool Passing = false> __device__ inline void put(T *p, const float *v) {
  if constexpr (E == 1) {
    *p = (T)v[0];
  } else {
    typedef T Vec __attribute__((ext_vector_type(E)));
    Vec w;
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = (T)v[e];
    if (Passing) __builtin_nontemporal_store(w, (Vec *)p);
    else *(Vec *)p = w;
  }
}

// sigmoid(x), and in `away` 1 - sigmoid(x) without its cancellation.  The reciprocal is corrected once: the
// errors of factors add up over hundreds of steps.  Fine: what the exponent's rounding took is put back too.
template <bool Fine> __device__ inline float exponential(float x) {  // e^-x
  constexpr float kLog2e = 1.44269504f, kRest = 1.92596299e-8f;
  const float t = -x * kLog2e, e = __builtin_amdgcn_exp2f(t);
  return Fine ? fmaf(e, 0.69314718f * fmaf(-x, kRest, fmaf(-x, kLog2e, -t)), e) : e;
}
__device__ inline float reciprocal(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return fmaf(fmaf(-x, r, 1.f), r, r);
}
template <bool Fine> __device__ inline float logistic(float x, float &away) {
  x = __builtin_elementwise_maximum(x, -80.f);  // (what is no number stays none)
  if (Fine) x = __builtin_elementwise_minimum(x, 200.f);
  const float e = exponential<Fine>(x), a = reciprocal(1.f + e);
  away = e * a;
  return a;
}
// The same for an output gate, which nothing adds up over and which is multiplied by it: nothing is left of it
// where e^-x leaves the range (x below -87, where x sigmoid(x) is above -1.5e-36).
template <bool Fine> __device__ inline float sigmoid(float x) {
  if (!Fine) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504f));
  const float y = __builtin_elementwise_minimum(__builtin_elementwise_maximum(x, -87.f), 200.f);
  return x < -87.f ? 0.f : reciprocal(1.f + exponential<true>(y));
}
template <typename T> constexpr bool kFine = sizeof(T) == 4;

struct Place {
  int b, segment, len;  // len: steps in use
  int c;                // this lane's first channel
  bool here;
};
// (what all lanes have in common in scalar registers: the addresses are these, and 32 bits a lane)
template <int E, int RowLanes>
__device__ inline Place place_of(const RecurParams &p, int index, int segments) {
  Place a;
  if (p.together) index = xcd_contiguous_tile(index, gridDim.x);
  const int columns = gridDim.x / segments;  // (neighbours have the same steps)
  a.segment = index / columns;
  index -= a.segment * columns;
  a.b = index / p.tiles;
  a.c = ((index - a.b * p.tiles) * RowLanes + (threadIdx.x & (RowLanes - 1))) * E;
  a.here = a.c < p.C;
  a.c = min(a.c, p.C - E);  // (lanes behind the last channel read it too, and write nothing)
  a.len = p.lengths ? __builtin_amdgcn_readfirstlane(min(max(p.lengths[a.b], 0), p.L)) : p.L;
  return a;
}
// The token of step s (behind the last in use: the place of its zeros)
__device__ inline int64_t token_of(const RecurParams &p, const Place &a, int s) {
  return p.reverse && s < a.len ? a.len - 1 - s : s;
}
// A tile of Tile steps in a tensor: the address of its first token, and from there in bytes that of a run's
// first step and the way to the next step.
template <typename T> struct Rows {
  const char *base;
  unsigned first, step;
  template <int Tile>
  static __device__ inline Rows of(const RecurParams &p, const Place &a, int s0, const void *x,
                                   int64_t sequence, int64_t stride, int j) {
    const int64_t t0 = p.reverse ? (int64_t)a.len - Tile - s0 : s0;
    const unsigned bytes = (unsigned)stride * (unsigned)sizeof(T);
    Rows r;
    r.base = (const char *)x + (a.b * sequence + t0 * stride) * (int64_t)sizeof(T);
    r.first = (unsigned)(p.reverse ? Tile - 1 - j : j) * bytes + (unsigned)a.c * (unsigned)sizeof(T);
    r.step = p.reverse ? 0u - bytes : bytes;
    return r;
  }
  __device__ inline T *at(int i) const { return (T *)(base + (first + (unsigned)i * step)); }
};

// Zeros at those of steps s to s + n that are not in use.
template <typename T, int E>
__device__ inline void put_zeros(const RecurParams &p, const Place &a, void *x, int s, int n) {
  if (!a.here) return;
  const float zeros[E] = {};
#pragma unroll 1
  for (int i = 0; i < n; i++)
    if (s + i >= a.len && s + i < p.L) put<T, E>((T *)x + ((int64_t)a.b * p.L + s + i) * p.C + a.c, zeros);
}

// (A, H) of the runs before (Up) or behind a lane's in its wave, and of the whole wave in its
// last (first) row.
template <int E, int RowLanes, bool Up>
__device__ inline void wave_scan(int row, float *A, float *H, float *before_a, float *before_h) {
#pragma unroll
  for (int d = 1; d < 64 / RowLanes; d *= 2) {
    const bool take = Up ? row >= d : row + d < 64 / RowLanes;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float pa = Up ? __shfl_up(A[e], d * RowLanes) : __shfl_down(A[e], d * RowLanes);
      const float ph = Up ? __shfl_up(H[e], d * RowLanes) : __shfl_down(H[e], d * RowLanes);
      H[e] = take ? fmaf(A[e], ph, H[e]) : H[e];
      A[e] = take ? A[e] * pa : A[e];
    }
  }
  const bool first = Up ? row == 0 : row == 64 / RowLanes - 1;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float pa = Up ? __shfl_up(A[e], RowLanes) : __shfl_down(A[e], RowLanes);
    const float ph = Up ? __shfl_up(H[e], RowLanes) : __shfl_down(H[e], RowLanes);
    before_a[e] = first ? 1.f : pa, before_h[e] = first ? 0.f : ph;
  }
}

// Whole waves' (A, H) of a tile.
template <int E, int RowLanes> struct Exchange {
  float a[kWaves][RowLanes][E], h[kWaves][RowLanes][E];
};

// The state that a segment begins with: (A, H) of the parts before it (Backward: behind it) over `carry`.  A row of
// lanes goes over some of them, then all over the rows.
template <int E, int RowLanes> struct Ranges {
  float a[kRuns<RowLanes>][RowLanes][E], h[kRuns<RowLanes>][RowLanes][E];
};
template <int E, int RowLanes, bool Backward>
__device__ inline void carry_in(const RecurParams &p, const Place &at, Ranges<E, RowLanes> &x, float *carry) {
  const int lane = threadIdx.x & (RowLanes - 1), row = threadIdx.x / RowLanes;
  const int n = Backward ? max(0, p.parts - (at.segment + 1) * p.share) : at.segment * p.share;
  constexpr int kRows = kRuns<RowLanes>;
  const int each = (n + kRows - 1) / kRows;
  const float *part = p.part + (int64_t)at.b * (p.parts + 1) * 2 * p.C + at.c;
  float A[E], H[E];
#pragma unroll
  for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
#pragma unroll 4
  for (int i = row * each; i < min(n, (row + 1) * each); i++) {
    const float *of = part + (int64_t)(Backward ? p.parts - 1 - i : i) * 2 * p.C;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float a = of[e];
      H[e] = fmaf(a, H[e], of[p.C + e]);
      A[e] *= a;
    }
  }
#pragma unroll
  for (int e = 0; e < E; e++) x.a[row][lane][e] = A[e], x.h[row][lane][e] = H[e];
  __syncthreads();
#pragma unroll 4
  for (int k = 0; k < kRows; k++)
#pragma unroll
    for (int e = 0; e < E; e++) carry[e] = fmaf(x.a[k][lane][e], carry[e], x.h[k][lane][e]);
}

// (A, H) of every part but those of the last segment, forward, and of the first, backward.  As in the tiles what
// values are multiplied by is at most 1: the largest overflow nothing, whatever the gates.
template <typename T, int E, int RowLanes, bool Gated, bool Backward>
__global__ __launch_bounds__(kThreads) void recurrence_parts_kernel(RecurParams p) {
  constexpr int N = 4;  // steps under way
  __shared__ float xa[kWaves][RowLanes][E], xh[kWaves][RowLanes][E];
  const Place at = place_of<E, RowLanes>(p, blockIdx.x, Backward ? p.parts - p.share : (p.segments - 1) * p.share);
  const int which = at.segment + (Backward ? p.share : 0), lane = threadIdx.x & (RowLanes - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = (threadIdx.x & 63) / RowLanes;
  const int begin = which * p.each, end = min(at.len, begin + p.each);
  const int run = p.each / (kThreads / RowLanes);  // steps of a run
  const int lo = begin + threadIdx.x / RowLanes * run, hi = min(end, lo + run);
  const int way = p.reverse != Backward ? -1 : 1;
  float A[E], H[E];
#pragma unroll
  for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
  // from the run's first step on, or backward from its last
  const int64_t t0 = token_of(p, at, Backward ? max(lo, hi - 1) : lo);
  const T *f = (const T *)p.f + at.b * p.fs[0] + t0 * p.fs[1] + at.c;
  const T *v = Backward ? (const T *)p.go + ((int64_t)at.b * p.L + t0) * p.C + at.c
                        : (const T *)p.v + at.b * p.vs[0] + t0 * p.vs[1] + at.c;
  const T *g = Backward && Gated ? (const T *)p.g + at.b * p.gs[0] + t0 * p.gs[1] + at.c : nullptr;
  const int64_t fs = way * p.fs[1], vs = way * (Backward ? (int64_t)p.C : p.vs[1]), gs = way * p.gs[1];
  const auto steps = [&](auto count, int i) {
    constexpr int K = decltype(count)::value;
    Raw<T, E> rf[K], rv[K], rg[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
      rf[k].load(f + (i + k) * fs);
      rv[k].load(v + (i + k) * vs);
      if (Backward && Gated) rg[k].load(g + (i + k) * gs);
    }
    const auto added = [&](int k, int e) {
      const float x = rv[k][e];
      return Backward && Gated ? x * (rg[k][e] * sigmoid<kFine<T>>(rg[k][e])) : x;
    };
    // one reciprocal for K steps: with x = e^-f the product of all 1 / a is D, and a value's share of the state
    // x (backward: 1) times D of the steps before it over the last D, at most 1
    float share[K][E], D[E];
    bool fits = true;
#pragma unroll
    for (int e = 0; e < E; e++) {
      D[e] = 1.f;
#pragma unroll
      for (int k = 0; k < K; k++) {
        float f = __builtin_elementwise_maximum((float)rf[k][e], -80.f);
        if (kFine<T>) f = __builtin_elementwise_minimum(f, 200.f);
        const float x = exponential<kFine<T>>(f);
        share[k][e] = Backward ? D[e] : x * D[e];
        D[e] = fmaf(x, D[e], D[e]);
      }
      fits &= D[e] <= 0x1p120f;
    }
    if (fits) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float r = reciprocal(D[e]);
        H[e] *= r, A[e] *= r;
#pragma unroll
        for (int k = 0; k < K; k++) H[e] = fmaf(share[k][e] * r, added(k, e), H[e]);
      }
      return;
    }
    // (several shut gates, or one that is no number: step by step)
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int e = 0; e < E; e++) {
        float away;
        const float a = logistic<kFine<T>>(rf[k][e], away);
        H[e] = Backward ? a * (added(k, e) + H[e]) : fmaf(a, H[e], away * added(k, e));
        A[e] *= a;
      }
  };
  int i = 0;
  for (; i + N <= hi - lo; i += N) steps(std::integral_constant<int, N>(), i);
  for (; i < hi - lo; i++) steps(std::integral_constant<int, 1>(), i);
  if constexpr (RowLanes < 64) {
    float before_a[E], before_h[E];
    wave_scan<E, RowLanes, !Backward>(row, A, H, before_a, before_h);
  }
  if (row == (Backward ? 0 : 64 / RowLanes - 1))
#pragma unroll
    for (int e = 0; e < E; e++) xa[wave][lane][e] = A[e], xh[wave][lane][e] = H[e];
  __syncthreads();
  if (threadIdx.x >= RowLanes || !at.here) return;
#pragma unroll
  for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
#pragma unroll
  for (int k = 0; k < kWaves; k++) {
    const int w = Backward ? kWaves - 1 - k : k;
#pragma unroll
    for (int e = 0; e < E; e++) {
      H[e] = fmaf(xa[w][lane][e], H[e], xh[w][lane][e]);
      A[e] *= xa[w][lane][e];
    }
  }
  float *part = p.part + (int64_t)at.b * (p.parts + 1) * 2 * p.C + at.c;
#pragma unroll
  for (int e = 0; e < E; e++) {
    part[(int64_t)which * 2 * p.C + e] = A[e], part[((int64_t)which * 2 + 1) * p.C + e] = H[e];
    // (the initial state too, since `final` may be the same memory)
    if (!Backward && which == 0)
      part[(int64_t)p.parts * 2 * p.C + e] = p.initial ? p.initial[(int64_t)at.b * p.C + at.c + e] : 0.f;
  }
}

template <typename T, int E, int N, int RowLanes, bool Gated, bool Passing>
__global__ __launch_bounds__(kThreads, 3) void recurrence_forward_kernel(RecurParams p) {
  constexpr int kTile = kRuns<RowLanes> * N;
  __shared__ Exchange<E, RowLanes> both[2];
  __shared__ Ranges<E, RowLanes> ranges;
  const int lane = threadIdx.x & (RowLanes - 1), run = threadIdx.x / RowLanes;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = (threadIdx.x & 63) / RowLanes;
  // (from the end, which the first launch read last)
  const Place at = place_of<E, RowLanes>(p, gridDim.x - 1 - blockIdx.x, p.segments);
  const int begin = at.segment * p.segment, end = min(p.L, begin + p.segment);
  Raw<T, E> rv[N], rf[N], rz[N];
  // the tile's values, the next one's while this one is worked on; gates when the tile's are used up
  const auto load = [&](int s0) {
    const auto v = Rows<T>::template of<kTile>(p, at, s0, p.v, p.vs[0], p.vs[1], run * N);
    const auto f = Rows<T>::template of<kTile>(p, at, s0, p.f, p.fs[0], p.fs[1], run * N);
    const int s = s0 + run * N;
    if (s0 + kTile <= at.len) {
#pragma unroll
      for (int i = 0; i < N; i++) rv[i].load(v.at(i)), rf[i].load(f.at(i));
      return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      // a step that leaves the state as it is
      rv[i].fill(0.f), rf[i].fill(__builtin_inff());
      if (s + i < at.len) rv[i].load(v.at(i)), rf[i].load(f.at(i));
    }
  };
  const auto load_gates = [&](int s0) {
    if (!Gated) return;
    const auto g = Rows<T>::template of<kTile>(p, at, s0, p.g, p.gs[0], p.gs[1], run * N);
    const int s = s0 + run * N;
    if (s0 + kTile <= at.len) {
#pragma unroll
      for (int i = 0; i < N; i++) rz[i].load(g.at(i));
      return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      rz[i].fill(0.f);
      if (s + i < at.len) rz[i].load(g.at(i));
    }
  };
  load(begin);
  load_gates(begin);
  float carry[E];
#pragma unroll
  for (int e = 0; e < E; e++) carry[e] = 0.f;
  if (p.segments > 1) {
#pragma unroll
    for (int e = 0; e < E; e++)
      carry[e] = p.part[((int64_t)at.b * (p.parts + 1) + p.parts) * 2 * p.C + at.c + e];
    carry_in<E, RowLanes, false>(p, at, ranges, carry);
  } else if (p.initial) {
#pragma unroll
    for (int e = 0; e < E; e++) carry[e] = p.initial[(int64_t)at.b * p.C + at.c + e];
  }
  int turn = 0;
  for (int s0 = begin; s0 < end; s0 += kTile, turn ^= 1) {
    const int s = s0 + run * N;
    const bool whole = s0 + kTile <= at.len;
    float a[N][E], u[N][E], A[E], H[E], before_a[E], before_h[E];
#pragma unroll
    for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        float away;
        a[i][e] = logistic<kFine<T>>(rf[i][e], away);
        u[i][e] = away * rv[i][e];
        A[e] *= a[i][e], H[e] = fmaf(a[i][e], H[e], u[i][e]);
      }
    }
    wave_scan<E, RowLanes, true>(row, A, H, before_a, before_h);
    Exchange<E, RowLanes> &x = both[turn];
    if (row == 64 / RowLanes - 1)
#pragma unroll
      for (int e = 0; e < E; e++) x.a[wave][lane][e] = A[e], x.h[wave][lane][e] = H[e];
    __syncthreads();
    if (s0 + kTile < end) load(s0 + kTile);
    float h[E];
#pragma unroll 1
    for (int w = 0; w < kWaves; w++) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (w == wave) h[e] = carry[e];
        carry[e] = fmaf(x.a[w][lane][e], carry[e], x.h[w][lane][e]);
      }
    }
#pragma unroll
    for (int e = 0; e < E; e++) h[e] = fmaf(before_a[e], h[e], before_h[e]);
    if (p.states && at.here && s < p.L && s % kSpan == 0)
#pragma unroll
      for (int e = 0; e < E; e++) p.states[((int64_t)at.b * p.spans + s / kSpan) * p.C + at.c + e] = h[e];
    const auto out = Rows<T>::template of<kTile>(p, at, s0, p.out, (int64_t)p.L * p.C, p.C, run * N);
#pragma unroll
    for (int i = 0; i < N; i++) {
      float y[E];
#pragma unroll
      for (int e = 0; e < E; e++) {
        h[e] = fmaf(a[i][e], h[e], u[i][e]);
        y[e] = h[e];
        if (Gated) y[e] *= rz[i][e] * sigmoid<kFine<T>>(rz[i][e]);
      }
      if (at.here && (whole || s + i < at.len)) put<T, E, Passing>(out.at(i), y);
    }
    if (!whole) put_zeros<T, E>(p, at, p.out, s, N);
    if (s0 + kTile < end) load_gates(s0 + kTile);
  }
  if (at.here && at.segment == p.segments - 1 && threadIdx.x < RowLanes)
#pragma unroll
    for (int e = 0; e < E; e++) p.final[(int64_t)at.b * p.C + at.c + e] = carry[e];
}

template <typename T, int E, int N, int RowLanes, bool Gated, bool Passing>
__global__ __launch_bounds__(kThreads, 2) void recurrence_backward_kernel(RecurParams p) {
  constexpr int kTile = kRuns<RowLanes> * N;
  __shared__ Exchange<E, RowLanes> ahead[2], back[2];
  __shared__ Ranges<E, RowLanes> ranges;
  const int lane = threadIdx.x & (RowLanes - 1), run = threadIdx.x / RowLanes;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = (threadIdx.x & 63) / RowLanes;
  // (from the beginning, which the first launch read last)
  const Place at = place_of<E, RowLanes>(p, blockIdx.x, p.segments);
  const int begin = at.segment * p.segment, end = min(p.L, begin + p.segment);
  const int last = begin + (end - begin - 1) / kTile * kTile;
  Raw<T, E> rv[N], rf[N], rg[N], ro[N];
  float kept[E];
  // (as forward: what is used up first is fetched first)
  const auto load = [&](int s0) {
    const auto v = Rows<T>::template of<kTile>(p, at, s0, p.v, p.vs[0], p.vs[1], run * N);
    const auto f = Rows<T>::template of<kTile>(p, at, s0, p.f, p.fs[0], p.fs[1], run * N);
    const int s = s0 + run * N;
#pragma unroll
    for (int e = 0; e < E; e++)
      kept[e] = p.states[((int64_t)at.b * p.spans + s0 / kSpan) * p.C + at.c + e];
    if (s0 + kTile <= at.len) {
#pragma unroll
      for (int i = 0; i < N; i++) rv[i].load(v.at(i)), rf[i].load(f.at(i));
      return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      // a step that leaves the state and its gradient as they are
      rv[i].fill(0.f), rf[i].fill(__builtin_inff());
      if (s + i < at.len) rv[i].load(v.at(i)), rf[i].load(f.at(i));
    }
  };
  const auto load_gradients = [&](int s0) {
    const auto g = Rows<T>::template of<kTile>(p, at, s0, p.g, p.gs[0], p.gs[1], run * N);
    const auto o = Rows<T>::template of<kTile>(p, at, s0, p.go, (int64_t)p.L * p.C, p.C, run * N);
    const int s = s0 + run * N;
    if (s0 + kTile <= at.len) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        if (Gated) rg[i].load(g.at(i));
        ro[i].load(o.at(i));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      ro[i].fill(0.f);
      if (Gated) rg[i].fill(0.f);
      if (s + i < at.len) {
        if (Gated) rg[i].load(g.at(i));
        ro[i].load(o.at(i));
      }
    }
  };
  load(last);
  load_gradients(last);
  float carry[E];
#pragma unroll
  for (int e = 0; e < E; e++) carry[e] = p.gfinal ? p.gfinal[(int64_t)at.b * p.C + at.c + e] : 0.f;
  if (p.segments > 1) carry_in<E, RowLanes, true>(p, at, ranges, carry);
  int turn = 0;
  for (int s0 = last; s0 >= begin; s0 -= kTile, turn ^= 1) {
    const int s = s0 + run * N;
    const bool whole = s0 + kTile <= at.len;
    float a[N][E], away[N][E], h[N][E], d[N][E], A[E], H[E], before_a[E], before_h[E], state[E];
#pragma unroll
    for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < E; e++) {
        a[i][e] = logistic<kFine<T>>(rf[i][e], away[i][e]);
        A[e] *= a[i][e], H[e] = fmaf(a[i][e], H[e], away[i][e] * rv[i][e]);
      }
    wave_scan<E, RowLanes, true>(row, A, H, before_a, before_h);
    Exchange<E, RowLanes> &x = ahead[turn];
    if (row == 64 / RowLanes - 1)
#pragma unroll
      for (int e = 0; e < E; e++) x.a[wave][lane][e] = A[e], x.h[wave][lane][e] = H[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++) state[e] = kept[e];
#pragma unroll 1
    for (int w = 0; w < wave; w++)
#pragma unroll
      for (int e = 0; e < E; e++) state[e] = fmaf(x.a[w][lane][e], state[e], x.h[w][lane][e]);
#pragma unroll
    for (int e = 0; e < E; e++) state[e] = fmaf(before_a[e], state[e], before_h[e]);
    const auto gv = Rows<T>::template of<kTile>(p, at, s0, p.gv, (int64_t)p.L * p.C, p.C, run * N);
    const auto gf = Rows<T>::template of<kTile>(p, at, s0, p.gf, (int64_t)p.L * p.C, p.C, run * N);
    const auto gg = Rows<T>::template of<kTile>(p, at, s0, p.gg, (int64_t)p.L * p.C, p.C, run * N);
    // h: what the state before a step differs from its value by
#pragma unroll
    for (int i = 0; i < N; i++) {
      float y[E];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float x = rv[i][e];
        h[i][e] = state[e] - x;
        state[e] = fmaf(a[i][e], state[e], away[i][e] * x);
        d[i][e] = ro[i][e];
        if (Gated) {
          const float z = rg[i][e], sg = sigmoid<kFine<T>>(z);
          y[e] = d[i][e] * state[e] * (sg * fmaf(z, 1.f - sg, 1.f));
          d[i][e] *= z * sg;
        }
      }
      if (Gated && p.gg && at.here && (whole || s + i < at.len)) put<T, E, Passing>(gg.at(i), y);
    }
    // (all at once in bf16; in single precision, whose words take twice the registers, the gradients later: 43 ->
    // 39 us of 3 sequences of up to 31250 steps of 90 channels)
    if (s0 > begin) load(s0 - kTile);
    if (!kFine<T> && s0 > begin) load_gradients(s0 - kTile);
#pragma unroll
    for (int e = 0; e < E; e++) A[e] = 1.f, H[e] = 0.f;
#pragma unroll
    for (int i = N - 1; i >= 0; i--)
#pragma unroll
      for (int e = 0; e < E; e++) H[e] = a[i][e] * (d[i][e] + H[e]), A[e] *= a[i][e];
    wave_scan<E, RowLanes, false>(row, A, H, before_a, before_h);
    Exchange<E, RowLanes> &y = back[turn];
    if (row == 0)
#pragma unroll
      for (int e = 0; e < E; e++) y.a[wave][lane][e] = A[e], y.h[wave][lane][e] = H[e];
    __syncthreads();
    float push[E];
#pragma unroll 1
    for (int w = kWaves - 1; w >= 0; w--)
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (w == wave) push[e] = carry[e];
        carry[e] = fmaf(y.a[w][lane][e], carry[e], y.h[w][lane][e]);
      }
#pragma unroll
    for (int e = 0; e < E; e++) push[e] = fmaf(before_a[e], push[e], before_h[e]);
#pragma unroll
    for (int i = N - 1; i >= 0; i--) {
      float y1[E], y2[E];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float D = d[i][e] + push[e];
        push[e] = a[i][e] * D;
        y1[e] = away[i][e] * D;
        y2[e] = push[e] * (h[i][e] * away[i][e]);
      }
      if (at.here && (whole || s + i < at.len)) {
        if (p.gv) put<T, E, Passing>(gv.at(i), y1);
        if (p.gf) put<T, E, Passing>(gf.at(i), y2);
      }
    }
    if (!whole) {
      if (p.gv) put_zeros<T, E>(p, at, p.gv, s, N);
      if (p.gf) put_zeros<T, E>(p, at, p.gf, s, N);
      if (Gated && p.gg) put_zeros<T, E>(p, at, p.gg, s, N);
    }
    if (kFine<T> && s0 > begin) load_gradients(s0 - kTile);
  }
  if (p.ginitial && at.here && at.segment == 0 && threadIdx.x < RowLanes)
#pragma unroll
    for (int e = 0; e < E; e++) p.ginitial[(int64_t)at.b * p.C + at.c + e] = carry[e];
}

// Up to kFew steps, and kFewBackward backward: a thread walks them all.
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
        const float a = logistic<kFine<T>>(rf[e], away);
        h[e] = fmaf(a, h[e], away * rv[e]);
        y[e] = h[e];
        if (Gated) y[e] *= rg[e] * sigmoid<kFine<T>>(rg[e]);
      }
    }
    put<T, E>((T *)p.out + ((int64_t)at.b * p.L + t) * p.C + at.c, y);
  }
#pragma unroll
  for (int e = 0; e < E; e++) p.final[state + e] = h[e];
}

template <typename T, int E, bool Gated>
__global__ __launch_bounds__(256) void recurrence_few_backward_kernel(RecurParams p, int64_t words) {
  constexpr int K = kFewBackward;
  const int64_t index = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (index >= words) return;
  const int row = p.C / E;
  Place at;
  at.b = (int)(index / row), at.c = (int)(index % row) * E;
  at.len = p.lengths ? min(max(p.lengths[at.b], 0), p.L) : p.L;
  Raw<T, E> rv[K], rf[K], rg[K], ro[K];
  int64_t to[K];
#pragma unroll
  for (int s = 0; s < K; s++) {
    const int64_t t = token_of(p, at, s);
    to[s] = ((int64_t)at.b * p.L + t) * p.C + at.c;
    if (s < at.len) {
      rv[s].load((const T *)p.v + at.b * p.vs[0] + t * p.vs[1] + at.c);
      rf[s].load((const T *)p.f + at.b * p.fs[0] + t * p.fs[1] + at.c);
      ro[s].load((const T *)p.go + to[s]);
      if (Gated) rg[s].load((const T *)p.g + at.b * p.gs[0] + t * p.gs[1] + at.c);
    }
  }
  const int64_t state = (int64_t)at.b * p.C + at.c;
  float h[E], push[E], a[K][E], away[K][E], before[K][E], d[K][E];
#pragma unroll
  for (int e = 0; e < E; e++) h[e] = p.states[state + e], push[e] = p.gfinal ? p.gfinal[state + e] : 0.f;
#pragma unroll
  for (int s = 0; s < K; s++) {
    float y[E];
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = 0.f;
    if (s < at.len) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        a[s][e] = logistic<kFine<T>>(rf[s][e], away[s][e]);
        const float x = rv[s][e];
        before[s][e] = h[e] - x;
        h[e] = fmaf(a[s][e], h[e], away[s][e] * x);
        d[s][e] = ro[s][e];
        if (Gated) {
          const float z = rg[s][e], sg = sigmoid<kFine<T>>(z);
          y[e] = d[s][e] * h[e] * (sg * fmaf(z, 1.f - sg, 1.f));
          d[s][e] *= z * sg;
        }
      }
    }
    if (Gated && p.gg && s < p.L) put<T, E>((T *)p.gg + to[s], y);
  }
#pragma unroll
  for (int s = K - 1; s >= 0; s--) {
    float y1[E], y2[E];
#pragma unroll
    for (int e = 0; e < E; e++) y1[e] = y2[e] = 0.f;
    if (s < at.len) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float D = d[s][e] + push[e];
        push[e] = a[s][e] * D;
        y1[e] = away[s][e] * D;
        y2[e] = push[e] * (before[s][e] * away[s][e]);
      }
    }
    if (p.gv && s < p.L) put<T, E>((T *)p.gv + to[s], y1);
    if (p.gf && s < p.L) put<T, E>((T *)p.gf + to[s], y2);
  }
  if (p.ginitial)
#pragma unroll
    for (int e = 0; e < E; e++) p.ginitial[state + e] = push[e];
}

// ---- host ----

int check_desc(const mcx_recurrence_desc *d, int dtype) {
  if (!d) return MCX_E_NULL;
  if (dtype != MCX_F32 && dtype != MCX_BF16) return MCX_E_DTYPE;
  if (d->B < 0 || d->L < 0 || d->C < 1 || d->L > 0x3fffffff || d->C > (1 << 22) || d->B > (1 << 24) ||
      d->B * ((d->C + 15) / 16) >= (1 << 23))  // workgroups of 256 threads, their threads in 32 bits
    return MCX_E_SHAPE;
  // (a tile's addresses are 32 bits from its first: 512 steps of 2 bytes or 256 of 4 where channels are few, 128
  // and 64 of up to 2^22 channels)
  for (int64_t stride : {d->v_stride[1], d->f_stride[1], d->g_stride[1]})
    if (d->L > 1 && (stride < 0 || stride > (1 << 22))) return MCX_E_SHAPE;
  return MCX_OK;
}
// The bits that addresses of rows have, in bytes.
uint64_t address_bits(const mcx_recurrence_desc *d, int size, bool gated, uint64_t addresses) {
  uint64_t bits = addresses;
  for (int k = 0; k < 2; k++) {
    if ((k ? d->L : d->B) <= 1) continue;
    bits |= (uint64_t)d->v_stride[k] * size | (uint64_t)d->f_stride[k] * size;
    if (gated) bits |= (uint64_t)d->g_stride[k] * size;
  }
  return bits;
}
// Values of a word: 8 bytes or two values; rows of one or two words are cut smaller, so that the four lanes of a row have
// something to do (50 sequences of 30000 steps of 8 bf16 channels, forward and gradients, 180 -> 115 us; 15000 of 100
// steps 273 -> 310, but 30000 of 4 channels 525 -> 477; shorter ones have a few lanes at work either way).
int word_of(const mcx_recurrence_desc *d, int size, uint64_t bits) {
  for (int w : {8 / size, 2})
    if (d->C % w == 0 && bits % (w * size) == 0 && (d->C > 2 * w || d->L <= 64)) return w;
  return 1;
}
// Rows that are not whole cache lines share them between workgroups: neighbours then go to one XCD and its
// cache (3 sequences of up to 31250 steps of 90 float32 channels 122 -> 101 us); whole lines are faster read from
// all of them (2 of 32768 steps of 1024 bf16 channels 435 us, on one XCD 444).
int split_lines(const mcx_recurrence_desc *d, int size, uint64_t bits) {
  return bits % kLine != 0 || d->C * size % kLine != 0;
}
// Two tiles of kNarrowLanes channels' words at most, where that makes fewer tiles of channels and steps than
// kRowLanes (250 sequences of 6000 steps of 8 bf16 channels, forward and gradients, 413 -> 159 us; three tiles:
// 1091 of 1000 steps of 11 float32 channels 165 -> 199).
int lanes_of(const mcx_recurrence_desc *d, int word, int size) {
  const auto tiles = [&](int lanes) {
    const int64_t tile = kThreads / lanes * run_steps(word, size);
    return (d->C + lanes * word - 1) / (lanes * word) * ((d->L + tile - 1) / tile);
  };
  return d->C <= 2 * kNarrowLanes * word && tiles(kNarrowLanes) < tiles(kRowLanes) ? kNarrowLanes : kRowLanes;
}
// Segments make kGroups workgroups of the second launch, parts of them kSums of the first, which has less to
// do and so needs more under way; two tiles and one at least.
struct Cut {
  int segments, segment, parts, each, share;
};
Cut cut_of(const mcx_recurrence_desc *d, int word, int size, int groups) {
  const int lanes = lanes_of(d, word, size);
  const int64_t columns = std::max<int64_t>(1, d->B * ((d->C + lanes * word - 1) / (lanes * word)));
  int64_t n = columns >= kAlone ? 1 : (groups + columns - 1) / columns;
  const int64_t tile = kThreads / lanes * run_steps(word, size);
  n = std::max<int64_t>(1, std::min(n, d->L / (2 * tile)));
  // in tiles
  const int64_t segment = ((d->L + n - 1) / n + tile - 1) / tile;
  const int64_t each = std::max<int64_t>(1, segment * columns * n / kSums);
  Cut c;
  c.share = (int)((segment + each - 1) / each), c.each = (int)(each * tile), c.segment = c.share * c.each;
  c.segments = (int)((d->L + c.segment - 1) / c.segment);
  c.parts = (int)((d->L + c.each - 1) / c.each);
  return c;
}
size_t part_bytes(const mcx_recurrence_desc *d, int dtype) {
  int64_t n = 0;
  for (int w : {1, 2, 4}) {  // (whichever the alignment gives)
    for (int groups : {kGroups, kGroupsBf16Backward}) {
      const Cut c = cut_of(d, w, dtype == MCX_BF16 ? 2 : 4, groups);
      if (c.segments > 1) n = std::max<int64_t>(n, c.parts + 1);
    }
  }
  return (size_t)(d->B * n * 2 * d->C) * sizeof(float);
}
RecurParams params_of(const mcx_recurrence_desc *d, int word, int size, int groups, void *workspace) {
  RecurParams p = {};
  for (int k = 0; k < 2; k++) p.vs[k] = d->v_stride[k], p.fs[k] = d->f_stride[k], p.gs[k] = d->g_stride[k];
  p.L = (int)d->L, p.C = (int)d->C;
  p.lanes = lanes_of(d, word, size);
  p.tiles = (int)((d->C + p.lanes * word - 1) / (p.lanes * word));
  const Cut c = cut_of(d, word, size, groups);
  p.segment = c.segment, p.segments = c.segments, p.parts = c.parts, p.each = c.each, p.share = c.share;
  p.spans = (int)((d->L + kSpan - 1) / kSpan);
  p.reverse = d->reverse != 0;
  p.part = (float *)workspace;
  return p;
}

template <typename T, int E, int RowLanes, bool Gated, bool Backward>
int launch_parts(RecurParams p, int64_t B, hipStream_t s) {
  p.tiles = (p.C + RowLanes * E - 1) / (RowLanes * E);
  const int64_t parts = Backward ? p.parts - p.share : (p.segments - 1) * p.share;
  hipLaunchKernelGGL((recurrence_parts_kernel<T, E, RowLanes, Gated, Backward>), dim3((unsigned)(B * p.tiles * parts)),
                     dim3(kThreads), 0, s, p);
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}
template <typename T, int E, bool Gated, bool Backward>
int sum_parts(const RecurParams &p, int64_t B, hipStream_t s) {
  if (p.lanes == kNarrowLanes) return launch_parts<T, E, kNarrowLanes, Gated, Backward>(p, B, s);
  return p.C / E >= kWideRow ? launch_parts<T, E, 64, Gated, Backward>(p, B, s)
                             : launch_parts<T, E, kRowLanes, Gated, Backward>(p, B, s);
}

template <typename T, int E> bool passing(const RecurParams &p, int64_t B) {
  return p.C * (int)sizeof(T) % kLine == 0 && B * p.L * p.C * (int64_t)sizeof(T) >= kPassingBytes;
}

// Few steps take a tile of as few (8192 sequences of 16 steps of 256 bf16 channels forward and backward 451 -> 208 us,
// of 32 steps 651 -> 451).
template <typename T, int E, int N, int RowLanes, bool Gated, bool Backward>
int launch_tiles(const RecurParams &p, int64_t B, hipStream_t s) {
  constexpr bool kWord = E * sizeof(T) == 8;
  const bool past = passing<T, E>(p, B);
  const dim3 groups((unsigned)(B * p.tiles * p.segments));
  if constexpr (Backward)
    hipLaunchKernelGGL((past ? recurrence_backward_kernel<T, E, N, RowLanes, Gated, kWord>
                             : recurrence_backward_kernel<T, E, N, RowLanes, Gated, false>),
                       groups, dim3(kThreads), 0, s, p);
  else
    hipLaunchKernelGGL((past ? recurrence_forward_kernel<T, E, N, RowLanes, Gated, kWord>
                             : recurrence_forward_kernel<T, E, N, RowLanes, Gated, false>),
                       groups, dim3(kThreads), 0, s, p);
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}
template <typename T, int E, bool Gated, bool Backward>
int launch_steps(const RecurParams &p, int64_t B, hipStream_t s) {
  if (p.L <= (Backward ? kFewBackward : kFew)) {
    const int64_t words = B * (p.C / E);
    hipLaunchKernelGGL((Backward ? recurrence_few_backward_kernel<T, E, Gated> : recurrence_few_kernel<T, E, Gated>),
                       dim3((unsigned)((words + 255) / 256)), dim3(256), 0, s, p, words);
    MCX_HIP_CHECK_LAUNCH();
    return MCX_OK;
  }
  if (p.segments > 1)
    if (int e = sum_parts<T, E, Backward && Gated, Backward>(p, B, s)) return e;
  constexpr int kSteps = run_steps(E, sizeof(T));
  if (p.lanes == kNarrowLanes) return launch_tiles<T, E, kSteps, kNarrowLanes, Gated, Backward>(p, B, s);
  if constexpr (Backward)
    if (p.L <= kRuns<kRowLanes>) return launch_tiles<T, E, 1, kRowLanes, Gated, true>(p, B, s);
  if (p.L <= 2 * kRuns<kRowLanes>) return launch_tiles<T, E, 2, kRowLanes, Gated, Backward>(p, B, s);
  return launch_tiles<T, E, kSteps, kRowLanes, Gated, Backward>(p, B, s);
}
template <typename T, bool Forward>
int launch(const RecurParams &p, int64_t B, int word, hipStream_t s) {
#define MCX_RECUR(E) \
  (p.g ? launch_steps<T, E, true, !Forward>(p, B, s) : launch_steps<T, E, false, !Forward>(p, B, s))
  if constexpr (sizeof(T) == 2)
    if (word == 4) return MCX_RECUR(4);
  return word == 2 ? MCX_RECUR(2) : MCX_RECUR(1);
#undef MCX_RECUR
}

}  // namespace
}  // namespace mcx

extern "C" {

int64_t mcx_gated_recurrence_spans(int64_t L) { return L < 0 ? 0 : (L + mcx::kSpan - 1) / mcx::kSpan; }

size_t mcx_gated_recurrence_workspace(const mcx_recurrence_desc *desc, int dtype) {
  using namespace mcx;
  if (check_desc(desc, dtype) != MCX_OK || !desc->B || !desc->L) return 0;
  return part_bytes(desc, dtype);
}

int mcx_gated_recurrence_forward(const void *value, const void *forget, const void *gate,
                                 const float *initial, const int32_t *lengths, void *out, float *final,
                                 float *states, void *workspace, size_t workspace_bytes,
                                 const mcx_recurrence_desc *desc, int dtype, void *stream) {
  using namespace mcx;
  if (int e = check_desc(desc, dtype)) return e;
  if (!desc->B || !desc->L) return MCX_OK;
  if (!value || !forget || !out || !final) return MCX_E_NULL;
  const size_t need = part_bytes(desc, dtype);
  if (need && (!workspace || workspace_bytes < need)) return MCX_E_WORKSPACE;
  const int size = dtype == MCX_BF16 ? 2 : 4;
  const uint64_t bits = address_bits(
      desc, size, gate != nullptr,
      (uintptr_t)value | (uintptr_t)forget | (uintptr_t)gate | (uintptr_t)out);
  const int word = word_of(desc, size, bits);
  RecurParams p = params_of(desc, word, size, kGroups, workspace);
  p.together = split_lines(desc, size, bits);
  p.v = value, p.f = forget, p.g = gate, p.initial = initial, p.lengths = lengths;
  p.out = out, p.final = final, p.states = states;
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
  const size_t need = part_bytes(desc, dtype);
  if (need && (!workspace || workspace_bytes < need)) return MCX_E_WORKSPACE;
  const int size = dtype == MCX_BF16 ? 2 : 4;
  const uint64_t bits = address_bits(
      desc, size, gate != nullptr,
      (uintptr_t)value | (uintptr_t)forget | (uintptr_t)gate | (uintptr_t)gout | (uintptr_t)gvalue |
          (uintptr_t)gforget | (uintptr_t)ggate);
  const int word = word_of(desc, size, bits);
  RecurParams p = params_of(desc, word, size, size == 2 ? kGroupsBf16Backward : kGroups, workspace);
  p.together = split_lines(desc, size, bits);
  p.v = value, p.f = forget, p.g = gate, p.go = gout, p.gfinal = gfinal, p.lengths = lengths;
  p.gv = gvalue, p.gf = gforget, p.gg = ggate, p.ginitial = ginitial;
  p.states = const_cast<float *>(states);
  return dtype == MCX_BF16 ? launch<__bf16, false>(p, desc->B, word, (hipStream_t)stream)
                           : launch<float, false>(p, desc->B, word, (hipStream_t)stream);
}

}  // extern "C"
