// Norm of queries and keys per head with the position rotation in the same pass, and its gradient.
//
//   r = (mean(x^2) + eps)^(-1/2),  n = x r w,  y = n c + s' n_partner      (tail: y = n)
//   dn = dy c - s' dy_partner,  dw = sum dn x r,  u = dn w,  dx = r (u - x r^2 mean(u x))
// with s' = -s for the first of a pair and s for the second.
//
// Bound by memory: every value is read and written once.  A row (one head of one token) lies in a
// group of lanes, 16 (or 8) bytes each, whose sums are lane exchanges; a group takes up to kHeads
// heads of its token, so that their loads are under way together and cos and sin are fetched once
// for them.  2048 x 512 tokens of 4 + 4 heads of 32 bf16 values: forward 239 us (4.5 TB/s), backward
// 344 us (4.7 TB/s), its weights' sums 5 us; 3 x 31250 tokens of 6 + 2 heads of 48 float32 values: 60
// and 97 us (4.8 and 4.5 TB/s).  A large copy reaches 4.9 TB/s.
#include <algorithm>

#include "mcx_mfma_common.h"

namespace mcx {
namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;        // heads of an item
constexpr int kNormMaxD = 256;
constexpr int kBlocks = 1280;      // of the forward launch, as many as are resident at a time
constexpr int kGradBlocks = 1024;  // of the gradient's: as many partial sums of dw

struct NormParams {
  const void *q, *k, *wq, *wk, *gq, *gk;
  const float *cos, *sin;
  const int64_t *positions;
  void *oq, *ok;
  float *partial;  // [blocks][2][D]
  int64_t qs[3], ks[3];
  int64_t tokens;
  int L, Hq, Hk, D, F, adjacent, lanes;  // lanes of a row
  int sums;        // the weights' gradients wanted: 1 the queries', 2 the keys'
  int64_t places;
  float eps;
};

__device__ inline float as_float(float v) { return v; }
__device__ inline float as_float(__bf16 v) { return (float)v; }

// a / b and a % b of numbers that seldom need 64 bits
__device__ inline int64_t divide(int64_t a, int b, int *rest) {
  if ((uint64_t)a >> 32) {
    *rest = (int)(a % b);
    return a / b;
  }
  const unsigned n = (unsigned)a, q = n / (unsigned)b;
  *rest = (int)(n - q * (unsigned)b);
  return q;
}

template <int Control> __device__ inline float exchanged(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), Control, 0xf, 0xf, true));
}
// The sum over a row's group of lanes (a power of two): within 16 lanes by lane exchange, neighbours
// first, then the mirrored halves of 8 and 16, whose lanes hold the same sums by then.
__device__ inline float row_sum(float x, int lanes) {
  if (lanes >= 2) x += exchanged<0xb1>(x);    // lanes 1 0 3 2
  if (lanes >= 4) x += exchanged<0x4e>(x);    // lanes 2 3 0 1
  if (lanes >= 8) x += exchanged<0x141>(x);   // the half row mirrored
  if (lanes >= 16) x += exchanged<0x140>(x);  // the row mirrored
  for (int m = 16; m < lanes; m <<= 1) x += __shfl_xor(x, m);
  return x;
}

// A lane has a word of 16 or 8 bytes in a row, the partners and the angles of its values lying in
// whole words too; or it has values lane, lane + 64, ... of a row that a wave has.
enum { kAnyRows, kWords8, kWords16 };
template <typename T, int Form> struct Lane {
  static constexpr bool Wide = Form != kAnyRows;
  static constexpr int V = Wide ? (Form == kWords16 ? 16 : 8) / (int)sizeof(T) : kNormMaxD / 64;
  typedef __attribute__((ext_vector_type(V))) T Vec;
  int in_row;  // the lane's place in its row
  __device__ inline int at(int e) const { return Wide ? in_row * V + e : in_row + 64 * e; }
  // the lane's values as they are
  __device__ inline Vec load(const T *row, int D) const {
    Vec v = {};
    if (Wide) {
      if (in_row * V < D) v = *(const Vec *)(row + in_row * V);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (at(e) < D) v[e] = row[at(e)];
    }
    return v;
  }
  __device__ inline void store(T *row, int D, const float *x) const {
    Vec v;
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = (T)x[e];
    if (Wide) {
      if (in_row * V < D) *(Vec *)(row + in_row * V) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (at(e) < D) row[at(e)] = v[e];
    }
  }
  // the other value of the pair (in the same lane, in a lane F values away, or read again); anything
  // finite's place is taken by 0 for what is not rotated
  __device__ inline Vec partner(const T *row, Vec x, const NormParams &p) const {
    Vec y = {};
    if (Wide && p.adjacent) {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (at(e) < 2 * p.F) y[e] = x[e ^ 1];
      return y;
    }
    if (Wide) {
      const int away = p.F / V, to = in_row + (in_row < away ? away : -away);
      const int source = (threadIdx.x & 63) - in_row + (to < p.lanes ? to : in_row);
      int w[sizeof(Vec) / 4];
      __builtin_memcpy(w, &x, sizeof(Vec));
#pragma unroll
      for (int n = 0; n < (int)sizeof(Vec) / 4; n++) w[n] = __builtin_amdgcn_ds_bpermute(source * 4, w[n]);
      if (in_row * V < 2 * p.F) __builtin_memcpy(&y, w, sizeof(Vec));
      return y;
    }
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int d = at(e), o = p.adjacent ? d ^ 1 : d < p.F ? d + p.F : d - p.F;
      if (d < 2 * p.F) y[e] = row[o];
    }
    return y;
  }
  // cos and signed sin of the lane's values; 1 and 0 behind the rotated ones
  __device__ inline void angles(const NormParams &p, int64_t place, float *c, float *s) const {
    const bool in = place >= 0 && place < p.places;
#pragma unroll
    for (int e = 0; e < V; e++) c[e] = 1.f, s[e] = 0.f;
    if (Wide) {
      const int d0 = in_row * V;
      if (d0 >= 2 * p.F) return;
      const bool second = !p.adjacent && d0 >= p.F;
      const int64_t f = (in ? place : 0) * p.F + (p.adjacent ? d0 / 2 : second ? d0 - p.F : d0);
      if (p.adjacent) {
        typedef __attribute__((ext_vector_type(V / 2))) float Half;
        const Half a = *(const Half *)(p.cos + f), b = *(const Half *)(p.sin + f);
#pragma unroll
        for (int e = 0; e < V; e++) c[e] = a[e / 2], s[e] = e & 1 ? b[e / 2] : -b[e / 2];
      } else {
        constexpr int N = V < 4 ? V : 4;
        typedef __attribute__((ext_vector_type(N))) float Some;
#pragma unroll
        for (int n = 0; n < V; n += N) {
          const Some a = *(const Some *)(p.cos + f + n), b = *(const Some *)(p.sin + f + n);
#pragma unroll
          for (int e = 0; e < N; e++) c[n + e] = a[e], s[n + e] = second ? b[e] : -b[e];
        }
      }
      if (!in)
#pragma unroll
        for (int e = 0; e < V; e++) c[e] = s[e] = __builtin_nanf("");
    } else {
#pragma unroll
      for (int e = 0; e < V; e++) {
        const int d = at(e);
        if (d < 2 * p.F) {
          const bool second = p.adjacent ? d & 1 : d >= p.F;
          const int f = p.adjacent ? d >> 1 : second ? d - p.F : d;
          c[e] = in ? p.cos[place * p.F + f] : __builtin_nanf("");
          s[e] = in ? p.sin[place * p.F + f] : __builtin_nanf("");
          if (!second) s[e] = -s[e];
        }
      }
    }
  }
};

// Items: up to kHeads heads of one token, of the queries or of the keys.
template <typename T, int Form, bool Grad>
__device__ inline void norm_items(const NormParams &p, bool keys, int64_t first, int64_t step,
                                  const Lane<T, Form> &lane, float *dw) {
  constexpr int V = Lane<T, Form>::V;
  typedef typename Lane<T, Form>::Vec Vec;
  const T *x0 = (const T *)(keys ? p.k : p.q), *w0 = (const T *)(keys ? p.wk : p.wq);
  const T *g0 = (const T *)(keys ? p.gk : p.gq);
  T *o0 = (T *)(keys ? p.ok : p.oq);
  const int64_t *stride = keys ? p.ks : p.qs;
  const int H = keys ? p.Hk : p.Hq, D = p.D;
  const int parts = (H + kHeads - 1) / kHeads;
  if (first >= p.tokens * parts) return;
  const float mean = 1.f / (float)D;
  float w[V], wp[V];  // the weights, and the partners'
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int d = lane.at(e), o = p.adjacent ? d ^ 1 : d < p.F ? d + p.F : d - p.F;
    w[e] = d < D ? as_float(w0[d]) : 0.f;
    wp[e] = !Grad && d < 2 * p.F ? as_float(w0[o]) : 0.f;
  }
  for (int64_t item = first; item < p.tokens * parts; item += step) {
    int part, l;
    const int64_t token = divide(item, parts, &part), b = divide(token, p.L, &l);
    const int h0 = part * kHeads;
    const T *row = x0 + b * stride[0] + l * stride[1] + h0 * stride[2];
    const int64_t dense = (token * H + h0) * D;
    Vec xv[kHeads], gv[kHeads];
#pragma unroll
    for (int n = 0; n < kHeads; n++)
      if (h0 + n < H) {
        xv[n] = lane.load(row + n * stride[2], D);
        if (Grad) gv[n] = lane.load(g0 + dense + n * D, D);
      }
    float c[V], s[V];
    lane.angles(p, p.positions ? p.positions[token] : l, c, s);
#pragma unroll
    for (int n = 0; n < kHeads; n++) {
      if (h0 + n >= H) break;
      float x[V], squares = 0.f;
#pragma unroll
      for (int e = 0; e < V; e++) {
        x[e] = as_float(xv[n][e]);
        squares = fmaf(x[e], x[e], squares);
      }
      const float r = rsqrtf(fmaf(row_sum(squares, p.lanes), mean, p.eps));
      float y[V];
      if (!Grad) {
        const Vec other = lane.partner(row + n * stride[2], xv[n], p);
#pragma unroll
        for (int e = 0; e < V; e++)
          y[e] = fmaf(x[e] * r * w[e], c[e], s[e] * (as_float(other[e]) * r * wp[e]));
      } else {
        const Vec other = lane.partner(g0 + dense + n * D, gv[n], p);
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float dn = fmaf(as_float(gv[n][e]), c[e], -s[e] * as_float(other[e]));
          dw[e] = fmaf(dn, x[e] * r, dw[e]);
          y[e] = dn * w[e];
          dot = fmaf(y[e], x[e], dot);
        }
        // the part of u along x leaves all but eps r^2 of itself behind: what the subtraction's
        // rounding left of it is taken out by a second one
        const float r2 = r * r, along = row_sum(dot, p.lanes) * mean;
        dot = 0.f;
#pragma unroll
        for (int e = 0; e < V; e++) {
          y[e] = fmaf(-x[e], along * r2, y[e]);
          dot = fmaf(y[e], x[e], dot);
        }
        const float rest = fmaf(row_sum(dot, p.lanes), mean, -p.eps * r2 * along) * r2;
#pragma unroll
        for (int e = 0; e < V; e++) y[e] = r * fmaf(-x[e], rest, y[e]);
      }
      if (!Grad || o0) lane.store(o0 + dense + n * D, D, y);
    }
  }
}

template <typename T, int Form, bool Grad>
__global__ __launch_bounds__(kThreads, 4) void qk_norm_rotate_kernel(NormParams p) {
  typedef Lane<T, Form> Own;
  constexpr int V = Own::V;
  const int tid = threadIdx.x, per = kThreads / p.lanes;  // rows of a workgroup at a time
  Own lane{tid % p.lanes};
  const int64_t group = (int64_t)blockIdx.x * per + tid / p.lanes, groups = (int64_t)gridDim.x * per;
  const int64_t q_items = p.tokens * ((p.Hq + kHeads - 1) / kHeads);
  if (!Grad) {
    norm_items<T, Form, Grad>(p, false, group, groups, lane, nullptr);
    // the keys' items go on where the queries' end, so that the last groups share them
    const int64_t left = q_items % groups;
    norm_items<T, Form, Grad>(p, true, (group + groups - left) % groups, groups, lane, nullptr);
    return;
  }
  __shared__ float sums[kThreads * V];
  for (int part = 0; part < 2; part++) {
    if (!(part ? p.ok : p.oq) && !(p.sums >> part & 1)) continue;  // nothing of it is wanted
    float dw[V];
#pragma unroll
    for (int e = 0; e < V; e++) dw[e] = 0.f;
    norm_items<T, Form, Grad>(p, part != 0, group, groups, lane, dw);
    if (!(p.sums >> part & 1)) continue;
#pragma unroll
    for (int e = 0; e < V; e++) sums[tid * V + e] = dw[e];
    __syncthreads();
    for (int d = tid; d < p.D; d += kThreads) {
      const int in_row = Own::Wide ? d / V : d % 64, e = Own::Wide ? d % V : d / 64;
      float x = 0.f;
      for (int n = 0; n < per; n++) x += sums[(n * p.lanes + in_row) * V + e];
      p.partial[((int64_t)blockIdx.x * 2 + part) * p.D + d] = x;
    }
    __syncthreads();
  }
}

// gw[d] of the queries (part 0) and keys, or of one of them: the blocks' sums in a fixed order, four
// columns a workgroup.
template <typename T>
__global__ __launch_bounds__(kThreads) void qk_norm_weight_grad_kernel(const float *partial, T *gwq,
                                                                       T *gwk, int blocks, int D) {
  __shared__ float sums[kThreads];
  const int column = blockIdx.x * 4 + (threadIdx.x & 3);
  float x = 0.f;
  if (column < 2 * D && (column < D ? gwq : gwk))
#pragma unroll 8
    for (int n = threadIdx.x >> 2; n < blocks; n += kThreads / 4) x += partial[(int64_t)n * 2 * D + column];
  sums[threadIdx.x] = x;
  __syncthreads();
  if (threadIdx.x < 4 && column < 2 * D) {
    for (int n = 1; n < kThreads / 4; n++) x += sums[n * 4 + threadIdx.x];
    T *to = column < D ? gwq : gwk;
    if (to) to[column < D ? column : column - D] = (T)x;
  }
}

int norm_lanes(int64_t D, int per16) {
  int lanes = 1;
  while (lanes * per16 < D) lanes *= 2;
  return lanes;
}

int64_t norm_items_of(int64_t tokens, int64_t Hq, int64_t Hk) {
  return tokens * ((Hq + kHeads - 1) / kHeads + (Hk + kHeads - 1) / kHeads);
}

int64_t grad_blocks(int64_t tokens, int64_t Hq, int64_t Hk) {
  return std::max<int64_t>(1, std::min<int64_t>(kGradBlocks, norm_items_of(tokens, Hq, Hk)));
}

int norm_check(const void *q, const void *k, const void *wq, const void *wk, const float *cos,
               const float *sin, const int64_t *q_stride, const int64_t *k_stride, int64_t B,
               int64_t L, int64_t Hq, int64_t Hk, int64_t D, int64_t F, int64_t places, double eps,
               int dtype) {
  if (dtype != MCX_F32 && dtype != MCX_BF16) return MCX_E_DTYPE;
  if (B < 0 || L < 0 || Hq < 1 || Hk < 1 || D < 1 || D > kNormMaxD || F < 0 || 2 * F > D ||
      places < 0 || !(eps >= 0))
    return MCX_E_SHAPE;
  const int64_t most = 0x7fffffffLL;
  if (B > most || L > most || (L && B > (1LL << 40) / L) || Hq > 65535 || Hk > 65535)
    return MCX_E_SHAPE;
  if (!q_stride || !k_stride || !wq || !wk) return MCX_E_NULL;
  if (B && L && (!q || !k)) return MCX_E_NULL;
  if (F && (!cos || !sin)) return MCX_E_NULL;
  return MCX_OK;
}

// Whether a row's values, the pairs' places and the angles come in words of so many bytes.
template <typename T> bool norm_words(const NormParams &p, int bytes) {
  const int V = bytes / (int)sizeof(T), angles = p.adjacent ? V / 2 : V;
  bool fits = p.D % V == 0 && p.F % angles == 0 && norm_lanes(p.D, V) <= 64;
  for (const void *at : {p.q, p.k, p.gq, p.gk, (const void *)p.oq, (const void *)p.ok})
    fits = fits && (uintptr_t)at % bytes == 0;
  for (const float *at : {p.cos, p.sin})
    fits = fits && (uintptr_t)at % std::min<int>(16, angles * (int)sizeof(float)) == 0;
  for (int n = 0; n < 3; n++) fits = fits && p.qs[n] % V == 0 && p.ks[n] % V == 0;
  return fits;
}

template <typename T, bool Grad>
int norm_launch(NormParams &p, int64_t *blocks, hipStream_t stream) {
  const int bytes = norm_words<T>(p, 16) ? 16 : norm_words<T>(p, 8) ? 8 : 0;
  p.lanes = bytes ? norm_lanes(p.D, bytes / (int)sizeof(T)) : 64;
  const int64_t per = kThreads / p.lanes;
  const int64_t full = (norm_items_of(p.tokens, p.Hq, p.Hk) + per - 1) / per;
  *blocks = std::max<int64_t>(1, std::min<int64_t>(full, *blocks));
#define MCX_NORM(FORM)                                                                          \
  hipLaunchKernelGGL((qk_norm_rotate_kernel<T, FORM, Grad>), dim3((unsigned)*blocks),           \
                     dim3(kThreads), 0, stream, p)
  if (bytes == 16) MCX_NORM(kWords16);
  else if (bytes == 8) MCX_NORM(kWords8);
  else MCX_NORM(kAnyRows);
#undef MCX_NORM
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}

}  // namespace
}  // namespace mcx

extern "C" {

int mcx_qk_norm_rotate_forward(const void *q, const void *k, const void *wq, const void *wk,
                               const float *cos, const float *sin, const int64_t *positions,
                               void *q_out, void *k_out, const int64_t *q_stride,
                               const int64_t *k_stride, int64_t B, int64_t L, int64_t Hq,
                               int64_t Hk, int64_t D, int64_t F, int64_t places, double eps,
                               int adjacent, int dtype, void *stream) {
  using namespace mcx;
  const int rc = norm_check(q, k, wq, wk, cos, sin, q_stride, k_stride, B, L, Hq, Hk, D, F, places,
                            eps, dtype);
  if (rc != MCX_OK) return rc;
  if (B == 0 || L == 0) return MCX_OK;
  if (!q_out || !k_out) return MCX_E_NULL;
  NormParams p = {};
  p.q = q, p.k = k, p.wq = wq, p.wk = wk, p.cos = cos, p.sin = sin, p.positions = positions;
  p.oq = q_out, p.ok = k_out;
  for (int n = 0; n < 3; n++) p.qs[n] = q_stride[n], p.ks[n] = k_stride[n];
  p.tokens = B * L, p.L = (int)L, p.Hq = (int)Hq, p.Hk = (int)Hk, p.D = (int)D, p.F = (int)F;
  p.places = places, p.eps = (float)eps, p.adjacent = adjacent != 0;
  int64_t blocks = kBlocks;
  return dtype == MCX_BF16 ? norm_launch<__bf16, false>(p, &blocks, (hipStream_t)stream)
                           : norm_launch<float, false>(p, &blocks, (hipStream_t)stream);
}

size_t mcx_qk_norm_rotate_backward_workspace(int64_t B, int64_t L, int64_t Hq, int64_t Hk,
                                             int64_t D, int dtype) {
  if (B < 0 || L < 0 || Hq < 1 || Hk < 1 || D < 1 || D > mcx::kNormMaxD) return 0;
  return (size_t)mcx::grad_blocks(B * L, Hq, Hk) * 2 * D * sizeof(float);
}

int mcx_qk_norm_rotate_backward(const void *gq, const void *gk, const void *q, const void *k,
                                const void *wq, const void *wk, const float *cos, const float *sin,
                                const int64_t *positions, void *gq_in, void *gk_in, void *gwq,
                                void *gwk, void *workspace, size_t workspace_bytes,
                                const int64_t *q_stride, const int64_t *k_stride, int64_t B,
                                int64_t L, int64_t Hq, int64_t Hk, int64_t D, int64_t F,
                                int64_t places, double eps, int adjacent, int dtype, void *stream) {
  using namespace mcx;
  int rc = norm_check(q, k, wq, wk, cos, sin, q_stride, k_stride, B, L, Hq, Hk, D, F, places, eps,
                      dtype);
  if (rc != MCX_OK) return rc;
  if (B && L && (!gq || !gk)) return MCX_E_NULL;
  if (!gwq && !gwk && (!B || !L || (!gq_in && !gk_in))) return MCX_OK;
  const size_t need = mcx_qk_norm_rotate_backward_workspace(B, L, Hq, Hk, D, dtype);
  if (!workspace || workspace_bytes < need) return MCX_E_WORKSPACE;
  NormParams p = {};
  p.q = q, p.k = k, p.wq = wq, p.wk = wk, p.gq = gq, p.gk = gk;
  p.cos = cos, p.sin = sin, p.positions = positions;
  p.oq = gq_in, p.ok = gk_in, p.partial = (float *)workspace;
  p.sums = (gwq ? 1 : 0) | (gwk ? 2 : 0);
  for (int n = 0; n < 3; n++) p.qs[n] = q_stride[n], p.ks[n] = k_stride[n];
  p.tokens = B * L, p.L = (int)std::max<int64_t>(L, 1), p.Hq = (int)Hq, p.Hk = (int)Hk;
  p.D = (int)D, p.F = (int)F, p.places = places, p.eps = (float)eps, p.adjacent = adjacent != 0;
  int64_t blocks = grad_blocks(p.tokens, Hq, Hk);
  rc = dtype == MCX_BF16 ? norm_launch<__bf16, true>(p, &blocks, (hipStream_t)stream)
                         : norm_launch<float, true>(p, &blocks, (hipStream_t)stream);
  if (rc != MCX_OK || !p.sums) return rc;
  const dim3 grid((unsigned)((2 * D + 3) / 4));
  if (dtype == MCX_BF16)
    hipLaunchKernelGGL((qk_norm_weight_grad_kernel<__bf16>), grid, dim3(kThreads), 0,
                       (hipStream_t)stream, p.partial, (__bf16 *)gwq, (__bf16 *)gwk, (int)blocks,
                       (int)D);
  else
    hipLaunchKernelGGL((qk_norm_weight_grad_kernel<float>), grid, dim3(kThreads), 0,
                       (hipStream_t)stream, p.partial, (float *)gwq, (float *)gwk, (int)blocks,
                       (int)D);
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}

}  // extern "C"
