// Norm of queries and keys per head with the position rotation in the same pass, and its gradient.
//
//   r = (mean(x^2) + eps)^(-1/2),  n = x r w,  y = n c + s' n_partner      (tail: y = n)
//   dn = dy c - s' dy_partner,  dw = sum dn x r,  u = dn w,  dx = r (u - x r^2 mean(u x))
// with s' = -s for the first of a pair and s for the second.
//
// Bound by memory: every value is read and written once.  A row (one head of one token) lies in a
// group of lanes, 16 bytes each, whose sums are shuffles; a group takes up to kHeads heads of its
// token, so that their loads are under way together and cos and sin are fetched once for them.
#include <algorithm>

#include "mcx_mfma_common.h"

namespace mcx {
namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;        // heads of an item
constexpr int kNormMaxD = 256;
constexpr int kGradBlocks = 1024;  // of the gradient's launch: as many partial sums of dw

struct NormParams {
  const void *q, *k, *wq, *wk, *gq, *gk;
  const float *cos, *sin;
  const int64_t *positions;
  void *oq, *ok;
  float *partial;  // [blocks][2][D]
  int64_t qs[3], ks[3];
  int64_t tokens;
  int L, Hq, Hk, D, F, adjacent, lanes;  // lanes of a row
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

// The sum over a row's group of lanes.
__device__ inline float row_sum(float x, int lanes) {
  for (int m = 1; m < lanes; m <<= 1) x += __shfl_xor(x, m);
  return x;
}

// Wide: a lane has 16 bytes in a row; else values lane, lane + 64, ... of a row that a wave has.
template <typename T, bool Wide> struct Lane {
  static constexpr int V = Wide ? 16 / (int)sizeof(T) : kNormMaxD / 64;
  typedef __attribute__((ext_vector_type(V))) T Vec;
  int in_row;  // the lane's place in its row
  __device__ inline int at(int e) const { return Wide ? in_row * V + e : in_row + 64 * e; }
  __device__ inline void load(const T *row, int D, float *x) const {
    if (Wide) {
      Vec v = {};
      if (in_row * V < D) v = *(const Vec *)(row + in_row * V);
#pragma unroll
      for (int e = 0; e < V; e++) x[e] = as_float(v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++) x[e] = at(e) < D ? as_float(row[at(e)]) : 0.f;
    }
  }
  __device__ inline void store(T *row, int D, const float *x) const {
    if (Wide) {
      Vec v;
#pragma unroll
      for (int e = 0; e < V; e++) v[e] = (T)x[e];
      if (in_row * V < D) *(Vec *)(row + in_row * V) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (at(e) < D) row[at(e)] = (T)x[e];
    }
  }
  // the other value of the pair (in the same lane, in a lane F values away, or read again); 0 for
  // what is not rotated
  __device__ inline void partner(const T *row, const float *x, const NormParams &p, float *y) const {
    if (Wide && p.adjacent) {
#pragma unroll
      for (int e = 0; e < V; e++) y[e] = at(e) < 2 * p.F ? x[e ^ 1] : 0.f;
    } else if (Wide) {
      const int away = p.F / V, to = in_row + (in_row < away ? away : -away);
      const int source = (threadIdx.x & 63) - in_row + (to < p.lanes ? to : in_row);
#pragma unroll
      for (int e = 0; e < V; e++) {
        y[e] = __shfl(x[e], source);
        if (at(e) >= 2 * p.F) y[e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; e++) {
        const int d = at(e), o = p.adjacent ? d ^ 1 : d < p.F ? d + p.F : d - p.F;
        y[e] = d < 2 * p.F ? as_float(row[o]) : 0.f;
      }
    }
  }
  // cos and signed sin of the lane's values; 1 and 0 behind the rotated ones
  __device__ inline void angles(const NormParams &p, int64_t place, float *c, float *s) const {
    const bool in = place >= 0 && place < p.places;
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int d = at(e);
      c[e] = 1.f, s[e] = 0.f;
      if (d < 2 * p.F) {
        const bool second = p.adjacent ? d & 1 : d >= p.F;
        const int f = p.adjacent ? d >> 1 : second ? d - p.F : d;
        c[e] = in ? p.cos[place * p.F + f] : __builtin_nanf("");
        s[e] = in ? p.sin[place * p.F + f] : __builtin_nanf("");
        if (!second) s[e] = -s[e];
      }
    }
  }
};

// Items: up to kHeads heads of one token, of the queries or of the keys.
template <typename T, bool Wide, bool Grad>
__device__ inline void norm_items(const NormParams &p, bool keys, int64_t first, int64_t step,
                                  const Lane<T, Wide> &lane, float *dw) {
  constexpr int V = Lane<T, Wide>::V;
  const T *x0 = (const T *)(keys ? p.k : p.q), *w0 = (const T *)(keys ? p.wk : p.wq);
  const T *g0 = (const T *)(keys ? p.gk : p.gq);
  T *o0 = (T *)(keys ? p.ok : p.oq);
  const int64_t *stride = keys ? p.ks : p.qs;
  const int H = keys ? p.Hk : p.Hq, D = p.D;
  const int parts = (H + kHeads - 1) / kHeads;
  const float mean = 1.f / (float)D;
  float w[V], wp[V];
#pragma unroll
  for (int e = 0; e < V; e++) w[e] = lane.at(e) < D ? as_float(w0[lane.at(e)]) : 0.f;
  {
    // (the weights of the partners, for the forward pass)
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int d = lane.at(e);
      const int o = p.adjacent ? d ^ 1 : d < p.F ? d + p.F : d - p.F;
      wp[e] = d < 2 * p.F ? as_float(w0[o]) : 0.f;
    }
  }
  for (int64_t item = first; item < p.tokens * parts; item += step) {
    int part, l;
    const int64_t token = divide(item, parts, &part), b = divide(token, p.L, &l);
    const int h0 = part * kHeads;
    float c[V], s[V];
    lane.angles(p, p.positions ? p.positions[token] : l, c, s);
    const T *row = x0 + b * stride[0] + l * stride[1] + h0 * stride[2];
    const int64_t dense = (token * H + h0) * D;
    float x[kHeads][V], g[kHeads][V];
#pragma unroll
    for (int n = 0; n < kHeads; n++)
      if (h0 + n < H) {
        lane.load(row + n * stride[2], D, x[n]);
        if (Grad) lane.load(g0 + dense + n * D, D, g[n]);
      }
#pragma unroll
    for (int n = 0; n < kHeads; n++) {
      if (h0 + n >= H) break;
      float squares = 0.f;
#pragma unroll
      for (int e = 0; e < V; e++) squares = fmaf(x[n][e], x[n][e], squares);
      const float r = rsqrtf(fmaf(row_sum(squares, p.lanes), mean, p.eps));
      float other[V], y[V];
      if (!Grad) {
        lane.partner(row + n * stride[2], x[n], p, other);
#pragma unroll
        for (int e = 0; e < V; e++)
          y[e] = fmaf(x[n][e] * r * w[e], c[e], s[e] * (other[e] * r * wp[e]));
      } else {
        lane.partner(g0 + dense + n * D, g[n], p, other);
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float dn = fmaf(g[n][e], c[e], -s[e] * other[e]);
          dw[e] = fmaf(dn, x[n][e] * r, dw[e]);
          y[e] = dn * w[e];
          dot = fmaf(y[e], x[n][e], dot);
        }
        // the part of u along x leaves all but eps r^2 of itself behind: what the subtraction's
        // rounding left of it is taken out by a second one
        const float r2 = r * r, along = row_sum(dot, p.lanes) * mean;
        dot = 0.f;
#pragma unroll
        for (int e = 0; e < V; e++) {
          y[e] = fmaf(-x[n][e], along * r2, y[e]);
          dot = fmaf(y[e], x[n][e], dot);
        }
        const float rest = fmaf(row_sum(dot, p.lanes), mean, -p.eps * r2 * along) * r2;
#pragma unroll
        for (int e = 0; e < V; e++) y[e] = r * fmaf(-x[n][e], rest, y[e]);
      }
      lane.store(o0 + dense + n * D, D, y);
    }
  }
}

template <typename T, bool Wide, bool Grad>
__global__ __launch_bounds__(kThreads) void qk_norm_rotate_kernel(NormParams p) {
  typedef Lane<T, Wide> Own;
  constexpr int V = Own::V;
  const int tid = threadIdx.x, per = kThreads / p.lanes;  // rows of a workgroup at a time
  Own lane{tid % p.lanes};
  const int64_t group = (int64_t)blockIdx.x * per + tid / p.lanes, groups = (int64_t)gridDim.x * per;
  const int64_t q_items = p.tokens * ((p.Hq + kHeads - 1) / kHeads);
  if (!Grad) {
    norm_items<T, Wide, Grad>(p, false, group, groups, lane, nullptr);
    // the keys' items go on where the queries' end, so that the last groups share them
    const int64_t left = q_items % groups;
    norm_items<T, Wide, Grad>(p, true, (group + groups - left) % groups, groups, lane, nullptr);
    return;
  }
  __shared__ float sums[kThreads * V];
  for (int part = 0; part < 2; part++) {
    float dw[V];
#pragma unroll
    for (int e = 0; e < V; e++) dw[e] = 0.f;
    norm_items<T, Wide, Grad>(p, part != 0, group, groups, lane, dw);
#pragma unroll
    for (int e = 0; e < V; e++) sums[tid * V + e] = dw[e];
    __syncthreads();
    for (int d = tid; d < p.D; d += kThreads) {
      const int in_row = Wide ? d / V : d % 64, e = Wide ? d % V : d / 64;
      float x = 0.f;
      for (int n = 0; n < per; n++) x += sums[(n * p.lanes + in_row) * V + e];
      p.partial[((int64_t)blockIdx.x * 2 + part) * p.D + d] = x;
    }
    __syncthreads();
  }
}

// gw[d] of the queries (part 0) and keys: the blocks' sums in a fixed order.
template <typename T>
__global__ __launch_bounds__(kThreads) void qk_norm_weight_grad_kernel(const float *partial, T *gwq,
                                                                       T *gwk, int blocks, int D) {
  __shared__ float sums[kThreads];
  const int column = blockIdx.x * 16 + (threadIdx.x & 15);
  float x = 0.f;
  if (column < 2 * D)
    for (int n = threadIdx.x >> 4; n < blocks; n += kThreads / 16) x += partial[(int64_t)n * 2 * D + column];
  sums[threadIdx.x] = x;
  __syncthreads();
  if (threadIdx.x < 16 && column < 2 * D) {
    for (int n = 1; n < kThreads / 16; n++) x += sums[n * 16 + threadIdx.x];
    if (column < D) gwq[column] = (T)x;
    else gwk[column - D] = (T)x;
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
  if (B > most || L > most || (L && B > (1LL << 40) / L) || Hq > 65536 || Hk > 65536)
    return MCX_E_SHAPE;
  if (!q_stride || !k_stride || !wq || !wk) return MCX_E_NULL;
  if (B && L && (!q || !k)) return MCX_E_NULL;
  if (F && (!cos || !sin)) return MCX_E_NULL;
  return MCX_OK;
}

bool aligned16(const void *p) { return (uintptr_t)p % 16 == 0; }

template <typename T, bool Grad>
int norm_launch(NormParams &p, int64_t *blocks, hipStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  bool wide = p.D % V == 0 && (p.adjacent || p.F % V == 0) && aligned16(p.q) && aligned16(p.k) &&
              aligned16(p.oq) && aligned16(p.ok) && aligned16(p.gq) && aligned16(p.gk);
  for (int n = 0; n < 3; n++) wide = wide && p.qs[n] % V == 0 && p.ks[n] % V == 0;
  p.lanes = wide ? norm_lanes(p.D, V) : 64;
  const int64_t per = kThreads / p.lanes;
  const int64_t full = (norm_items_of(p.tokens, p.Hq, p.Hk) + per - 1) / per;
  *blocks = std::max<int64_t>(1, std::min<int64_t>(full, *blocks));
  if (wide)
    hipLaunchKernelGGL((qk_norm_rotate_kernel<T, true, Grad>), dim3((unsigned)*blocks),
                       dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((qk_norm_rotate_kernel<T, false, Grad>), dim3((unsigned)*blocks),
                       dim3(kThreads), 0, stream, p);
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
  int64_t blocks = 1 << 20;
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
  if (!gwq || !gwk || (B && L && (!gq || !gk || !gq_in || !gk_in))) return MCX_E_NULL;
  const size_t need = mcx_qk_norm_rotate_backward_workspace(B, L, Hq, Hk, D, dtype);
  if (!workspace || workspace_bytes < need) return MCX_E_WORKSPACE;
  NormParams p = {};
  p.q = q, p.k = k, p.wq = wq, p.wk = wk, p.gq = gq, p.gk = gk;
  p.cos = cos, p.sin = sin, p.positions = positions;
  p.oq = gq_in, p.ok = gk_in, p.partial = (float *)workspace;
  for (int n = 0; n < 3; n++) p.qs[n] = q_stride[n], p.ks[n] = k_stride[n];
  p.tokens = B * L, p.L = (int)std::max<int64_t>(L, 1), p.Hq = (int)Hq, p.Hk = (int)Hk;
  p.D = (int)D, p.F = (int)F, p.places = places, p.eps = (float)eps, p.adjacent = adjacent != 0;
  int64_t blocks = grad_blocks(p.tokens, Hq, Hk);
  rc = dtype == MCX_BF16 ? norm_launch<__bf16, true>(p, &blocks, (hipStream_t)stream)
                         : norm_launch<float, true>(p, &blocks, (hipStream_t)stream);
  if (rc != MCX_OK) return rc;
  const dim3 grid((unsigned)((2 * D + 15) / 16));
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
