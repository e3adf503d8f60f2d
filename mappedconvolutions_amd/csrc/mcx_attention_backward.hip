// Gradients of attention with a bias by relative-position buckets.
//
//   p_ij = exp(scale u_ij - lse_i),  dp_ij = do_i . v_j,  delta_i = do_i . o_i
//   ds_ij = p_ij (dp_ij - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//   dT[h, n] = sum of ds over the pairs of bucket n
//
// Scores are computed again in both kernels (seven products of a tile instead of five): every
// gradient then has one owner, who sums it in registers in a fixed order.  No atomics on memory,
// the same bits each time.
#include <algorithm>

#include "mcx_attention.h"

namespace mcx {
namespace attention {

// c + a b^T of a column a (rows) and a row b (columns), the upper half-wave's a being 0: takes
// delta from dp in the matrix pipe, which has the time, and after dp's last addition: equal sums
// of equal terms then leave nothing.
__device__ inline floatx16 add_outer(float a, float b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// A probability from u: through lse = scale log2(e) ref + log2(sum), +inf for a row that nothing
// is left of; or, where that is too large to hold its second term, from ref and 1 / sum.
template <bool Huge>
__device__ inline float probability(float u, float c, float lse, float ref, float inv) {
  if (Huge) return ref == -kInf ? 0.f : exp2_fast((u - ref) * c) * inv;
  return exp2_fast(fmaf(u, c, -lse));
}

// Queries' gradients, the sums per bucket, and the rows' statistics for the other kernel.  The
// same walk as the forward product's: a wave holds 32 queries, their o gradient beside them.
//   The bias' gradient: ds of a wave's 32 x 64 pairs goes by its difference j - i into a ring of
// 128 sums that only this wave writes; the 64 differences that the next tile no longer meets are
// then added to the wave's sums per bucket.
template <typename T, int DP>
__global__ __launch_bounds__(64 * kWaves) void attention_query_grad_kernel(
    Params p, const T *out, const T *gout, const float *stats, float *lses, float *deltas, T *gq,
    float *partial, int nq) {
  constexpr int P = pitch<T, DP>(), Chunks = DP / 16, Blocks = DP / 32;
  __shared__ __attribute__((aligned(16))) T ks[2][kTile * P];
  __shared__ __attribute__((aligned(16))) T vs[2][kTile * P];
  __shared__ __attribute__((aligned(16))) Window window[2];
  __shared__ int window_bucket[2][kWindow];
  __shared__ float ring[kWaves][128];
  extern __shared__ float table[];  // NB values, then kWaves x NB sums

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const int wg = xcd_contiguous_tile(blockIdx.x, gridDim.x);
  const int bh = wg / nq, b = bh / p.Hq, h = bh % p.Hq;
  const int block = nq - 1 - wg % nq, i0 = block * kBlock;
  const int kh = h / (p.Hq / p.Hk);
  const int start = first_position(p, b), length = key_length(p, b);
  const int local = wave * kLanesRows + (lane & 31), i = i0 + local;
  const bool live = i < p.Lq;
  const int limit = p.causal ? min(length, start + i + 1) : length;
  const int last = min(i0 + kBlock, p.Lq) - 1;
  const int keys = p.causal ? max(0, min(length, start + last + 1)) : length;
  const int wave_limit = p.causal ? min(length, start + i0 + wave * kLanesRows + 1) : length;

  const T *q = (const T *)p.q + b * p.qs[0] + (int64_t)i * p.qs[1] + h * p.qs[2];
  const T *k = (const T *)p.k + b * p.ks[0] + kh * p.ks[2];
  const T *v = (const T *)p.v + b * p.vs[0] + kh * p.vs[2];
  const int64_t row = ((int64_t)b * p.Lq + i) * p.Hq + h;
  const bool out_wide = p.D % (16 / (int)sizeof(T)) == 0;
  const bool biased = p.table != nullptr, table_grad = partial != nullptr;
  float *sums = table + p.NB + wave * p.NB;

  Frag<T> qf[Chunks], gf[Chunks];
  // delta is the diagonal of a product of the same kind as dp's: where a row's output is one of
  // its values, the two are the same number and their difference is nothing
  floatx16 products = (floatx16)(0.f);
#pragma unroll
  for (int c = 0; c < Chunks; c++) {
    qf[c] = global_frag<T>(live ? q : nullptr, c, half, p.D, p.q_wide);
    gf[c] = global_frag<T>(live ? gout + row * p.D : nullptr, c, half, p.D, out_wide);
    products = mma(global_frag<T>(live ? out + row * p.D : nullptr, c, half, p.D, out_wide), gf[c],
                   products);
  }
  float delta = 0.f;
#pragma unroll
  for (int n = 0; n < 16; n++)  // row 8 (n >> 2) + 4 half + (n & 3)
    if ((lane & 31) == 8 * (n >> 2) + 4 * half + (n & 3)) delta = products[n];
  delta += other_half(delta);
  const float c = p.scale * kLog2e;
  float ref = -kInf, sum = 0.f;
  const int64_t stat = ((int64_t)b * p.Hq + h) * p.Lq + i;
  if (live) {
    ref = stats[2 * stat];
    sum = stats[2 * stat + 1];
  }
  const float lse = ref == -kInf ? kInf : fmaf(ref, c, __log2f(sum));
  const float inv = 1.f / sum;
  if (live && half == 0) {
    lses[stat] = lse;
    deltas[stat] = -delta;
  }
  if (!gq && !table_grad) return;

  const int base = -(start + i0 + kBlock - 1);
  if (biased) load_table<T>(p, h, table, tid, 64 * kWaves);
  if (table_grad) {
    for (int n = lane; n < p.NB; n += 64) sums[n] = 0.f;
    ring[wave][lane] = ring[wave][64 + lane] = 0.f;
  }
  Tile<T, DP> kt, vt;
  int bucket = 0;
  const int tiles = (keys + kTile - 1) / kTile;
  if (tiles > 0) {
    kt.load(k, p.ks[1], keys, p.D, p.k_wide, tid);
    vt.load(v, p.vs[1], keys, p.D, p.v_wide, tid);
    if (biased) bucket = bucket_of(p, base + tid);
  }
  __syncthreads();
  if (tiles > 0) {
    kt.store(ks[0], tid);
    vt.store(vs[0], tid);
    if (biased && tid < kWindow) {
      window[0].put(tid, bias_of(table, p.NB, bucket));
      window_bucket[0][tid] = bucket;
    }
  }
  __syncthreads();

  const int at = kBlock - 1 - local, shift = at & 3;
  const bool huge = __any(lse < kInf && fabsf(lse) > kHugeStat);
  floatx16 acc[Blocks];
#pragma unroll
  for (int d = 0; d < Blocks; d++) acc[d] = (floatx16)(0.f);

  for (int t = 0; t < tiles; t++) {
    const int j0 = t * kTile, buf = t & 1;
    if (t + 1 < tiles) {
      const int64_t next = j0 + kTile;
      kt.load(k + next * p.ks[1], p.ks[1], keys - (int)next, p.D, p.k_wide, tid);
      vt.load(v + next * p.vs[1], p.vs[1], keys - (int)next, p.D, p.v_wide, tid);
      if (biased) bucket = bucket_of(p, base + (int)next + tid);
    }
#pragma unroll
    for (int blk = 0; blk < 2; blk++) {
      floatx16 u, dp;
      if (biased) {
        const floatx8 lo = window[buf].get(at + 32 * blk + 8 * half, shift);
        const floatx8 hi = window[buf].get(at + 32 * blk + 16 + 8 * half, shift);
        u = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15);
      } else {
        u = (floatx16)(0.f);
      }
      dp = (floatx16)(0.f);
#pragma unroll
      for (int ch = 0; ch < Chunks; ch++) {
        u = mma(row_frag<T, DP>(ks[buf], 32 * blk + row_of(lane & 31), ch, half), qf[ch], u);
        dp = mma(row_frag<T, DP>(vs[buf], 32 * blk + row_of(lane & 31), ch, half), gf[ch], dp);
      }
      dp = add_outer(half ? 0.f : 1.f, -delta, dp);
      if (j0 + kTile > wave_limit) {
#pragma unroll
        for (int n = 0; n < 16; n++)
          if (j0 + 32 * blk + 16 * (n >> 3) + 8 * half + (n & 7) >= limit) u[n] = -kInf;
      }
      if (huge) {
#pragma unroll
        for (int n = 0; n < 16; n++) dp[n] *= probability<true>(u[n], c, lse, ref, inv);
      } else {
#pragma unroll
        for (int n = 0; n < 16; n++) dp[n] *= probability<false>(u[n], c, lse, ref, inv);
      }
      if (table_grad) {
        // place of difference j - i in the ring: (j - j0) - (i - wave's first) + 64 t + 64, mod 128
        const int place = 32 * blk + 8 * half - (lane & 31) + 64 * (t + 1);
#pragma unroll
        for (int n = 0; n < 16; n++)
          atomicAdd(&ring[wave][(place + 16 * (n >> 3) + (n & 7)) & 127], dp[n]);
      }
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const floatx8 x = s == 0
            ? __builtin_shufflevector(dp, dp, 0, 1, 2, 3, 4, 5, 6, 7)
            : __builtin_shufflevector(dp, dp, 8, 9, 10, 11, 12, 13, 14, 15);
        const Frag<T> f = Frag<T>::pack(x);
#pragma unroll
        for (int d = 0; d < Blocks; d++)
          acc[d] = mma(col_frag<DP>(ks[buf], 32 * blk + 16 * s, d, lane), f, acc[d]);
      }
    }
    if (table_grad) {
      // differences -31 .. 32 of the tile (from the wave's first query) are met no more
      const int x = lane - 31, place = (x + 64 * (t + 1)) & 127;
      const float value = ring[wave][place];
      ring[wave][place] = 0.f;
      const int n = window_bucket[buf][x + kBlock - 1 - wave * kLanesRows];
      if ((unsigned)n < (unsigned)p.NB) atomicAdd(&sums[n], value);
    }
    if (t + 1 < tiles) {
      kt.store(ks[buf ^ 1], tid);
      vt.store(vs[buf ^ 1], tid);
      if (biased && tid < kWindow) {
        window[buf ^ 1].put(tid, bias_of(table, p.NB, bucket));
        window_bucket[buf ^ 1][tid] = bucket;
      }
    }
    __syncthreads();
  }
  if (table_grad) {
    if (tiles > 0 && lane < 31) {  // differences 33 .. 63 of the last tile
      const int x = lane + 33, place = (x + 64 * tiles) & 127;
      const int n = window_bucket[(tiles - 1) & 1][x + kBlock - 1 - wave * kLanesRows];
      if ((unsigned)n < (unsigned)p.NB) atomicAdd(&sums[n], ring[wave][place]);
    }
    __syncthreads();
    float *to = partial + ((int64_t)bh * nq + block) * p.NB;
    for (int n = tid; n < p.NB; n += 64 * kWaves) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; w++) x += table[p.NB + w * p.NB + n];
      to[n] = x;
    }
  }
  if (live && gq) store_column<T, Blocks>(gq + row * p.D, acc, p.scale, p.D, half, p.D % 4 == 0);
}

// Keys' and values' gradients: a workgroup holds 128 keys of a key head, a wave 32 of them as
// columns, and walks the queries of all heads that share them, 64 at a time.
template <typename T, int DP>
__global__ __launch_bounds__(64 * kWaves) void attention_key_grad_kernel(
    Params p, const T *gout, const float *stats, const float *lses, const float *deltas, T *gk,
    T *gv, int nk) {
  constexpr int P = pitch<T, DP>(), Chunks = DP / 16, Blocks = DP / 32;
  __shared__ __attribute__((aligned(16))) T qs[2][kTile * P];
  __shared__ __attribute__((aligned(16))) T gs[2][kTile * P];
  __shared__ __attribute__((aligned(16))) Window window[2];
  __shared__ __attribute__((aligned(16))) float row_lse[2][kTile], row_delta[2][kTile],
      row_ref[2][kTile], row_inv[2][kTile];
  extern __shared__ float table[];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const int wg = xcd_contiguous_tile(blockIdx.x, gridDim.x);
  const int bh = wg / nk, b = bh / p.Hk, kh = bh % p.Hk;
  const int j0 = (wg % nk) * kBlock;  // the longest columns of a causal map first
  const int group = p.Hq / p.Hk;
  const int start = first_position(p, b), length = key_length(p, b);
  const int local = wave * kLanesRows + (lane & 31), j = j0 + local;
  const bool live = j < p.Lk, used = j < length;
  // the first query that sees a key of this workgroup, and of this lane
  const int first = p.causal ? max(0, j0 - start) : 0;
  const int own_first = p.causal ? j - start : 0;
  const int t0 = first / kTile, t1 = j0 < length ? (p.Lq + kTile - 1) / kTile : 0;
  const int wave_safe = p.causal ? j0 + wave * kLanesRows + kLanesRows - 1 - start : 0;

  const T *k = (const T *)p.k + b * p.ks[0] + (int64_t)j * p.ks[1] + kh * p.ks[2];
  const T *v = (const T *)p.v + b * p.vs[0] + (int64_t)j * p.vs[1] + kh * p.vs[2];
  const bool out_wide = p.D % (16 / (int)sizeof(T)) == 0;
  const bool biased = p.table != nullptr;
  Frag<T> kf[Chunks], vf[Chunks];
#pragma unroll
  for (int c = 0; c < Chunks; c++) {
    kf[c] = global_frag<T>(used ? k : nullptr, c, half, p.D, p.k_wide);
    vf[c] = global_frag<T>(used ? v : nullptr, c, half, p.D, p.v_wide);
  }
  const float c = p.scale * kLog2e;
  const int at = kBlock - 1 - local, shift = at & 3;
  floatx16 dk[Blocks], dv[Blocks];
#pragma unroll
  for (int d = 0; d < Blocks; d++) dk[d] = dv[d] = (floatx16)(0.f);

  Tile<T, DP> qt, gt;
  int bucket = 0;
  float lse = 0.f, delta = 0.f, ref = 0.f, sum = 1.f;
  for (int g = 0; g < group && t0 < t1; g++) {
    const int h = kh * group + g;
    const T *q = (const T *)p.q + b * p.qs[0] + h * p.qs[2];
    const T *go = gout + ((int64_t)b * p.Lq * p.Hq + h) * p.D;
    const int64_t go_row = (int64_t)p.Hq * p.D;
    const int64_t stat = ((int64_t)b * p.Hq + h) * p.Lq;
    // window value x: query - key = (first query of the tile) - (j0 + kBlock - 1) + x, so the
    // bucket's difference is j0 + kBlock - 1 - start - first query - x
    const int base = j0 + kBlock - 1 - start;
    auto fetch = [&](int t) {
      const int64_t i = (int64_t)t * kTile;
      qt.load(q + i * p.qs[1], p.qs[1], p.Lq - (int)i, p.D, p.q_wide, tid);
      gt.load(go + i * go_row, go_row, p.Lq - (int)i, p.D, out_wide, tid);
      if (biased) bucket = bucket_of(p, base - (int)i - tid);
      if (tid < kTile) {
        const bool in = i + tid < p.Lq;
        lse = in ? lses[stat + i + tid] : kInf;
        delta = in ? deltas[stat + i + tid] : 0.f;
        ref = in ? stats[2 * (stat + i + tid)] : -kInf;
        sum = in ? stats[2 * (stat + i + tid) + 1] : 1.f;
      }
    };
    auto put = [&](int buf) {
      qt.store(qs[buf], tid);
      gt.store(gs[buf], tid);
      if (biased && tid < kWindow) window[buf].put(tid, bias_of(table, p.NB, bucket));
      if (tid < kTile) {
        row_lse[buf][tid] = lse;
        row_delta[buf][tid] = delta;
        row_ref[buf][tid] = ref;
        row_inv[buf][tid] = 1.f / sum;
      }
    };
    if (biased) load_table<T>(p, h, table, tid, 64 * kWaves);
    fetch(t0);
    __syncthreads();
    put(0);
    __syncthreads();
    for (int t = t0; t < t1; t++) {
      const int buf = (t - t0) & 1, i0 = t * kTile;
      if (t + 1 < t1) fetch(t + 1);
      const float mine = row_lse[buf][lane];
      const bool huge = __any(mine < kInf && fabsf(mine) > kHugeStat);
#pragma unroll
      for (int blk = 0; blk < 2; blk++) {
        floatx16 u, dp;
        if (biased) {
          const floatx8 lo = window[buf].get(at + 32 * blk + 8 * half, shift);
          const floatx8 hi = window[buf].get(at + 32 * blk + 16 + 8 * half, shift);
          u = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15);
        } else {
          u = (floatx16)(0.f);
        }
        auto rows8 = [&](const float *x, int s) {
          const floatx4 *w = (const floatx4 *)(x + 32 * blk + 16 * s + 8 * half);
          const floatx4 lo = w[0], hi = w[1];
          return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        dp = (floatx16)(0.f);
#pragma unroll
        for (int ch = 0; ch < Chunks; ch++) {
          u = mma(row_frag<T, DP>(qs[buf], 32 * blk + row_of(lane & 31), ch, half), kf[ch], u);
          dp = mma(row_frag<T, DP>(gs[buf], 32 * blk + row_of(lane & 31), ch, half), vf[ch], dp);
        }
        dp = add_outer(half ? 0.f : row_delta[buf][32 * blk + row_of(lane & 31)], 1.f, dp);
        if (i0 < wave_safe || i0 + kTile > p.Lq) {
#pragma unroll
          for (int n = 0; n < 16; n++) {
            const int i = i0 + 32 * blk + 16 * (n >> 3) + 8 * half + (n & 7);
            if (i < own_first || i >= p.Lq) u[n] = -kInf;
          }
        }
#pragma unroll
        for (int s = 0; s < 2; s++) {
          floatx8 x, y;
          const floatx8 l8 = rows8(row_lse[buf], s);
          if (huge) {
            const floatx8 r8 = rows8(row_ref[buf], s), i8 = rows8(row_inv[buf], s);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = probability<true>(u[8 * s + e], c, l8[e], r8[e], i8[e]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = probability<false>(u[8 * s + e], c, l8[e], 0.f, 0.f);
          }
#pragma unroll
          for (int e = 0; e < 8; e++) y[e] = x[e] * dp[8 * s + e];
          const Frag<T> pf = Frag<T>::pack(x), sf = Frag<T>::pack(y);
#pragma unroll
          for (int d = 0; d < Blocks; d++) {
            dv[d] = mma(col_frag<DP>(gs[buf], 32 * blk + 16 * s, d, lane), pf, dv[d]);
            dk[d] = mma(col_frag<DP>(qs[buf], 32 * blk + 16 * s, d, lane), sf, dk[d]);
          }
        }
      }
      if (t + 1 < t1) put(buf ^ 1);
      __syncthreads();
    }
  }
  if (!live) return;
  const int64_t row = ((int64_t)b * p.Lk + j) * p.Hk + kh;
  // a key that is not in use has no part in anything
  if (!used) {
#pragma unroll
    for (int d = 0; d < Blocks; d++) dk[d] = dv[d] = (floatx16)(0.f);
  }
  if (gk) store_column<T, Blocks>(gk + row * p.D, dk, p.scale, p.D, half, p.D % 4 == 0);
  if (gv) store_column<T, Blocks>(gv + row * p.D, dv, 1.f, p.D, half, p.D % 4 == 0);
}

// Sums per bucket of a head over the batch and the blocks of queries, in a fixed order: a
// workgroup has one head and 64 buckets, its waves every kWaves-th part.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void attention_table_grad_kernel(const float *partial,
                                                                           T *gtable, int B, int Hq,
                                                                           int nq, int NB) {
  __shared__ float part[kWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = blockIdx.y, n = blockIdx.x * 64 + lane;
  float x = 0.f;
  if (n < NB)
    for (int64_t s = wave; s < (int64_t)B * nq; s += kWaves)
      x += partial[((s / nq * Hq + h) * nq + s % nq) * NB + n];
  part[wave][lane] = x;
  __syncthreads();
  if (wave == 0 && n < NB) {
    for (int w = 1; w < kWaves; w++) x += part[w][lane];
    gtable[(int64_t)h * NB + n] = (T)x;
  }
}

static int64_t query_blocks(const Params &p) { return (p.Lq + kBlock - 1) / kBlock; }

static size_t backward_bytes(const Params &p) {
  const size_t rows = (size_t)p.B * p.Hq * p.Lq;
  return 2 * align256(rows * sizeof(float)) +
         align256((size_t)p.B * p.Hq * query_blocks(p) * p.NB * sizeof(float));
}

template <typename T>
static int launch_backward(const Params &p, const void *gout, const void *out, const float *stats,
                           void *gq, void *gk, void *gv, void *gtable, char *ws,
                           hipStream_t stream) {
  const size_t rows = (size_t)p.B * p.Hq * p.Lq;
  float *lses = (float *)ws, *deltas = (float *)(ws + align256(rows * sizeof(float)));
  float *partial = (float *)(ws + 2 * align256(rows * sizeof(float)));
  const int nq = (int)query_blocks(p), nk = (p.Lk + kBlock - 1) / kBlock;
  const dim3 threads(64 * kWaves);
  if (rows) {
    const dim3 grid((unsigned)((int64_t)p.B * p.Hq * nq));
    const size_t lds = (gtable ? 1 + kWaves : 1) * p.NB * sizeof(float);
#define MCX_GRAD(DP)                                                                              \
  hipLaunchKernelGGL((attention_query_grad_kernel<T, DP>), grid, threads, lds, stream, p,          \
                     (const T *)out, (const T *)gout, stats, lses, deltas, (T *)gq,               \
                     gtable ? partial : nullptr, nq)
    if (p.D <= 32) MCX_GRAD(32);
    else if (p.D <= 64) MCX_GRAD(64);
    else if (p.D <= 96) MCX_GRAD(96);
    else MCX_GRAD(128);
#undef MCX_GRAD
    MCX_HIP_CHECK_LAUNCH();
  }
  if (gtable) {
    hipLaunchKernelGGL((attention_table_grad_kernel<T>), dim3((p.NB + 63) / 64, p.Hq), threads, 0,
                       stream, partial, (T *)gtable, p.B, p.Hq, nq, p.NB);
    MCX_HIP_CHECK_LAUNCH();
  }
  if ((gk || gv) && p.B && p.Lk) {
    const dim3 grid((unsigned)((int64_t)p.B * p.Hk * nk));
    const size_t lds = p.NB * sizeof(float);
#define MCX_GRAD(DP)                                                                          \
  hipLaunchKernelGGL((attention_key_grad_kernel<T, DP>), grid, threads, lds, stream, p,        \
                     (const T *)gout, stats, lses, deltas, (T *)gk, (T *)gv, nk)
    if (p.D <= 32) MCX_GRAD(32);
    else if (p.D <= 64) MCX_GRAD(64);
    else if (p.D <= 96) MCX_GRAD(96);
    else MCX_GRAD(128);
#undef MCX_GRAD
    MCX_HIP_CHECK_LAUNCH();
  }
  return MCX_OK;
}

}  // namespace attention
}  // namespace mcx

extern "C" {

size_t mcx_attention_backward_workspace(const mcx_attention_desc *desc, int dtype) {
  using namespace mcx::attention;
  Params p;
  static const int32_t any = 0;  // (stands for pointers that are not read here)
  const bool biased = desc && desc->table_size > 0;
  if (make_params(p, &any, &any, &any, biased ? &any : nullptr, biased ? &any : nullptr, nullptr,
                  nullptr, desc, dtype) != MCX_OK)
    return 0;
  return backward_bytes(p);
}

int mcx_attention_backward(const void *gout, const void *q, const void *k, const void *v,
                           const void *out, const float *stats, const void *table,
                           const int32_t *buckets, const int32_t *query_start,
                           const int32_t *key_lengths, void *gq, void *gk, void *gv, void *gtable,
                           void *workspace, size_t workspace_bytes, const mcx_attention_desc *desc,
                           int dtype, void *stream) {
  using namespace mcx::attention;
  Params p;
  const int rc = make_params(p, q, k, v, table, buckets, query_start, key_lengths, desc, dtype);
  if (rc != MCX_OK) return rc;
  if (gtable && !table) return MCX_E_NULL;
  if (!gq && !gk && !gv && !gtable) return MCX_OK;
  if (p.B && p.Lq && (!gout || !out || !stats)) return MCX_E_NULL;
  if ((int64_t)p.B * p.Hq * query_blocks(p) > 0x7fffffffLL ||
      (int64_t)p.B * p.Hk * ((p.Lk + kBlock - 1) / kBlock) > 0x7fffffffLL)
    return MCX_E_SHAPE;
  const size_t need = backward_bytes(p);
  if (need && (!workspace || workspace_bytes < need)) return MCX_E_WORKSPACE;
  return dtype == MCX_BF16
             ? launch_backward<__bf16>(p, gout, out, stats, gq, gk, gv, gtable, (char *)workspace,
                                       (hipStream_t)stream)
             : launch_backward<float>(p, gout, out, stats, gq, gk, gv, gtable, (char *)workspace,
                                      (hipStream_t)stream);
}

}  // extern "C"
