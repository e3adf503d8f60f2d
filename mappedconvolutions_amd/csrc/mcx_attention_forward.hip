// Attention with a bias by relative-position buckets: the forward product and the C entry points.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "mcx_attention.h"

namespace mcx {
namespace attention {

// What rounding takes from ref c (0 where the difference from ref is formed first).
__device__ inline float residue_of(float ref, float c) {
  const float shift = ref * c;
  return fabsf(shift) > kHugeStat ? 0.f : fmaf(ref, c, -shift);
}

// One pass over the keys with a running reference and sum (both fp32): a workgroup holds 128
// queries of one head, a wave 32 of them, and walks the keys 64 at a time through two LDS buffers,
// the next tile's loads under way while the current one is multiplied.
//   The reference is the row's maximum, but it follows it only when a score exceeds it by 2^8:
// sums stay far inside fp32, and the accumulated output is seldom rescaled.
//   Exponents are one fma, u c - shift, with shift = ref c rounded: against u - ref they are off by
// residue = ref c - shift, the same for all keys.  It grows with the reference (0.03 at 10^6), so it is
// taken account of where references meet: when one moves, and in the sum that the gradients and the
// joining of parts take together with the reference itself.
//   bf16: probabilities are rounded to bf16 (2^-9 of each) to be the value product's operands, which the
// matrix instructions have at 8 times the rate of float32 ones; their sum takes them before that, in
// fp32.  Against 64 bits the output is off by 0.0021 .. 0.0024 of itself instead of 0.0016 .. 0.0017 with
// products in 32 bits and one rounding at the end.
//   Bound by vector and matrix instructions that mostly take turns.  512 x 8 heads of 512 rows of 64
// bf16 values: 0.50 ms, 548 TFLOP/s, vector instructions 56 % of the time (a score's exponent,
// maximum, sum and conversion), matrix instructions 26 %, LDS 27 %; 16 heads of 8192 rows of 128
// sharing 4: 0.58 ms, 950 TFLOP/s, 44 and 45 %.  A large bf16 product reaches 1244 TFLOP/s.
template <typename T, int DP, bool Wide>
__global__ __launch_bounds__(64 * kWaves, (waves_per_simd<T, DP>(3))) void attention_forward_kernel(
    Params p, T *out, float *stats, T *rest, float *outs, float *sums, int nq, int parts) {
  constexpr int Chunks = DP / 16, Blocks = DP / 32;
  __shared__ Word ks[2][kTile * words<T, DP>()];
  __shared__ Word vs[2][kTile * words<T, DP>()];
  __shared__ __attribute__((aligned(16))) Window window[2];
  extern __shared__ float table[];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int wg = group_of_call(p), part = wg % parts, unit = wg / parts;
  const Unit u0 = unit_of(p, unit, p.Hq / p.Hk, nq);
  const int b = u0.b, kh = u0.kh, h = kh * (p.Hq / p.Hk) + u0.g;
  const int i0 = (nq - 1 - u0.block) * kBlock;  // the longest rows of a causal map first
  const int start = first_position(p, b), length = key_length(p, b);
  const int local = wave * kLanesRows + (lane & 31), i = i0 + local;
  const bool live = i < p.Lq;
  const int limit = p.causal ? min(length, start + i + 1) : length;  // keys of this query
  const int last = min(i0 + kBlock, p.Lq) - 1;
  const int keys = p.causal ? max(0, min(length, start + last + 1)) : length;
  const int wave_limit = p.causal ? min(length, start + i0 + wave * kLanesRows + 1) : length;

  const T *q = (const T *)p.q + b * p.qs[0] + (int64_t)i * p.qs[1] + h * p.qs[2];
  const T *k = (const T *)p.k + b * p.ks[0] + kh * p.ks[2];
  const T *v = (const T *)p.v + b * p.vs[0] + kh * p.vs[2];
  const bool biased = p.table != nullptr;

  Frag<T> qf[Chunks];
#pragma unroll
  for (int c = 0; c < Chunks; c++) qf[c] = global_frag<Wide>(live ? q : nullptr, c, half, p.D);

  // window value t stands for the difference (first key of the tile) - (position of query
  // i0 + kBlock) + t
  const int base = -(start + i0 + kBlock);
  Feed<T, DP, Wide> kt(p.ks[1], p.D, tid), vt(p.vs[1], p.D, tid);
  int bucket = 0;
  const int all = (keys + kTile - 1) / kTile, each = (all + parts - 1) / parts;
  const int first = part * each, tiles = min(all, first + each);  // of this part
  if (first < tiles) {
    const int64_t next = (int64_t)first * kTile;
    kt.start(k + next * p.ks[1], p.ks[1], keys - (int)next, ks[0], p.D, tid);
    vt.start(v + next * p.vs[1], p.vs[1], keys - (int)next, vs[0], p.D, tid);
    if (biased) bucket = bucket_of(p, base + (int)next + tid);
  }
  if (biased) load_table<T>(p, h, table, tid, 64 * kWaves);
  else clear(window, tid);
  loads_done();
  __syncthreads();  // the table
  if (first < tiles) {
    kt.finish(ks[0], tid);
    vt.finish(vs[0], tid);
    if (biased && tid < kWindow) window[0].put(tid, bias_of(table, p.NB, bucket));
  }
  __syncthreads();

  const float c = p.scale * kLog2e;
  const int at = kBlock - local + 32 * half, shift = at & 3;
  floatx16 o[Blocks];
#pragma unroll
  for (int d = 0; d < Blocks; d++) o[d] = (floatx16)(0.f);
  float ref = -kInf, sum = 0.f;

  // (one copy for each buffer: its place is then part of the instructions)
  auto tile = [&](int t, auto which) {
    constexpr int buf = decltype(which)::value;
    const int j0 = t * kTile;
    if (t + 1 < tiles) {
      const int64_t next = j0 + kTile;
      kt.start(k + next * p.ks[1], p.ks[1], keys - (int)next, ks[buf ^ 1], p.D, tid);
      vt.start(v + next * p.vs[1], p.vs[1], keys - (int)next, vs[buf ^ 1], p.D, tid);
      if (biased) bucket = bucket_of(p, base + (int)next + tid);
    }
    floatx16 u[2];
#pragma unroll
    for (int blk = 0; blk < 2; blk++) {
      u[blk] = sixteen(window[buf].get(at + 16 * blk, shift), window[buf].get(at + 16 * blk + 8, shift));
#pragma unroll
      for (int ch = 0; ch < Chunks; ch++)
        u[blk] = mma(row_frag<T, DP>(ks[buf], row_of(lane & 31, blk), ch, half), qf[ch], u[blk]);
    }
    if (j0 + kTile > wave_limit) {
#pragma unroll
      for (int blk = 0; blk < 2; blk++)
        keep_between(u[blk], 0, limit - (j0 + 32 * half + 16 * blk));
    }
    float top = u[0][0];
#pragma unroll
    for (int blk = 0; blk < 2; blk++)
#pragma unroll
      for (int n = 0; n < 16; n++) top = fmaxf(top, u[blk][n]);
    top = fmaxf(top, other_half(top));
    if (__any((top - ref) * c > 8.f)) {  // (-inf against -inf is no number: not above)
      const float next = fmaxf(ref, top);
      const float moved = residue_of(next, c) - residue_of(ref, c);
      const float keep = next == -kInf ? 1.f : exp2_fast(fmaf(ref - next, c, moved));
      ref = next;
      sum *= keep;
#pragma unroll
      for (int d = 0; d < Blocks; d++) o[d] *= keep;
    }
    const float used = ref == -kInf ? 0.f : ref;
    if (__any(fabsf(used) * c > kHugeStat)) {
      const float residue = residue_of(used, c);
#pragma unroll
      for (int blk = 0; blk < 2; blk++)
#pragma unroll
        for (int n = 0; n < 16; n++) u[blk][n] = exp2_fast(fmaf(u[blk][n] - used, c, residue));
    } else {
      const float shiftc = -used * c;
#pragma unroll
      for (int blk = 0; blk < 2; blk++)
#pragma unroll
        for (int n = 0; n < 16; n++) u[blk][n] = exp2_fast(fmaf(u[blk][n], c, shiftc));
    }
    float part = 0.f;
#pragma unroll
    for (int blk = 0; blk < 2; blk++) {
#pragma unroll
      for (int n = 0; n < 16; n++) part += u[blk][n];
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const Frag<T> pf = Frag<T>::pack(eight(u[blk], s));
#pragma unroll
        for (int d = 0; d < Blocks; d++)
          o[d] = mma(Column<T, DP, 32>::get(vs[buf], 16 * blk + 8 * s, d, lane), pf, o[d]);
      }
    }
    sum += part;
    if (t + 1 < tiles) {
      kt.finish(ks[buf ^ 1], tid);
      vt.finish(vs[buf ^ 1], tid);
      if (biased && tid < kWindow) window[buf ^ 1].put(tid, bias_of(table, p.NB, bucket));
    }
    __syncthreads();
  };
  for (int t = first; t < tiles; t += 2) {
    tile(t, std::integral_constant<int, 0>{});
    if (t + 1 < tiles) tile(t + 1, std::integral_constant<int, 1>{});
  }
  sum += other_half(sum);
  if (!live) return;
  const int64_t row = ((int64_t)b * p.Lq + i) * p.Hq + h;
  const int64_t stat = ((int64_t)b * p.Hq + h) * p.Lq + i;
  const float of_ref = exp2_fast(-residue_of(ref, c));
  if (parts > 1) {
    const int64_t rows = (int64_t)p.B * p.Lq * p.Hq;
    store_column<Wide, float, Blocks>(outs + (part * rows + row) * p.D, o, of_ref, p.D, half);
    stats = sums + part * rows * 2;
  } else {
    store_column<Wide, T, Blocks>(out + row * p.D, o, sum == 0.f ? 0.f : 1.f / sum, p.D, half,
                                  rest ? rest + row * p.D : nullptr);
  }
  if (stats && half == 0) {
    stats[2 * stat] = ref;
    stats[2 * stat + 1] = sum * of_ref;
  }
}

// Joins the parts of the keys: a thread has one value of the output.
template <typename T>
__global__ __launch_bounds__(256) void attention_join_values_kernel(Params p, const float *outs,
                                                                    const float *sums, T *out,
                                                                    float *stats, T *rest, int parts) {
  const int64_t rows = (int64_t)p.B * p.Lq * p.Hq, n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= rows * p.D) return;
  const int64_t row = n / p.D, bi = row / p.Hq, b = bi / p.Lq;
  const int64_t stat = (b * p.Hq + row % p.Hq) * p.Lq + bi % p.Lq;
  const float c = p.scale * kLog2e;
  float top = -kInf, all = 0.f, x = 0.f;
  for (int s = 0; s < parts; s++) top = fmaxf(top, sums[(s * rows + stat) * 2]);
  for (int s = 0; s < parts; s++) {
    const float ref = sums[(s * rows + stat) * 2];
    const float w = ref == -kInf ? 1.f : exp2_fast((ref - top) * c);  // (a NaN part stays one)
    all = fmaf(w, sums[(s * rows + stat) * 2 + 1], all);
    x = fmaf(w, outs[s * rows * p.D + n], x);
  }
  store_value(out, rest, n, all == 0.f ? 0.f : x / all);
  if (stats && n % p.D == 0) {
    stats[2 * stat] = top;
    stats[2 * stat + 1] = all;
  }
}

static int64_t query_units(const Params &p) {
  return (int64_t)p.B * p.Hq * ((p.Lq + kBlock - 1) / kBlock);
}
static int forward_parts(const Params &p) {
  return parts_of(query_units(p), (p.Lk + kTile - 1) / kTile);
}
static size_t forward_bytes(const Params &p) {
  const int parts = forward_parts(p);
  if (parts == 1) return 0;
  const size_t rows = (size_t)p.B * p.Hq * p.Lq * parts;
  return align256(rows * 2 * sizeof(float)) + align256(rows * p.D * sizeof(float));
}

template <typename T>
static int launch_forward(const Params &p, void *out, float *stats, void *rest, void *workspace,
                          hipStream_t stream) {
  const int nq = (p.Lq + kBlock - 1) / kBlock, parts = forward_parts(p);
  const dim3 threads(64 * kWaves);
  const int64_t rows = (int64_t)p.B * p.Hq * p.Lq;
  float *sums = (float *)workspace;
  float *outs = (float *)((char *)workspace + align256((size_t)rows * parts * 2 * sizeof(float)));
  const size_t lds = p.table ? p.NB * sizeof(float) : 0;
  const int rc = launch_in_pieces(p, query_units(p) * parts, [&](const Params &piece, dim3 grid) {
#define MCX_FORWARD(DP, W)                                                                          \
  hipLaunchKernelGGL((attention_forward_kernel<T, DP, W>), grid, threads, lds, stream, piece, (T *)out, \
                     stats, (T *)rest, outs, sums, nq, parts)
    MCX_ATTENTION_DISPATCH(p.D, p.wide && aligned16(out) && aligned16(rest), MCX_FORWARD);
#undef MCX_FORWARD
  });
  if (rc != MCX_OK) return rc;
  if (parts > 1) {
    hipLaunchKernelGGL((attention_join_values_kernel<T>), dim3((unsigned)((rows * p.D + 255) / 256)),
                       dim3(256), 0, stream, p, outs, sums, (T *)out, stats, (T *)rest, parts);
    MCX_HIP_CHECK_LAUNCH();
  }
  return MCX_OK;
}

// Whether rows are whole 16-byte words, and a tile's offsets fit 32 bits.
static bool wide_rows(const void *p, const int64_t *strides, int64_t D, int64_t per16) {
  return aligned16(p) && D % per16 == 0 && strides[0] % per16 == 0 && strides[1] % per16 == 0 &&
         strides[2] % per16 == 0 && strides[1] >= 0 && strides[1] < (1 << 22);
}

int parts_of(int64_t units, int64_t tiles) {
  if (units >= 256) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>((384 + units - 1) / units, tiles / 4));
}

int make_params(Params &p, const void *q, const void *k, const void *v, const void *table,
                const int32_t *buckets, const int32_t *query_start, const int32_t *key_lengths,
                const mcx_attention_desc *d, int dtype) {
  if (!d) return MCX_E_NULL;
  if (dtype != MCX_F32 && dtype != MCX_BF16) return MCX_E_DTYPE;
  const int64_t most = 1 << 28;
  if (d->B < 0 || d->Lq < 0 || d->Lk < 0 || d->B > most || d->Lq > most || d->Lk > most)
    return MCX_E_SHAPE;
  if (d->D < 1 || d->D > kMaxD || d->Hk < 1 || d->Hq < 1 || d->Hq > 65535 || d->Hq % d->Hk)
    return MCX_E_SHAPE;
  if (!(d->scale >= 1e-6 && d->scale <= 1e6)) return MCX_E_SHAPE;
  if (d->B && d->Lq && (!q || (d->Lk && (!k || !v)))) return MCX_E_NULL;
  if ((table != nullptr) != (buckets != nullptr)) return MCX_E_NULL;
  if (table && (d->table_size < 1 || d->table_size > kMaxTable || d->bucket_count < 1 ||
                d->bucket_count > kMostPosition || d->bucket_zero < 0 ||
                d->bucket_zero >= d->bucket_count))
    return MCX_E_SHAPE;
  p.q = q, p.k = k, p.v = v, p.table = table;
  p.buckets = buckets, p.start = query_start, p.lengths = key_lengths;
  for (int n = 0; n < 3; n++)
    p.qs[n] = d->q_stride[n], p.ks[n] = d->k_stride[n], p.vs[n] = d->v_stride[n];
  p.B = (int)d->B, p.Lq = (int)d->Lq, p.Lk = (int)d->Lk;
  p.Hq = (int)d->Hq, p.Hk = (int)d->Hk, p.D = (int)d->D;
  p.R = table ? (int)d->bucket_count : 0, p.zero = table ? (int)d->bucket_zero : 0;
  p.NB = table ? (int)d->table_size : 0, p.causal = d->causal != 0;
  p.scale = (float)d->scale;
  const int64_t per16 = dtype == MCX_BF16 ? 8 : 4;
  p.wide = wide_rows(q, p.qs, p.D, per16) && wide_rows(k, p.ks, p.D, per16) &&
           wide_rows(v, p.vs, p.D, per16);
  // The order of the work (plain, this, in us; bf16, forward and gradients where not said): 16
  // heads of 64 sharing 4, 4 causal sequences of 2048: 438, 379; forward over up to 2562: 100, 85;
  // 16 x 8 heads of up to 1024 rows: 231, 168; 8 x 8 heads of up to 1024, not causal: 134, 124.
  //   All heads of an XCD together where their keys and values fit its 4 MB of L2, since all of them
  // are then read again and again.  8 x 32 heads of 128 sharing 8 over up to 8192: forward 4770, 4310
  // with one key head after the other.
  //   From 32 sequences on, an XCD's own are mixed enough, and all heads of one stay with it: their
  // rows lie side by side (64 x 16 heads of up to 512: 520 plain, 541 with every eighth head, 513).
  const int64_t held = ((int64_t)p.B * p.Hk + 7) / 8 * 2 * p.Lk * p.D * (16 / per16);
  p.order = !p.causal && !p.lengths ? kPlain : p.causal && held <= (4 << 20) ? kTogether : kMixed;
  p.run = p.B >= 32 ? p.Hk : 1;
  p.first = 0;
  return MCX_OK;
}

}  // namespace attention
}  // namespace mcx

extern "C" {

size_t mcx_attention_forward_workspace(const mcx_attention_desc *desc, int dtype) {
  using namespace mcx::attention;
  Params p;
  static const int32_t any = 0;  // (stands for pointers that are not read here)
  const int32_t *table = desc && desc->table_size > 0 ? &any : nullptr;
  if (make_params(p, &any, &any, &any, table, table, nullptr, nullptr, desc, dtype) != MCX_OK)
    return 0;
  if (p.B == 0 || p.Lq == 0) return 0;
  const int parts = split_parts(p, dtype);
  return parts ? split_bytes(p, parts) : forward_bytes(p);
}

int mcx_attention_forward(const void *q, const void *k, const void *v, const void *table,
                          const int32_t *buckets, const int32_t *query_start,
                          const int32_t *key_lengths, void *out, float *stats, void *out_rest,
                          void *workspace, size_t workspace_bytes, const mcx_attention_desc *desc, int dtype,
                          void *stream) {
  using namespace mcx::attention;
  Params p;
  const int rc = make_params(p, q, k, v, table, buckets, query_start, key_lengths, desc, dtype);
  if (rc != MCX_OK) return rc;
  if (p.B == 0 || p.Lq == 0) return MCX_OK;
  if (!out) return MCX_E_NULL;
  const int parts = split_parts(p, dtype);
  if (parts) {
    if (split_bytes(p, parts) && (!workspace || workspace_bytes < split_bytes(p, parts)))
      return MCX_E_WORKSPACE;
    return launch_split(p, parts, out, stats, out_rest, workspace, dtype, (hipStream_t)stream);
  }
  if (query_units(p) > 0x7fffffffLL) return MCX_E_SHAPE;
  if (forward_bytes(p) && (!workspace || workspace_bytes < forward_bytes(p))) return MCX_E_WORKSPACE;
  return dtype == MCX_BF16
             ? launch_forward<__bf16>(p, out, stats, out_rest, workspace, (hipStream_t)stream)
             : launch_forward<float>(p, out, stats, nullptr, workspace, (hipStream_t)stream);
}

}  // extern "C"
