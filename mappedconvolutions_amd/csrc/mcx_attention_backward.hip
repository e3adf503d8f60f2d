// Gradients of attention with a bias by relative-position buckets.
//
//   p_ij = exp(scale (u_ij - ref_i)) / sum_i,  dp_ij = do_i . v_j,  delta_i = do_i . o_i
//   ds_ij = p_ij (dp_ij - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//   dT[h, n] = sum of ds over the pairs of bucket n
//
// bf16: p and ds are formed in fp32 and rounded to bf16 (2^-9 of each) as operands of the last three
// products; the sums per bucket take ds before that.
//
// Scores are computed again in both kernels (seven products of a tile instead of five): every
// gradient then has one owner, who sums it in registers in a fixed order.  No atomics on memory,
// the same bits each time.
#include <algorithm>
#include <type_traits>

#include "mcx_attention.h"

namespace mcx {
namespace attention {

// What the two kernels share of every row: [B, Hq, Lq].  delta is negative; ref is +inf for a row
// that nothing is left of.
struct Rows {
  float *ref, *log_sum, *delta;
};

// c + a b^T of a column a (rows) and a row b (columns), the upper half-wave's a being 0: takes
// delta from dp in the matrix pipe, which has the time, and after dp's last addition: equal sums
// of equal terms then leave nothing.
__device__ inline floatx16 add_outer(float a, float b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// A step along two chains of diagonals: ds plus the running sum of the lane below (lane 63's for lane
// 0), none for the lane where `kept` is 0.  The wait is what a lane exchange needs after a write of
// its source: two chains share it.
__device__ inline void next_diagonals(float &ds0, float sum0, float &ds1, float sum1, float kept) {
  asm("s_nop 1\n\t"
      "v_fmac_f32_dpp %0, %2, %4 wave_ror:1 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %1, %3, %4 wave_ror:1 row_mask:0xf bank_mask:0xf"
      : "+&v"(ds0), "+v"(ds1) : "v"(sum0), "v"(sum1), "v"(kept));
}

// The sum of x over the lanes up to this one in its run of lanes with the same n, and whether the run
// ends here.  (Neighbouring differences mostly share a bucket, and 64 lanes' additions to one
// place in LDS take four clocks each.)
template <int Control, int Rows> __device__ inline float from_lane(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), Control, Rows, 0xf, false));
}
__device__ inline float run_sum(float x, int n, int lane, bool &last) {
  const int below = __builtin_amdgcn_update_dpp(0, n, 0x138, 0xf, 0xf, false);  // lane - 1
  const uint64_t starts = __builtin_amdgcn_ballot_w64(lane == 0 || below != n);
  last = lane == 63 || (starts >> (lane + 1)) & 1;
  const int before = lane - (63 - __builtin_clzll(starts & (~0ull >> (63 - lane))));  // in the run
  float y = from_lane<0x111, 0xf>(x);  // 1, 2, 4, 8 lanes down, within 16
  x += before >= 1 ? y : 0.f;
  y = from_lane<0x112, 0xf>(x);
  x += before >= 2 ? y : 0.f;
  y = from_lane<0x114, 0xf>(x);
  x += before >= 4 ? y : 0.f;
  y = from_lane<0x118, 0xf>(x);
  x += before >= 8 ? y : 0.f;
  y = from_lane<0x142, 0xa>(x);  // lane 15 to lanes 16 .. 31, lane 47 to 48 .. 63
  x += before > (lane & 15) ? y : 0.f;
  y = from_lane<0x143, 0xc>(x);  // lane 31 to lanes 32 .. 63
  x += before > lane - 32 ? y : 0.f;
  return x;
}
// The upper half-wave's values in the lower, zeros in the upper.
__device__ inline float upper_to_lower(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), 0u, false, false);
  return __uint_as_float(r[1]);
}

// x, which the compiler takes for new: what is computed from it is computed here, and not kept in
// registers from before the loop.
__device__ inline int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A step of a pipeline ends here: the compiler's scheduler keeps its instructions together.
__device__ inline void step_end() { __builtin_amdgcn_sched_barrier(0); }

// u += rows of `a` times x, dp += rows of `b` times y, for one 32 x 32 block of a tile's pairs.  The
// operands are loaded `Ahead` chunks before their products, and `beside(n)`, n = 0 .. Chunks - 1, is
// vector work that the matrix pipe's time is long enough for.
template <typename T, int DP, int Ahead, typename F>
__device__ inline void scores(const Word *a, const Word *b, int blk, int lane, const Frag<T> *x,
                              const Frag<T> *y, floatx16 &u, floatx16 &dp, F beside) {
  constexpr int Chunks = DP / 16;
  const int row = row_of(lane & 31, blk), half = lane >> 5;
  Frag<T> fa[Chunks], fb[Chunks];
#pragma unroll
  for (int ch = -Ahead; ch < Chunks; ch++) {
    if (ch + Ahead < Chunks) {
      fa[ch + Ahead] = row_frag<T, DP>(a, row, ch + Ahead, half);
      fb[ch + Ahead] = row_frag<T, DP>(b, row, ch + Ahead, half);
    }
    if (ch < 0) continue;
    u = mma(fa[ch], x[ch], u);
    dp = mma(fb[ch], y[ch], dp);
    beside(ch);
    step_end();
  }
}
// The part [n of steps) of the 16 values of a block.
__device__ inline constexpr int part_start(int n, int steps) { return 16 * n / steps; }

// Queries' gradients, the sums per bucket, and the rows' statistics for the other kernel.  The
// same walk as the forward product's: a wave holds 32 queries, their o gradient beside them.
//   The bias' gradient needs the sums of ds along the diagonals j - i.  A lane holds query lane & 31
// and the keys 32 (lane >> 5) + n, n = 0 .. 31: from n to n + 1 a diagonal moves one lane up, so
// one instruction a value adds it to its neighbour's running sum.  What reaches lane 31 is finished
// and leaves (lane 32 starts anew); what leaves lane 63 is the part of a diagonal that lane 0 goes
// on with.  Two chains, over n < 16 and n >= 16, run side by side, and the first one's ends are added
// where their 16 further steps would have taken them: lane l to lane l + 16, or, past lane 31, out at
// step 47 - l.  The 64 diagonals that a tile finishes are added to the wave's sums per bucket.
//   (Adding each ds to a sum in LDS costs about 3 clocks a value: 6.9 ms for 512 x 8 heads of 512 rows
// of 64 bf16 values, which take 0.90 ms this way.)
//   Bound by vector and matrix instructions that mostly take turns: these 0.90 ms are 457 TFLOP/s of
// three products (vector instructions 48 %, matrix 25 %, LDS 30 % of the time), 16 heads of 8192 rows
// of 128 sharing 4 take 0.96 ms, 862 TFLOP/s.
template <typename T, int DP, bool Wide, bool Table>
__global__ __launch_bounds__(64 * kWaves, (waves_per_simd<T, DP>(3))) void attention_query_grad_kernel(
    Params p, const T *out, const T *rest, const T *gout, const float *stats, Rows rows, T *gq, float *gq_parts,
    float *partial, int nq, int parts) {
  constexpr int Chunks = DP / 16, Blocks = DP / 32;
  constexpr int Ahead = DP * (int)sizeof(T) > 128 ? 1 : 2;  // (registers: two waves a SIMD)
  __shared__ Word ks[2][kTile * words<T, DP>()];
  __shared__ Word vs[2][kTile * words<T, DP>()];
  __shared__ __attribute__((aligned(16))) Window window[2];
  __shared__ int window_bucket[2][kWindow];
  __shared__ __attribute__((aligned(16))) float finished[kWaves][64];
  __shared__ float chain_end[kWaves][64];
  extern __shared__ float table[];  // NB values, then kWaves x NB sums

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int wg = group_of_call(p), part = wg % parts, unit = wg / parts;
  const Unit u0 = unit_of(p, unit, p.Hq / p.Hk, nq);
  const int b = u0.b, kh = u0.kh, h = kh * (p.Hq / p.Hk) + u0.g, bh = b * p.Hq + h;
  const int block = nq - 1 - u0.block, i0 = block * kBlock;
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
  const bool biased = p.table != nullptr;
  float *sums = table + p.NB + wave * p.NB;

  // the first tile is on its way while the rows' own values are loaded; none where only the
  // statistics are asked for
  const int base = -(start + i0 + kBlock);
  Feed<T, DP, Wide> kt(p.ks[1], p.D, tid), vt(p.vs[1], p.D, tid);
  int bucket = 0;
  const int all = (keys + kTile - 1) / kTile, each = (all + parts - 1) / parts;
  const int first = part * each, tiles = gq || Table ? min(all, first + each) : 0;  // of this part
  if (first < tiles) {
    const int64_t next = (int64_t)first * kTile;
    kt.start(k + next * p.ks[1], p.ks[1], keys - (int)next, ks[0], p.D, tid);
    vt.start(v + next * p.vs[1], p.vs[1], keys - (int)next, vs[0], p.D, tid);
    if (biased) bucket = bucket_of(p, base + (int)next + tid);
  }

  Frag<T> qf[Chunks], gf[Chunks];
  // delta is the diagonal of a product of the same kind as dp's: where a row's output is one of
  // its values, the two are the same number and their difference is nothing.  It takes in what the
  // output's rounding left over: all pairs of a row share delta's error, so it does not cancel in
  // the sums per bucket (512 bf16 rows of 512: the bias' gradient is off by 0.0034 of itself without
  // it and 0.0028 with it; what is left is the probabilities' rounding before the forward product)
  floatx16 products = (floatx16)(0.f);
#pragma unroll
  for (int c = 0; c < Chunks; c++) {
    qf[c] = global_frag<Wide>(live ? q : nullptr, c, half, p.D);
    gf[c] = global_frag<Wide>(live ? gout + row * p.D : nullptr, c, half, p.D);
    if (rest)
      products = mma(global_frag<Wide>(live ? rest + row * p.D : nullptr, c, half, p.D), gf[c], products);
    products = mma(global_frag<Wide>(live ? out + row * p.D : nullptr, c, half, p.D), gf[c], products);
  }
  float delta = 0.f;
#pragma unroll
  for (int n = 0; n < 16; n++)  // row 8 (n >> 2) + 4 half + (n & 3)
    if ((lane & 31) == 8 * (n >> 2) + 4 * half + (n & 3)) delta = products[n];
  delta += other_half(delta);
  const float c = p.scale * kLog2e;
  // (a row that nothing is left of: every difference from ref is -inf)
  float ref = kInf, log_sum = 0.f;
  const int64_t stat = ((int64_t)b * p.Hq + h) * p.Lq + i;
  if (live) {
    const float row_ref = stats[2 * stat], row_sum = stats[2 * stat + 1];
    if (row_ref != -kInf) ref = row_ref, log_sum = __log2f(row_sum);
  }
  if (live && half == 0 && part == 0) {
    rows.ref[stat] = ref;
    rows.log_sum[stat] = log_sum;
    rows.delta[stat] = -delta;
  }
  if (!gq && !Table) return;

  if (Table) {
    for (int n = lane; n < p.NB; n += 64) sums[n] = 0.f;
    finished[wave][lane] = chain_end[wave][lane] = 0.f;
  }
  if (biased) load_table<T>(p, h, table, tid, 64 * kWaves);
  else clear(window, tid);
  loads_done();
  __syncthreads();
  if (first < tiles) {
    kt.finish(ks[0], tid);
    vt.finish(vs[0], tid);
    if (biased && tid < kWindow) {
      window[0].put(tid, bias_of(table, p.NB, bucket));
      window_bucket[0][tid] = bucket;
    }
  }
  __syncthreads();

  const int at = kBlock - local + 32 * half, shift = at & 3;
  const float kept = lane == 32 ? 0.f : 1.f;
  float diagonals = 0.f, second = 0.f;  // the two chains
  int finished_bucket = -1;
  // What a tile has finished goes to the sums while the next one's products are under way; what its
  // upper half-wave holds goes on in that one's lower half, one lane up.
  auto finish_diagonals = [&] {
    const float above = chain_end[wave][(lane - 16) & 63];
    const float first_chain = chain_end[wave][(47 - lane) & 63];
    diagonals = upper_to_lower(second + (lane >= 48 ? above : 0.f));
    bool last;
    const float value = run_sum(finished[wave][lane] + (lane >= 16 ? first_chain : 0.f),
                                finished_bucket, lane, last);
    if (last && (unsigned)finished_bucket < (unsigned)p.NB) atomicAdd(&sums[finished_bucket], value);
    wave_order();
  };
  floatx16 acc[Blocks];
#pragma unroll
  for (int d = 0; d < Blocks; d++) acc[d] = (floatx16)(0.f);

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
    floatx16 u[2], dp[2];
#pragma unroll
    for (int blk = 0; blk < 2; blk++) {
      u[blk] = sixteen(window[buf].get(at + 16 * blk, shift), window[buf].get(at + 16 * blk + 8, shift));
      dp[blk] = (floatx16)(0.f);
      // (what is -inf before the product stays it)
      if (j0 + kTile > wave_limit) keep_between(u[blk], 0, limit - (j0 + 32 * half + 16 * blk));
    }
    {
      // A pipeline over the two blocks of 32 keys: the vector work of one stands beside the
      // products of the other.
      const int lane = here(threadIdx.x & 63), half = lane >> 5;
      Frag<T> ds[2];
      auto begin = [&](int blk, auto beside) {
        scores<T, DP, Ahead>(ks[buf], vs[buf], blk, lane, qf, gf, u[blk], dp[blk], beside);
        dp[blk] = add_outer(half ? 0.f : 1.f, -delta, dp[blk]);
      };
      auto gradients = [&](int blk, int n0, int n1) {
#pragma unroll
        for (int n = n0; n < n1; n++) dp[blk][n] *= exp2_fast(fmaf(u[blk][n] - ref, c, -log_sum));
      };
      auto to_queries = [&](int blk, auto beside) {
        ds[0] = Frag<T>::pack(eight(dp[blk], 0));
        ds[1] = Frag<T>::pack(eight(dp[blk], 1));
        Frag<T> f[2 * Blocks];
#pragma unroll
        for (int n = -Ahead; n < 2 * Blocks; n++) {
          if (const int m = n + Ahead; m < 2 * Blocks)
            f[m] = Column<T, DP, 32>::get(ks[buf], 16 * blk + 8 * (m / Blocks), m % Blocks, lane);
          if (n < 0) continue;
          acc[n % Blocks] = mma(f[n], ds[n / Blocks], acc[n % Blocks]);
          beside(n);
          step_end();
        }
      };
      begin(0, [](int) {});
      if constexpr (Table) finish_diagonals();
      begin(1, [&](int n) { gradients(0, part_start(n, Chunks), part_start(n + 1, Chunks)); });
      to_queries(0, [&](int n) { gradients(1, part_start(n, 2 * Blocks), part_start(n + 1, 2 * Blocks)); });
      floatx16 left[2];  // what lane 31 held before each step: a finished diagonal
      second = 0.f;
      to_queries(1, [&](int n) {
        if constexpr (Table) {
#pragma unroll
          for (int m = part_start(n, 2 * Blocks); m < part_start(n + 1, 2 * Blocks); m++) {
            left[0][m] = diagonals, left[1][m] = second;
            float x = dp[0][m], y = dp[1][m];
            next_diagonals(x, diagonals, y, second, kept);
            diagonals = x, second = y;
          }
        }
      });
      if constexpr (Table) {
        chain_end[wave][lane] = diagonals;
        if (lane == 31) {
          floatx4 *to = (floatx4 *)finished[wave];
#pragma unroll
          for (int n = 0; n < 8; n++)
            to[n] = floatx4{left[n / 4][4 * (n % 4)], left[n / 4][4 * (n % 4) + 1],
                            left[n / 4][4 * (n % 4) + 2], left[n / 4][4 * (n % 4) + 3]};
        }
        // the lower half-wave's sums are finished (difference 31 - lane)
        if (half == 0) finished[wave][63 - lane] = second;
        finished_bucket = window_bucket[buf][lane + kBlock - 32 - wave * kLanesRows];
        wave_order();
      }
    }
    if (t + 1 < tiles) {
      kt.finish(ks[buf ^ 1], tid);
      vt.finish(vs[buf ^ 1], tid);
      if (biased && tid < kWindow) {
        window[buf ^ 1].put(tid, bias_of(table, p.NB, bucket));
        window_bucket[buf ^ 1][tid] = bucket;
      }
    }
    __syncthreads();
  };
  for (int t = first; t < tiles; t += 2) {
    tile(t, std::integral_constant<int, 0>{});
    if (t + 1 < tiles) tile(t + 1, std::integral_constant<int, 1>{});
  }
  if constexpr (Table) {
    finish_diagonals();
    if (first < tiles && half == 0) {  // differences 63 - lane of the last tile
      const int n = window_bucket[(tiles - 1 - first) & 1][63 - lane + kBlock - wave * kLanesRows];
      if ((unsigned)n < (unsigned)p.NB) atomicAdd(&sums[n], diagonals);
    }
    __syncthreads();
    float *to = partial + (((int64_t)bh * nq + block) * parts + part) * p.NB;
    for (int n = tid; n < p.NB; n += 64 * kWaves) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; w++) x += table[p.NB + w * p.NB + n];
      to[n] = x;
    }
  }
  if (!live || !gq) return;
  if (parts == 1) {
    store_column<Wide, T, Blocks>(gq + row * p.D, acc, p.scale, p.D, half);
  } else {
    const int64_t size = (int64_t)p.B * p.Lq * p.Hq;
    store_column<Wide, float, Blocks>(gq_parts + (part * size + row) * p.D, acc, p.scale, p.D, half);
  }
}

// Keys' and values' gradients: a workgroup holds 128 keys of a key head, a wave 32 of them as
// columns, and walks the queries of all heads that share them, 64 at a time.
//   Bound as the others: 512 x 8 heads of 512 rows of 64 bf16 values take 0.89 ms, 618 TFLOP/s of four
// products (vector instructions 40 %, matrix 32 %, LDS 30 % of the time), 16 heads of 8192 rows of 128
// sharing 4 take 1.34 ms, 818 TFLOP/s, with one wave a SIMD: two sums, the held keys and values fill
// its registers.
template <typename T, int DP, bool Wide>
__global__ __launch_bounds__(64 * kWaves, (waves_per_simd<T, DP>(6))) void attention_key_grad_kernel(
    Params p, const T *gout, Rows rows, T *gk, T *gv, float *gk_parts, float *gv_parts, int nk, int parts) {
  constexpr int Chunks = DP / 16, Blocks = DP / 32, Ahead = 3;
  __shared__ Word qs[2][kTile * words<T, DP>()];
  __shared__ Word gs[2][kTile * words<T, DP>()];
  __shared__ __attribute__((aligned(16))) Window window[2];
  __shared__ __attribute__((aligned(16))) float row_ref[2][kTile], row_log[2][kTile], row_delta[2][kTile];
  extern __shared__ float table[];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int wg = group_of_call(p), part = wg % parts, unit = wg / parts;
  const Unit u0 = unit_of(p, unit, 1, nk);
  const int b = u0.b, kh = u0.kh;
  const int j0 = u0.block * kBlock;  // the longest columns of a causal map first
  const int group = p.Hq / p.Hk;
  const int start = first_position(p, b), length = key_length(p, b);
  const int local = wave * kLanesRows + (lane & 31), j = j0 + local;
  const bool live = j < p.Lk, used = j < length;
  // the first query that sees a key of this workgroup, and of this lane
  const int first = p.causal ? max(0, j0 - start) : 0;
  const int own_first = p.causal ? j - start : 0;
  const int tf = first / kTile, per_head = j0 < length ? max(0, (p.Lq + kTile - 1) / kTile - tf) : 0;
  // this part's of the tiles of all heads, one head after the other
  const int each = (group * per_head + parts - 1) / parts, from = part * each;
  const int upto = min(group * per_head, from + each);
  const int wave_safe = p.causal ? j0 + wave * kLanesRows + kLanesRows - 1 - start : 0;

  const T *k = (const T *)p.k + b * p.ks[0] + (int64_t)j * p.ks[1] + kh * p.ks[2];
  const T *v = (const T *)p.v + b * p.vs[0] + (int64_t)j * p.vs[1] + kh * p.vs[2];
  const bool biased = p.table != nullptr;
  Frag<T> kf[Chunks], vf[Chunks];
#pragma unroll
  for (int c = 0; c < Chunks; c++) {
    kf[c] = global_frag<Wide>(used ? k : nullptr, c, half, p.D);
    vf[c] = global_frag<Wide>(used ? v : nullptr, c, half, p.D);
  }
  const float c = p.scale * kLog2e;
  const int at = kBlock - local + 32 * half, shift = at & 3;
  floatx16 dk[Blocks], dv[Blocks];
#pragma unroll
  for (int d = 0; d < Blocks; d++) dk[d] = dv[d] = (floatx16)(0.f);

  const int64_t go_row = (int64_t)p.Hq * p.D;
  Feed<T, DP, Wide> qt(p.qs[1], p.D, tid), gt(go_row, p.D, tid);
  int bucket = 0;
  float ref = 0.f, log_sum = 0.f, delta = 0.f;
  if (!biased) clear(window, tid);
  for (int g = 0; g < group; g++) {
    const int t0 = tf + max(0, from - g * per_head), t1 = tf + min(per_head, upto - g * per_head);
    if (t0 >= t1) continue;
    const int h = kh * group + g;
    const T *q = (const T *)p.q + b * p.qs[0] + h * p.qs[2];
    const T *go = gout + ((int64_t)b * p.Lq * p.Hq + h) * p.D;
    const int64_t stat = ((int64_t)b * p.Hq + h) * p.Lq;
    // window value x: query - key = (first query of the tile) - (j0 + kBlock) + x, so the bucket's
    // difference is j0 + kBlock - start - first query - x
    const int base = j0 + kBlock - start;
    auto fetch = [&](int t, int buf) {
      const int64_t i = (int64_t)t * kTile;
      qt.start(q + i * p.qs[1], p.qs[1], p.Lq - (int)i, qs[buf], p.D, tid);
      gt.start(go + i * go_row, go_row, p.Lq - (int)i, gs[buf], p.D, tid);
      if (biased) bucket = bucket_of(p, base - (int)i - tid);
      if (tid < kTile) {
        const bool in = i + tid < p.Lq;
        ref = in ? rows.ref[stat + i + tid] : kInf;
        log_sum = in ? rows.log_sum[stat + i + tid] : 0.f;
        delta = in ? rows.delta[stat + i + tid] : 0.f;
      }
    };
    auto put = [&](int buf) {
      qt.finish(qs[buf], tid);
      gt.finish(gs[buf], tid);
      if (biased && tid < kWindow) window[buf].put(tid, bias_of(table, p.NB, bucket));
      if (tid < kTile) {
        row_ref[buf][tid] = ref;
        row_log[buf][tid] = log_sum;
        row_delta[buf][tid] = delta;
      }
    };
    fetch(t0, 0);
    if (biased) load_table<T>(p, h, table, tid, 64 * kWaves);
    loads_done();
    __syncthreads();
    put(0);
    __syncthreads();
    auto tile = [&](int t, auto which) {
      constexpr int buf = decltype(which)::value;
      const int i0 = t * kTile;
      if (t + 1 < t1) fetch(t + 1, buf ^ 1);
      floatx16 u[2], dp[2];
#pragma unroll
      for (int blk = 0; blk < 2; blk++) {
        u[blk] = sixteen(window[buf].get(at + 16 * blk, shift), window[buf].get(at + 16 * blk + 8, shift));
        dp[blk] = (floatx16)(0.f);
        if (i0 < wave_safe || i0 + kTile > p.Lq) {
          const int row0 = i0 + 32 * half + 16 * blk;
          keep_between(u[blk], own_first - row0, p.Lq - row0);
        }
      }
      {
        // (the same pipeline; the rows are queries here)
        const int lane = here(threadIdx.x & 63), half = lane >> 5;
        Frag<T> pf[2][2], sf[2][2];
        auto rows8 = [&](const float *x, int blk, int s) {
          const floatx4 *w = (const floatx4 *)(x + 32 * half + 16 * blk + 8 * s);
          const floatx4 lo = w[0], hi = w[1];
          return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        auto begin = [&](int blk, auto beside) {
          scores<T, DP, Ahead>(qs[buf], gs[buf], blk, lane, kf, vf, u[blk], dp[blk], beside);
          const float delta_row = row_delta[buf][row_of(lane & 31, blk)];
          dp[blk] = add_outer(half ? 0.f : delta_row, 1.f, dp[blk]);
        };
        floatx8 ref8, log8;
        auto gradients = [&](int blk, int n0, int n1) {
#pragma unroll
          for (int n = n0; n < n1; n++) {
            if (n % 8 == 0) ref8 = rows8(row_ref[buf], blk, n / 8), log8 = rows8(row_log[buf], blk, n / 8);
            const float x = exp2_fast(fmaf(u[blk][n] - ref8[n % 8], c, -log8[n % 8]));
            u[blk][n] = x;
            dp[blk][n] *= x;
            if (n % 8 == 7) {
              pf[blk][n / 8] = Frag<T>::pack(eight(u[blk], n / 8));
              sf[blk][n / 8] = Frag<T>::pack(eight(dp[blk], n / 8));
            }
          }
        };
        auto to_keys = [&](int blk, auto beside) {
          Frag<T> fg[2 * Blocks], fq[2 * Blocks];
#pragma unroll
          for (int n = -Ahead; n < 2 * Blocks; n++) {
            if (const int m = n + Ahead; m < 2 * Blocks) {
              fg[m] = Column<T, DP, 32>::get(gs[buf], 16 * blk + 8 * (m / Blocks), m % Blocks, lane);
              fq[m] = Column<T, DP, 32>::get(qs[buf], 16 * blk + 8 * (m / Blocks), m % Blocks, lane);
            }
            if (n < 0) continue;
            dv[n % Blocks] = mma(fg[n], pf[blk][n / Blocks], dv[n % Blocks]);
            dk[n % Blocks] = mma(fq[n], sf[blk][n / Blocks], dk[n % Blocks]);
            beside(n);
            step_end();
          }
        };
        begin(0, [](int) {});
        begin(1, [&](int n) { gradients(0, part_start(n, Chunks), part_start(n + 1, Chunks)); });
        to_keys(0, [&](int n) { gradients(1, part_start(n, 2 * Blocks), part_start(n + 1, 2 * Blocks)); });
        to_keys(1, [](int) {});
      }
      if (t + 1 < t1) put(buf ^ 1);
      __syncthreads();
    };
    for (int t = t0; t < t1; t += 2) {
      tile(t, std::integral_constant<int, 0>{});
      if (t + 1 < t1) tile(t + 1, std::integral_constant<int, 1>{});
    }
  }
  if (!live) return;
  const int64_t row = ((int64_t)b * p.Lk + j) * p.Hk + kh;
  // a key that is not in use has no part in anything
  if (!used) {
#pragma unroll
    for (int d = 0; d < Blocks; d++) dk[d] = dv[d] = (floatx16)(0.f);
  }
  if (parts == 1) {
    if (gk) store_column<Wide, T, Blocks>(gk + row * p.D, dk, p.scale, p.D, half);
    if (gv) store_column<Wide, T, Blocks>(gv + row * p.D, dv, 1.f, p.D, half);
  } else {
    const int64_t at = ((int64_t)part * p.B * p.Lk * p.Hk + row) * p.D;
    if (gk) store_column<Wide, float, Blocks>(gk_parts + at, dk, p.scale, p.D, half);
    if (gv) store_column<Wide, float, Blocks>(gv_parts + at, dv, 1.f, p.D, half);
  }
}

// The sums of up to three gradients' parts, each in order.
struct PartSums {
  const float *parts[3];
  void *to[3];
  int64_t size[3];
  unsigned first[4];  // workgroups before each
  int count[3], n;
  void add(const float *from, void *gradient, int64_t values, int parts_of_it) {
    parts[n] = from, to[n] = gradient, size[n] = values, count[n] = parts_of_it;
    first[n + 1] = first[n] + (unsigned)((values + 255) / 256);
    n++;
  }
};
template <typename T>
__global__ __launch_bounds__(256) void attention_sum_parts_kernel(PartSums sums) {
  int s = 0;
  while (s + 1 < sums.n && blockIdx.x >= sums.first[s + 1]) s++;
  const int64_t size = sums.size[s], i = (int64_t)(blockIdx.x - sums.first[s]) * 256 + threadIdx.x;
  if (i >= size) return;
  const float *parts = sums.parts[s];
  float x = parts[i];
  for (int n = 1; n < sums.count[s]; n++) x += parts[n * size + i];
  ((T *)sums.to[s])[i] = (T)x;
}

// Sums per bucket of a head, in a fixed order.  Of `rows` sums of a head ([B][Hq][nq] with rows =
// B nq, or [Hq][rows] with nq = rows), slice blockIdx.z of gridDim.z takes every gridDim.z-th; a
// workgroup has one head and 64 buckets, its waves every kWaves-th row of the slice.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void attention_table_grad_kernel(const float *partial,
                                                                           T *to, int64_t rows,
                                                                           int Hq, int nq, int NB) {
  __shared__ float part[kWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = blockIdx.y, n = blockIdx.x * 64 + lane;
  float x = 0.f;
  if (n < NB)
#pragma unroll 4
    for (int64_t s = blockIdx.z * kWaves + wave; s < rows; s += kWaves * gridDim.z)
      x += partial[((s / nq * Hq + h) * nq + s % nq) * NB + n];
  part[wave][lane] = x;
  __syncthreads();
  if (wave == 0 && n < NB) {
    for (int w = 1; w < kWaves; w++) x += part[w][lane];
    to[((int64_t)h * gridDim.z + blockIdx.z) * NB + n] = (T)x;
  }
}

constexpr int kSlices = 64;  // of the sums per bucket, where there are many

// How the work is split (`parts_of`): the query gradients' over the keys, the key gradients' over
// the queries and the heads that share them.
struct Plan {
  int64_t nq, nk, q_units, k_units;
  int q_parts, k_parts;
  size_t rows_at, partial_at, slices_at, q_at, k_at, v_at, bytes;  // in the workspace
};

static Plan plan_of(const Params &p) {
  Plan n = {};
  n.nq = (p.Lq + kBlock - 1) / kBlock, n.nk = (p.Lk + kBlock - 1) / kBlock;
  n.q_units = (int64_t)p.B * p.Hq * n.nq, n.k_units = (int64_t)p.B * p.Hk * n.nk;
  const int64_t q_tiles = (p.Lq + kTile - 1) / kTile, k_tiles = (p.Lk + kTile - 1) / kTile;
  n.q_parts = n.q_units ? parts_of(n.q_units, k_tiles) : 1;
  n.k_parts = 1;
  if (n.k_units) {
    n.k_parts = parts_of(n.k_units, q_tiles * (p.Hq / p.Hk));
    // The key kernel mostly has a compute unit's registers for itself: parts of the same length in
    // one round (256 workgroups at most instead of 384 at least, forward and gradients in us: 2562
    // bf16 rows of 4 heads of 128 sharing one 158, 179; 2 x 1000 float32 rows of 8 heads of 32 148,
    // 163).  A causal map's parts differ, and more of them even out (3000 bf16 rows of 8 heads of 128
    // sharing 4 279, 266).
    if (!p.causal) n.k_parts = std::max(1, std::min(n.k_parts, (int)(256 / n.k_units)));
  }
  const size_t rows = (size_t)p.B * p.Hq * p.Lq, keys = (size_t)p.B * p.Hk * p.Lk, f = sizeof(float);
  n.rows_at = align256(rows * f);
  n.partial_at = n.rows_at + 2 * align256(rows * f);
  n.slices_at = n.partial_at + align256((size_t)n.q_units * n.q_parts * p.NB * f);
  n.q_at = n.slices_at + align256((size_t)kSlices * p.Hq * p.NB * f);
  n.k_at = n.q_at + (n.q_parts > 1 ? align256(n.q_parts * rows * p.D * f) : 0);
  n.v_at = n.k_at + (n.k_parts > 1 ? align256(n.k_parts * keys * p.D * f) : 0);
  n.bytes = n.v_at + (n.k_parts > 1 ? align256(n.k_parts * keys * p.D * f) : 0);
  return n;
}

template <typename T>
static int launch_backward(const Params &p, const Plan &n, const void *gout, const void *out,
                           const void *rest, const float *stats, void *gq, void *gk, void *gv, void *gtable, char *ws,
                           hipStream_t stream) {
  const Rows rows = {(float *)ws, (float *)(ws + n.rows_at), (float *)(ws + 2 * n.rows_at)};
  float *partial = (float *)(ws + n.partial_at), *slices = (float *)(ws + n.slices_at);
  float *q_parts = (float *)(ws + n.q_at);
  float *k_parts = (float *)(ws + n.k_at), *v_parts = (float *)(ws + n.v_at);
  const dim3 threads(64 * kWaves);
  PartSums sums = {};
  if (n.q_units) {
    const int parts = gq || gtable ? n.q_parts : 1;
    const size_t lds = (gtable ? 1 + kWaves : 1) * p.NB * sizeof(float);
    const int rc = launch_in_pieces(p, n.q_units * parts, [&](const Params &piece, dim3 grid) {
#define MCX_GRAD(DP, W)                                                                           \
  hipLaunchKernelGGL((gtable ? attention_query_grad_kernel<T, DP, W, true>                        \
                             : attention_query_grad_kernel<T, DP, W, false>), grid, threads, lds, \
                     stream, piece,                                                               \
                     (const T *)out, (const T *)rest, (const T *)gout, stats, rows, (T *)gq,       \
                     q_parts,                                                                     \
                     gtable ? partial : nullptr, (int)n.nq, parts)
      MCX_ATTENTION_DISPATCH(p.D, p.wide && aligned16(out) && aligned16(rest) && aligned16(gout) && aligned16(gq),
                             MCX_GRAD);
#undef MCX_GRAD
    });
    if (rc != MCX_OK) return rc;
    if (gq && parts > 1) sums.add(q_parts, gq, (int64_t)p.B * p.Lq * p.Hq * p.D, parts);
  }
  if (gtable) {
    const int64_t count = (int64_t)p.B * n.nq * n.q_parts;
    const int nq = std::max(1, (int)n.nq * n.q_parts), wide = (p.NB + 63) / 64;
    if (count <= 2 * kSlices) {
      hipLaunchKernelGGL((attention_table_grad_kernel<T>), dim3(wide, p.Hq), threads, 0, stream,
                         partial, (T *)gtable, count, p.Hq, nq, p.NB);
    } else {
      hipLaunchKernelGGL((attention_table_grad_kernel<float>), dim3(wide, p.Hq, kSlices), threads, 0,
                         stream, partial, slices, count, p.Hq, nq, p.NB);
      hipLaunchKernelGGL((attention_table_grad_kernel<T>), dim3(wide, p.Hq), threads, 0, stream,
                         slices, (T *)gtable, (int64_t)kSlices, p.Hq, kSlices, p.NB);
    }
    MCX_HIP_CHECK_LAUNCH();
  }
  if ((gk || gv) && n.k_units) {
    const size_t lds = p.NB * sizeof(float);
    const int rc = launch_in_pieces(p, n.k_units * n.k_parts, [&](const Params &piece, dim3 grid) {
#define MCX_GRAD(DP, W)                                                                         \
  hipLaunchKernelGGL((attention_key_grad_kernel<T, DP, W>), grid, threads, lds, stream, piece,   \
                     (const T *)gout, rows, (T *)gk, (T *)gv, k_parts, v_parts,                   \
                     (int)n.nk, n.k_parts)
      MCX_ATTENTION_DISPATCH(p.D, p.wide && aligned16(gout) && aligned16(gk) && aligned16(gv), MCX_GRAD);
#undef MCX_GRAD
    });
    if (rc != MCX_OK) return rc;
    if (n.k_parts > 1) {
      const int64_t size = (int64_t)p.B * p.Lk * p.Hk * p.D;
      if (gk) sums.add(k_parts, gk, size, n.k_parts);
      if (gv) sums.add(v_parts, gv, size, n.k_parts);
    }
  }
  if (sums.n) {
    hipLaunchKernelGGL((attention_sum_parts_kernel<T>), dim3(sums.first[sums.n]), dim3(256), 0, stream,
                       sums);
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
  return plan_of(p).bytes;
}

int mcx_attention_backward(const void *gout, const void *q, const void *k, const void *v,
                           const void *out, const void *out_rest, const float *stats,
                           const void *table, const int32_t *buckets, const int32_t *query_start,
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
  const Plan n = plan_of(p);
  if (n.q_units > 0x7fffffffLL || n.k_units > 0x7fffffffLL) return MCX_E_SHAPE;
  if (n.bytes && (!workspace || workspace_bytes < n.bytes)) return MCX_E_WORKSPACE;
  return dtype == MCX_BF16
             ? launch_backward<__bf16>(p, n, gout, out, out_rest, stats, gq, gk, gv, gtable, (char *)workspace,
                                       (hipStream_t)stream)
             : launch_backward<float>(p, n, gout, out, nullptr, stats, gq, gk, gv, gtable, (char *)workspace,
                                      (hipStream_t)stream);
}

}  // extern "C"
