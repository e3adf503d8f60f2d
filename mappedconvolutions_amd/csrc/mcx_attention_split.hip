// Attention of few queries over many keys: the keys are split over workgroups and the parts joined.
//
// Bound by memory: one token reads the whole cache once.  The query heads that share a key head
// are rows of one product (row r = query r / group, head r % group), 32 to a workgroup, so their
// keys are read once for all.  A wave takes every fourth 32 keys of its workgroup's part: the keys
// come straight into the product's operand registers, the values through LDS that only this wave
// uses, the next tile's loads under way meanwhile; there is no barrier in the loop.
//   64 bf16 tokens over up to 8192 keys of 8 heads of 128 (1.6 GB): 304 us and 7 for the join,
// 5.2 TB/s; two float32 tokens over 100001 keys of 2 heads of 64 (205 MB): 48 us and 5, 3.9 TB/s.  A
// large copy reaches 4.9 TB/s.
#include <algorithm>

#include "mcx_attention.h"

namespace mcx {
namespace attention {

constexpr int kRows = 32;       // rows of a workgroup
constexpr int kStep = 32;       // keys of a wave's tile
constexpr int kMostParts = 256;

// As `row_of`, for 32 rows: a lane gets rows 16 c + 8 (lane >> 5) + 0 .. 7 (bits 2 and 3 swapped).
__device__ inline int row_of_32(int m) { return (m & 0x13) | ((m & 4) << 1) | ((m & 8) >> 1); }

struct Split {
  int parts;       // of the keys
  int blocks;      // of 32 rows, of a key head
  int rows;        // Lq * group
  float *sums;     // [B * Hk * blocks][parts][32][2]: reference and sum
  float *outs;     // [B * Hk * blocks][parts][32][D]
};

template <typename T, int DP, bool Wide>
__global__ __launch_bounds__(64 * kWaves, (waves_per_simd<T, DP>(3))) void attention_split_kernel(
    Params p, Split sp, T *out, float *stats, T *rest) {
  constexpr int Chunks = DP / 16, Blocks = DP / 32;
  constexpr int E = 16 / (int)sizeof(T), PerRow = words<T, DP>(), N = kStep * PerRow / 64;
  // a wave's values; at the end all waves' sums, half a block of columns at a time
  constexpr int kTileWords = kStep * PerRow;
  __shared__ Word tiles_lds[kWaves * kTileWords];
  __shared__ int buckets_lds[kWaves][64];
  __shared__ float merge[kWaves][kRows][2];
  extern __shared__ float table[];  // [min(group, 32)][NB]

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int wg = xcd_contiguous_tile(blockIdx.x, gridDim.x);
  const int part = wg % sp.parts, unit = wg / sp.parts;
  const int block = unit % sp.blocks, bk = unit / sp.blocks, b = bk / p.Hk, kh = bk % p.Hk;
  const int group = p.Hq / p.Hk;
  const int r = block * kRows + (lane & 31);
  const bool live = r < sp.rows;
  const int i = r / group, h = kh * group + r % group;
  const int start = first_position(p, b), length = key_length(p, b);
  const int limit = !live ? 0 : p.causal ? min(length, start + i + 1) : length;
  const int first_i = block * kRows / group;
  const int last_i = min(block * kRows + kRows - 1, sp.rows - 1) / group;
  const int keys = p.causal ? max(0, min(length, start + last_i + 1)) : length;
  const int wave_limit = p.causal ? min(length, start + first_i + 1) : length;

  const bool biased = p.table != nullptr;
  const int slots = min(group, kRows), slot = group <= kRows ? r % group : lane & 31;
  if (biased) {
    for (int n = tid; n < slots * p.NB; n += 64 * kWaves) {
      const int s = n / p.NB, hs = kh * group + (group <= kRows ? s : (block * kRows + s) % group);
      float x = to_float(((const T *)p.table)[(int64_t)hs * p.NB + n % p.NB]);
      if (fabsf(x) < kInf) x = fminf(fmaxf(x, -kBiasLimit), kBiasLimit);
      table[n] = x / p.scale;
    }
  }
  __syncthreads();

  const int total = (keys + kStep - 1) / kStep, each = (total + sp.parts - 1) / sp.parts;
  const int t_end = min(total, (part + 1) * each);
  int t = part * each + wave;

  const T *k = (const T *)p.k + b * p.ks[0] + kh * p.ks[2];
  const T *v = (const T *)p.v + b * p.vs[0] + kh * p.vs[2];
  const T *q = (const T *)p.q + b * p.qs[0] + (int64_t)i * p.qs[1] + h * p.qs[2];
  Frag<T> qf[Chunks], kf[Chunks];
  Word vr[N];
#pragma unroll
  for (int c = 0; c < Chunks; c++) qf[c] = global_frag<Wide>(live ? q : nullptr, c, half, p.D);

  const int key_row = row_of_32(lane & 31);
  // bias: difference x of a tile = j - (position of the block's last query)
  const int origin = start + last_i, own = live ? last_i - i : 0;
  int bucket = 0;
  bool varied = false;  // whether the tile's pairs are of more than one bucket
  // (a key behind the last one is the last one: its pairs are taken out below)
  auto fetch_keys = [&](int tile) {
    const T *row = k + (int64_t)min(tile * kStep + key_row, keys - 1) * p.ks[1];
#pragma unroll
    for (int c = 0; c < Chunks; c++) kf[c] = global_frag<Wide>(row, c, half, p.D);
  };
  auto fetch_values = [&](int tile) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int id = lane + 64 * n, j = min(tile * kStep + id / PerRow, keys - 1);
      const int d0 = (id % PerRow) * E;
      const T *vrow = v + (int64_t)j * p.vs[1];
      vr[n] = Wide ? *(const Word *)(vrow + (d0 < p.D ? d0 : 0)) : load16<false>(vrow, d0, p.D);
    }
    if (biased) bucket = bucket_of(p, tile * kStep - origin + lane);
  };
  const float c = p.scale * kLog2e;
  Word *vs = tiles_lds + wave * kTileWords;
  floatx16 o[Blocks];
#pragma unroll
  for (int d = 0; d < Blocks; d++) o[d] = (floatx16)(0.f);
  float ref = -kInf, sum = 0.f;
  if (t < t_end) {
    fetch_keys(t);
    fetch_values(t);
  }
  for (; t < t_end; t += kWaves) {
    const int j0 = t * kStep;
    wave_order();
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int id = lane + 64 * n;
      vs[word_at<T, DP>(id / PerRow, id % PerRow)] = vr[n];
    }
    buckets_lds[wave][lane] = bucket;
    wave_order();
    floatx16 u = (floatx16)(0.f);
    if (biased) {
      const int one = __builtin_amdgcn_readfirstlane(bucket);
      varied = __any(bucket != one);
      if (varied) {
#pragma unroll
        for (int n = 0; n < 16; n++) {
          const int x = buckets_lds[wave][16 * (n >> 3) + 8 * half + (n & 7) + own];
          u[n] = (unsigned)x < (unsigned)p.NB ? table[slot * p.NB + x] : 0.f;
        }
      } else {
        u = (floatx16)((unsigned)one < (unsigned)p.NB ? table[slot * p.NB + one] : 0.f);
      }
    }
    if (t + kWaves < t_end) fetch_values(t + kWaves);
#pragma unroll
    for (int n = 0; n < Chunks; n++) u = mma(kf[n], qf[n], u);
    if (t + kWaves < t_end) fetch_keys(t + kWaves);
    if (j0 + kStep > wave_limit) {
#pragma unroll
      for (int n = 0; n < 16; n++)
        if (j0 + 16 * (n >> 3) + 8 * half + (n & 7) >= limit) u[n] = -kInf;
    }
    float top = u[0];
#pragma unroll
    for (int n = 1; n < 16; n++) top = fmaxf(top, u[n]);
    top = fmaxf(top, other_half(top));
    if (__any((top - ref) * c > 8.f)) {
      const float next = fmaxf(ref, top);
      const float keep = next == -kInf ? 1.f : exp2_fast((ref - next) * c);
      ref = next;
      sum *= keep;
#pragma unroll
      for (int d = 0; d < Blocks; d++) o[d] *= keep;
    }
    const float used = ref == -kInf ? 0.f : ref;
#pragma unroll
    for (int n = 0; n < 16; n++) {
      u[n] = exp2_fast((u[n] - used) * c);
      sum += u[n];
    }
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const Frag<T> pf = Frag<T>::pack(eight(u, s));
#pragma unroll
      for (int d = 0; d < Blocks; d++) o[d] = mma(Column<T, DP, 8>::get(vs, 16 * s, d, lane), pf, o[d]);
    }
  }
  sum += other_half(sum);

  // the four waves' parts: a common reference, then block by block of columns through LDS
  if (half == 0) {
    merge[wave][lane][0] = ref;
    merge[wave][lane][1] = sum;
  }
  __syncthreads();
  float top = -kInf;
#pragma unroll
  for (int w = 0; w < kWaves; w++) top = fmaxf(top, merge[w][lane & 31][0]);
  float all = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    const float x = merge[w][lane & 31][0];
    all += x == -kInf ? merge[w][lane & 31][1] : merge[w][lane & 31][1] * exp2_fast((x - top) * c);
  }
  const float factor = ref == -kInf ? 1.f : exp2_fast((ref - top) * c);
  // 16 columns at a time: [wave][16 columns][32 rows], of which a thread sums two columns of a row
  float *part_lds = (float *)tiles_lds;
  static_assert(kTileWords * 16 >= 32 * 16 * 4, "a block's sums fit two halves");
  const int64_t at = (int64_t)unit * sp.parts + part;
#pragma unroll
  for (int d = 0; d < Blocks; d++)
#pragma unroll
    for (int hh = 0; hh < 2; hh++) {  // 16 of the 32 columns at a time
      __syncthreads();
#pragma unroll
      for (int g = 0; g < 2; g++)
#pragma unroll
        for (int a = 0; a < 4; a++)
          part_lds[(wave * 16 + 8 * g + 4 * half + a) * 32 + (lane & 31)] =
              o[d][8 * hh + 4 * g + a] * factor;
      __syncthreads();
      // 256 threads, 16 columns x 32 rows: two columns each
#pragma unroll
      for (int n = 0; n < 2; n++) {
        const int column = 2 * (tid >> 5) + n, row = tid & 31, rr = block * kRows + row;
        const int dd = 32 * d + 16 * hh + column;
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) x += part_lds[(w * 16 + column) * 32 + row];
        if (rr < sp.rows && dd < p.D) {
          if (sp.parts == 1) {
            // (lane & 31 is this thread's row too, so `all` is its row's sum)
            const int64_t to = ((int64_t)b * p.Lq + rr / group) * p.Hq + kh * group + rr % group;
            store_value(out, rest, to * p.D + dd, all == 0.f ? 0.f : x / all);
          } else {
            sp.outs[(at * kRows + row) * p.D + dd] = x;
          }
        }
      }
    }
  if (wave == 0 && half == 0 && live) {
    if (sp.parts > 1) {
      sp.sums[(at * kRows + lane) * 2] = top;
      sp.sums[(at * kRows + lane) * 2 + 1] = all;
    } else if (stats) {
      float *s = stats + 2 * (((int64_t)b * p.Hq + h) * p.Lq + i);
      s[0] = top;
      s[1] = all;
    }
  }
}

// Joins the parts of a row: a workgroup has one row, its waves every kJoinWaves-th part.  What it
// costs is the time of its loads from the first to the last, so they are many at once.
constexpr int kJoinWaves = 16;
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void attention_join_kernel(Params p, Split sp, T *out,
                                                                         float *stats, T *rest) {
  __shared__ float merge[kJoinWaves][kMaxD];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = p.Hq / p.Hk;
  const int bk = blockIdx.x / sp.rows, r = blockIdx.x % sp.rows, b = bk / p.Hk, kh = bk % p.Hk;
  const int unit = bk * sp.blocks + r / kRows, row = r % kRows;
  const float *sums = sp.sums + ((int64_t)unit * sp.parts * kRows + row) * 2;
  const float *from = sp.outs + ((int64_t)unit * sp.parts * kRows + row) * p.D;
  const float c = p.scale * kLog2e;
  // the wave's parts, eight at a time, are on their way while it finds the common reference
  float ref[kMostParts / 64], part_sum[kMostParts / 64], top = -kInf, all = 0.f;
#pragma unroll
  for (int n = 0; n < kMostParts / 64; n++) {
    const int s = lane + 64 * n;
    ref[n] = s < sp.parts ? sums[(int64_t)s * kRows * 2] : -kInf;
    part_sum[n] = s < sp.parts ? sums[(int64_t)s * kRows * 2 + 1] : 0.f;
  }
#pragma unroll
  for (int n = 0; n < kMostParts / 64; n++) top = fmaxf(top, ref[n]);
  for (int m = 32; m; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
#pragma unroll
  for (int n = 0; n < kMostParts / 64; n++) {
    ref[n] = ref[n] == -kInf ? 1.f : exp2_fast((ref[n] - top) * c);  // (a NaN part stays one)
    all = fmaf(ref[n], part_sum[n], all);
  }
  for (int m = 32; m; m >>= 1) all += __shfl_xor(all, m);
  float x = 0.f, y = 0.f;
#pragma unroll
  for (int n = 0; n < kMostParts / 64; n++)
#pragma unroll
    for (int q = 0; q < 64 / kJoinWaves; q++) {
      const int s = 64 * n + q * kJoinWaves + wave;
      if (s < sp.parts) {
        const float w = __shfl(ref[n], q * kJoinWaves + wave);
        const float *f = from + (int64_t)s * kRows * p.D;
        if (lane < p.D) x = fmaf(w, f[lane], x);
        if (lane + 64 < p.D) y = fmaf(w, f[lane + 64], y);
      }
    }
  merge[wave][lane] = x;
  merge[wave][lane + 64] = y;
  __syncthreads();
  const int h = kh * group + r % group, i = r / group;
  if (tid < p.D) {
    x = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWaves; w++) x += merge[w][tid];
    store_value(out, rest, (((int64_t)b * p.Lq + i) * p.Hq + h) * p.D + tid, all == 0.f ? 0.f : x / all);
  }
  if (stats && tid == 0) {
    float *s = stats + 2 * (((int64_t)b * p.Hq + h) * p.Lq + i);
    s[0] = top;
    s[1] = all;
  }
}

// The same for a few parts of many rows: a thread has one value of the output.
constexpr int kFewParts = 16;
template <typename T>
__global__ __launch_bounds__(256) void attention_join_few_kernel(Params p, Split sp, T *out,
                                                                 float *stats, T *rest,
                                                                 int64_t total) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;  // [bk][row][value]
  if (n >= total) return;
  const int64_t br = n / p.D;
  const int d = (int)(n - br * p.D);
  const int bk = (int)(br / sp.rows), r = (int)(br - (int64_t)bk * sp.rows);
  const int group = p.Hq / p.Hk, b = bk / p.Hk, kh = bk % p.Hk;
  const int64_t first = ((int64_t)bk * sp.blocks + r / kRows) * sp.parts * kRows + r % kRows;
  const float c = p.scale * kLog2e;
  float top = -kInf, all = 0.f, x = 0.f;
  for (int s = 0; s < sp.parts; s++) top = fmaxf(top, sp.sums[(first + s * kRows) * 2]);
  for (int s = 0; s < sp.parts; s++) {
    const float ref = sp.sums[(first + s * kRows) * 2];
    const float w = ref == -kInf ? 1.f : exp2_fast((ref - top) * c);  // (a NaN part stays one)
    all = fmaf(w, sp.sums[(first + s * kRows) * 2 + 1], all);
    x = fmaf(w, sp.outs[(first + s * kRows) * p.D + d], x);
  }
  const int64_t i = r / group, h = kh * group + r % group;
  store_value(out, rest, ((b * (int64_t)p.Lq + i) * p.Hq + h) * p.D + d, all == 0.f ? 0.f : x / all);
  if (stats && d == 0) {
    float *s = stats + 2 * (((int64_t)b * p.Hq + h) * p.Lq + i);
    s[0] = top;
    s[1] = all;
  }
}

// 0: the other kernel is the better one.  Both work on blocks of 32 rows; this one shares a key's
// loads among the heads of a group but not among blocks, and fills its blocks with a group's heads
// where the other one leaves waves of a head's 128 without queries.  Its block of keys costs up to
// three times the other's in bf16, where the other one reaches half the matrix rate, and 1.5 times
// in fp32 (this, other, in us): 16 x 32 queries, 2000 keys, 32 heads sharing 8 of 64: bf16 31, 49,
// fp32 96, 275; 16 x 64 queries of 32 heads of 128 sharing 8: bf16 88, 74, fp32 382, 566; 128 x 100
// queries and keys, 8 heads of 64: bf16 54, 18, fp32 90, 50.
int split_parts(const Params &p, int dtype) {
  const int64_t group = p.Hq / p.Hk, rows = p.Lq * group;
  const int64_t blocks = (rows + kRows - 1) / kRows, units = (int64_t)p.B * p.Hk * blocks;
  const int64_t here = p.Hk * blocks * ((p.Lk + kWaves * kStep - 1) / (kWaves * kStep)) * (kWaves * kStep);
  const int64_t there = (int64_t)p.Hq * ((p.Lq + kBlock - 1) / kBlock) * kWaves *
                        ((p.Lk + kTile - 1) / kTile) * kTile;
  if ((dtype == MCX_BF16 ? 6 : 3) * here > 2 * there) return 0;
  if (units >= (1 << 24)) return 0;  // (more threads than a launch has)
  // One workgroup for every compute unit where there are fewer units of work: more parts cost more
  // in their ends and in the join than they win (one bf16 token over 20000 keys of 8 heads of 128:
  // 23.0, 25.8, 33.5 us with 256, 512, 1024 workgroups in all).  Where there are enough, parts of at
  // least 2048 keys even out the last round (64 bf16 tokens over up to 8192 keys of 8 heads: 368,
  // 338, 319 us with one, two, four parts).
  const int64_t tiles = (p.Lk + kWaves * kStep - 1) / (kWaves * kStep);
  // A short cache takes less time in one part than the join's launch (one token, 8 heads, a call
  // through the binding, one part and split, in us): bf16, 1000 keys of 64 14.3, 18.9; 500 of 128
  // 15.3, 18.9; 1000 of 128 19.6, 19.1; 2000 of 64 21.0, 18.9; fp32, 256 of 64 14.1, 18.7; 500 of 64
  // 19.1, 18.8; 1000 of 64 30.0, 18.9.
  if ((int64_t)p.Lk * p.D <= (dtype == MCX_BF16 ? 64 << 10 : 16 << 10)) return 1;
  const int64_t parts = units < 256 ? std::min<int64_t>((256 + units - 1) / units, tiles)
                                    : std::min<int64_t>((2048 + units - 1) / units, p.Lk / 2048);
  return (int)std::max<int64_t>(1, std::min<int64_t>(parts, kMostParts));
}

static Split split_of(const Params &p, int parts) {
  Split sp = {};
  sp.parts = parts;
  sp.rows = p.Lq * (p.Hq / p.Hk);
  sp.blocks = (sp.rows + kRows - 1) / kRows;
  return sp;
}

size_t split_bytes(const Params &p, int parts) {
  if (parts <= 1) return 0;
  const Split sp = split_of(p, parts);
  const size_t rows = (size_t)p.B * p.Hk * sp.blocks * parts * kRows;
  return align256(rows * 2 * sizeof(float)) + align256(rows * p.D * sizeof(float));
}

template <typename T>
static int launch(const Params &p, Split sp, void *out, float *stats, void *rest,
                  hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)p.B * p.Hk * sp.blocks * sp.parts)), threads(64 * kWaves);
  const size_t lds = p.table ? std::min(p.Hq / p.Hk, kRows) * p.NB * sizeof(float) : 0;
#define MCX_SPLIT(DP, W)                                                                           \
  hipLaunchKernelGGL((attention_split_kernel<T, DP, W>), grid, threads, lds, stream, p, sp, (T *)out, \
                     stats, (T *)rest)
  MCX_ATTENTION_DISPATCH(p.D, p.wide, MCX_SPLIT);
#undef MCX_SPLIT
  MCX_HIP_CHECK_LAUNCH();
  const int64_t rows = (int64_t)p.B * p.Hk * sp.rows, total = rows * p.D;
  if (sp.parts > kFewParts) {
    hipLaunchKernelGGL((attention_join_kernel<T>), dim3((unsigned)rows), dim3(64 * kJoinWaves), 0,
                       stream, p, sp, (T *)out, stats, (T *)rest);
  } else if (sp.parts > 1) {
    hipLaunchKernelGGL((attention_join_few_kernel<T>), dim3((unsigned)((total + 255) / 256)),
                       dim3(256), 0, stream, p, sp, (T *)out, stats, (T *)rest, total);
  }
  MCX_HIP_CHECK_LAUNCH();
  return MCX_OK;
}

int launch_split(const Params &p, int parts, void *out, float *stats, void *rest, void *workspace,
                 int dtype, hipStream_t stream) {
  Split sp = split_of(p, parts);
  if (parts > 1) {
    const size_t rows = (size_t)p.B * p.Hk * sp.blocks * parts * kRows;
    sp.sums = (float *)workspace;
    sp.outs = (float *)((char *)workspace + align256(rows * 2 * sizeof(float)));
  }
  return dtype == MCX_BF16 ? launch<__bf16>(p, sp, out, stats, rest, stream)
                           : launch<float>(p, sp, out, stats, nullptr, stream);
}

}  // namespace attention
}  // namespace mcx
