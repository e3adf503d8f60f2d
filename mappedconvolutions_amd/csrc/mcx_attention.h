// What the attention kernels share: operand fragments of the 32x32 matrix instructions for both
// data types, tiles that travel from memory through registers into LDS, and the window of bias
// values that belongs to a tile of pairs.
//
//   u_ij = q_i . k_j + T[h, bucket(j - pos_i)] / scale,   p_ij = softmax_j(scale * u_ij)
//
// The bias is divided by the scale so that it can be the matrix product's starting value: adding
// it then costs no vector instruction, and the scale goes into the exponent's factor.
//
// Orientation.  The product's result has one column per lane (lane & 31) and, in its 16 values,
// rows 8 g + 4 (lane >> 5) + a (value 4 g + a).  Keys are the rows and queries the columns (the
// other way round where the gradients of keys are formed), so that a softmax row lies in one lane
// and its other half-wave partner.  The rows are loaded in the order `row_of`, which makes values
// 8 c .. 8 c + 7 of a lane belong to rows 16 c + 8 (lane >> 5) + 0 .. 7: exactly what the next
// product wants as its operand, so probabilities never leave their lane.
#pragma once

#include "mcx_mfma_common.h"

namespace mcx {
namespace attention {

constexpr int kWaves = 4;          // of a workgroup
constexpr int kLanesRows = 32;     // columns (queries, or keys) of a wave
constexpr int kBlock = kWaves * kLanesRows;  // columns of a workgroup
constexpr int kTile = 64;          // rows walked at a time
constexpr int kMaxD = 128;
constexpr int kMaxTable = 512;     // buckets of a head: their values and sums stay in LDS
// A finite bias is held within this: its sum with a score then swallows the score, as the
// lowest value of the type does, and neither the scale nor log2(e) takes it to infinity.
constexpr float kBiasLimit = 1e30f;
// Where a row's statistic is beyond this, one fma no longer holds the difference in the exponent.
constexpr float kHugeStat = 1e9f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

struct Params {
  const void *q, *k, *v;
  const void *table;      // [Hq, NB] or null
  const int *buckets;     // [R]
  const int *start;       // [B] or null: position of the first query
  const int *lengths;     // [B] or null: keys in use
  int64_t qs[3], ks[3], vs[3];  // strides of batch, token, head (values)
  int B, Lq, Lk, Hq, Hk, D;
  int R, zero, NB, causal;
  float scale;
  int q_wide, k_wide, v_wide;  // 16-byte loads are in place
};

__device__ inline int first_position(const Params &p, int b) {
  if (!p.start) return 0;
  return min(max(p.start[b], -(1 << 30)), 1 << 30);
}
__device__ inline int key_length(const Params &p, int b) {
  if (!p.lengths) return p.Lk;
  return min(max(p.lengths[b], 0), p.Lk);
}

// Row of the operand that the result's row m has to stand for (see above): bits 2 and 3 swapped.
__device__ inline int row_of(int m) { return (m & 0x13) | ((m & 4) << 1) | ((m & 8) >> 1); }

__device__ inline float to_float(float v) { return v; }
__device__ inline float to_float(__bf16 v) { return (float)v; }

// ---- operands of a 32 x 32 x 16 product --------------------------------------------------
// A fragment holds, of the 16 values of the summed axis, values 8 (lane >> 5) + 0 .. 7.
template <typename T> struct Frag;

template <> struct Frag<__bf16> {
  bf16x8 v;
  static __device__ inline Frag pack(const floatx8 &x) {
    return {__builtin_convertvector(x, bf16x8)};
  }
};
template <> struct Frag<float> {
  floatx8 v;
  static __device__ inline Frag pack(const floatx8 &x) { return {x}; }
};

__device__ inline floatx16 mma(const Frag<__bf16> &a, const Frag<__bf16> &b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
// Eight products of two values each: value e of the lower and of the upper half-wave.
__device__ inline floatx16 mma(const Frag<float> &a, const Frag<float> &b, floatx16 c) {
#pragma unroll
  for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
  return c;
}

// Values of a row of an LDS tile: 16 bytes more than the row, so that rows start in other banks.
template <typename T, int DP> constexpr int pitch() { return DP + 16 / (int)sizeof(T); }

// Operand whose summed axis runs along the rows of a tile: row `row`, values 16 chunk + ...
template <typename T, int DP>
__device__ inline Frag<T> row_frag(const T *tile, int row, int chunk, int half) {
  const uint4 *at = (const uint4 *)(tile + row * pitch<T, DP>() + 16 * chunk + 8 * half);
  struct { uint4 w[sizeof(T) / 2]; } f;
#pragma unroll
  for (int n = 0; n < (int)sizeof(T) / 2; n++) f.w[n] = at[n];
  return __builtin_bit_cast(Frag<T>, f);
}

// Operand whose summed axis runs down the rows: column 32 block + (lane & 31), rows r0 + ...
template <int DP>
__device__ inline Frag<float> col_frag(const float *tile, int r0, int block, int lane) {
  const float *at = tile + (r0 + 8 * (lane >> 5)) * pitch<float, DP>() + 32 * block + (lane & 31);
  Frag<float> f;
#pragma unroll
  for (int e = 0; e < 8; e++) f.v[e] = at[e * pitch<float, DP>()];
  return f;
}
// (the transposing load: of 16 lanes, four address a row's 16 values and lane c gets column c of
// the four rows)
template <int DP>
__device__ inline Frag<__bf16> col_frag(const __bf16 *tile, int r0, int block, int lane) {
  const __bf16 *at = tile + (r0 + 8 * (lane >> 5) + ((lane & 15) >> 2)) * pitch<__bf16, DP>() +
                     32 * block + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  typedef __attribute__((address_space(3))) shortx4 *lds4;
  struct { shortx4 lo, hi; } f;
  f.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
  f.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 4 * pitch<__bf16, DP>()));
  return __builtin_bit_cast(Frag<__bf16>, f);
}

// 16 bytes of a row: values d0 .. of `row`, zeros behind the row's end.
template <typename T>
__device__ inline uint4 load16(const T *row, int d0, int D, bool wide) {
  constexpr int E = 16 / (int)sizeof(T);
  if (wide) return d0 < D ? *(const uint4 *)(row + d0) : make_uint4(0, 0, 0, 0);
  T x[E];
#pragma unroll
  for (int e = 0; e < E; e++) x[e] = d0 + e < D ? row[d0 + e] : (T)0.f;
  return __builtin_bit_cast(uint4, *(const __attribute__((ext_vector_type(E))) T *)x);
}

// Column operand straight from memory: row `row` (null: zeros) of this lane, values 16 chunk + ...
template <typename T>
__device__ inline Frag<T> global_frag(const T *row, int chunk, int half, int D, bool wide) {
  constexpr int E = 16 / (int)sizeof(T), N = 8 / E;
  struct { uint4 w[N]; } f;
#pragma unroll
  for (int n = 0; n < N; n++)
    f.w[n] = row ? load16(row, 16 * chunk + 8 * half + n * E, D, wide) : make_uint4(0, 0, 0, 0);
  return __builtin_bit_cast(Frag<T>, f);
}

// kTile rows of a matrix on their way from memory to LDS, in the registers of a workgroup.
template <typename T, int DP> struct Tile {
  static constexpr int E = 16 / (int)sizeof(T), PerRow = DP / E;
  static constexpr int N = kTile * PerRow / (64 * kWaves);
  uint4 r[N];
  // rows [0, rows) of `base`; the others are zeros
  __device__ inline void load(const T *base, int64_t stride, int rows, int D, bool wide, int tid) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int id = tid + n * 64 * kWaves, row = id / PerRow, d0 = (id % PerRow) * E;
      r[n] = row < rows ? load16(base + row * stride, d0, D, wide) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ inline void store(T *tile, int tid) const {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int id = tid + n * 64 * kWaves, row = id / PerRow, d0 = (id % PerRow) * E;
      *(uint4 *)(tile + row * pitch<T, DP>() + d0) = r[n];
    }
  }
};

// ---- the bias of a tile of pairs -----------------------------------------------------------
// A tile of kTile rows and kBlock columns has kTile + kBlock - 1 differences.  A lane wants eight
// consecutive ones from any place on: four copies, each shifted by one value, let it read them as
// two aligned 16-byte words.  The copies lie 16 banks apart, which keeps the four lanes of one
// word's neighbourhood out of each other's banks.
constexpr int kWindow = kTile + kBlock;  // 192 (the last one unused)
constexpr int kCopy = 208;
struct Window {
  float copy[4][kCopy];
  __device__ inline void put(int t, float x) {
#pragma unroll
    for (int s = 0; s < 4; s++)
      if (t >= s) copy[s][t - s] = x;
  }
  // differences at .. at + 7, `shift` = at & 3
  __device__ inline floatx8 get(int at, int shift) const {
    const floatx4 *w = (const floatx4 *)&copy[shift][at - shift];
    const floatx4 a = w[0], b = w[1];
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

__device__ inline int bucket_of(const Params &p, int difference) {
  const int64_t at = (int64_t)difference + p.zero;
  return p.buckets[at < 0 ? 0 : at >= p.R ? p.R - 1 : (int)at];
}
// A bucket outside the table has no bias and no gradient.
__device__ inline float bias_of(const float *table, int NB, int bucket) {
  return (unsigned)bucket < (unsigned)NB ? table[bucket] : 0.f;
}
// A head's table over the scale, in LDS.
template <typename T>
__device__ inline void load_table(const Params &p, int head, float *table, int tid, int threads) {
  const T *t = (const T *)p.table + (int64_t)head * p.NB;
  for (int n = tid; n < p.NB; n += threads) {
    float x = to_float(t[n]);
    if (fabsf(x) < kInf) x = fminf(fmaxf(x, -kBiasLimit), kBiasLimit);
    table[n] = x / p.scale;
  }
}

// The other half-wave's value of the same column.
__device__ inline float other_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A lane's column of a transposed result ([DP] values in blocks of 32) to a row of memory.
template <typename T, int NBlocks>
__device__ inline void store_column(T *row, const floatx16 *acc, float factor, int D, int half,
                                    bool wide) {
#pragma unroll
  for (int blk = 0; blk < NBlocks; blk++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int d0 = 32 * blk + 8 * g + 4 * half;
      typedef __attribute__((ext_vector_type(4))) T T4;
      floatx4 x = {acc[blk][4 * g] * factor, acc[blk][4 * g + 1] * factor,
                   acc[blk][4 * g + 2] * factor, acc[blk][4 * g + 3] * factor};
      const T4 y = __builtin_convertvector(x, T4);
      if (wide) {
        if (d0 < D) *(T4 *)(row + d0) = y;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (d0 + e < D) row[d0 + e] = y[e];
      }
    }
}

// Checks the arguments of an entry point and fills in `p`: MCX_OK, or what is wrong with them.
int make_params(Params &p, const void *q, const void *k, const void *v, const void *table,
                const int32_t *buckets, const int32_t *query_start, const int32_t *key_lengths,
                const mcx_attention_desc *desc, int dtype);

// The form for few queries against many keys (mcx_attention_split.hip): over how many parts of the
// keys (0: not the form for these sizes), its workspace, and its launch.
int split_parts(const Params &p);
size_t split_bytes(const Params &p, int parts);
int launch_split(const Params &p, int parts, void *out, float *stats, void *workspace, int dtype,
                 hipStream_t stream);

}  // namespace attention
}  // namespace mcx
