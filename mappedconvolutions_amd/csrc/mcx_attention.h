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
// and its other half-wave partner.  The next product sums over what are rows here, and wants eight
// consecutive values of that axis in a lane: which rows they stand for is free as long as both its
// operands agree.  The rows are loaded in the order `row_of`, which gives a lane the consecutive
// rows 32 (lane >> 5) + 0 .. 31 of a tile of 64, in the values' own order: probabilities never leave
// their lane, and neighbouring lanes hold neighbouring diagonals.
#pragma once

#include <algorithm>

#include "mcx_mfma_common.h"

namespace mcx {
namespace attention {

constexpr int kWaves = 4;          // of a workgroup
constexpr int kLanesRows = 32;     // columns (queries, or keys) of a wave
constexpr int kBlock = kWaves * kLanesRows;  // columns of a workgroup
constexpr int kTile = 64;          // rows walked at a time
constexpr int kMaxD = 128;
// Waves of a SIMD at once that the kernels' registers are fitted to: two where what a lane holds
// (`values`: head sizes' worth of accumulators and operands) leaves room for the rest.  Registers that
// go to scratch memory all the same: 10 of the bf16 query gradient with a bias' at 128 and 1 of the bf16
// key gradient at 64; 110 of the float32 key gradient at 128 (gradients of 8 x 16 heads of
// 1024 rows sharing 4: 57 TFLOP/s, heads of 96 67); in the forms for rows that are not whole words up
// to 87 (bf16, with a bias' gradient), 165 (without) and 312 (float32 keys), at 128.
template <typename T, int DP> constexpr int waves_per_simd(int values) {
  return values * DP * (int)sizeof(T) <= 768 ? 2 : 1;
}
constexpr int kMostPosition = 1 << 29;  // positions and entries of `buckets`: sums of two fit 32 bits
constexpr int kMaxTable = 512;     // buckets of a head: their values and sums stay in LDS
// A finite bias is held within this: its sum with a score then swallows the score, as the
// lowest value of the type does, and neither the scale nor log2(e) takes it to infinity.
constexpr float kBiasLimit = 1e30f;
// The forward kernel's exponents share an error of half a unit in the last place of a row's reference
// (32 here): beyond this it could take sums out of fp32, and differences are formed first.
constexpr float kHugeStat = 1e9f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef unsigned Word __attribute__((ext_vector_type(4)));  // 16 bytes

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
  int wide;  // rows are whole 16-byte words
  int order;  // of the work: below
  int run;    // key heads that an XCD takes in a row
  int first;  // workgroup of a call that a launch begins with: below
};

// Which head (of B x the call's `per_key` heads of each of Hk key heads) and which block a unit of
// work is.  An XCD works on a run of an eighth of all units.
//   kPlain: one head after the other, the block with the longest rows of a causal map first.
//   kMixed: where sequences differ in length, an XCD gets every eighth run of key heads, so that all
// have long and short ones.
//   kTogether: and the longest blocks of all these heads come first, so that the short ones even out
// the end.
enum { kPlain, kMixed, kTogether };
struct Unit {
  int b, kh, g, block;  // key head; which of the heads that share it; block in the order of work
};
__device__ inline Unit unit_of(const Params &p, int unit, int per_key, int blocks) {
  int kv, g, block;
  if (p.order == kPlain) {
    block = unit % blocks, unit /= blocks;
    g = unit % per_key, kv = unit / per_key;
  } else {
    const int runs = p.B * p.Hk / p.run, q = runs / 8, r = runs % 8, each = per_key * blocks;
    int xcd, in, count = (q + 1) * p.run;  // key heads of this XCD
    if (unit < r * count * each) {
      xcd = unit / (count * each), in = unit % (count * each);
    } else {
      unit -= r * count * each, count = q * p.run;
      xcd = r + unit / (count * each), in = unit % (count * each);
    }
    int first = 0;
    if (p.order == kMixed) first = in / each, in %= each, count = 1;
    const int place = in % (count * per_key);
    block = in / (count * per_key);
    first += place / per_key;
    g = place % per_key, kv = (xcd + 8 * (first / p.run)) * p.run + first % p.run;
  }
  return Unit{kv / p.Hk, kv % p.Hk, g, block};
}

__device__ inline int first_position(const Params &p, int b) {
  if (!p.start) return 0;
  return min(max(p.start[b], -kMostPosition), kMostPosition);
}
__device__ inline int key_length(const Params &p, int b) {
  if (!p.lengths) return p.Lk;
  return min(max(p.lengths[b], 0), p.Lk);
}

// Row of a tile that row m of product `blk` (0, 1) has to stand for (see above).
__device__ inline int row_of(int m, int blk) {
  return 32 * ((m >> 2) & 1) + 16 * blk + 4 * (m >> 3) + (m & 3);
}

// -inf in place of the values n of a product with n < first or n >= end.  Two comparisons at a time:
// the compiler would make all sixteen first, and keep their masks in more scalar registers than
// there are.
__device__ inline void keep_between(floatx16 &x, int first, int end) {
#pragma unroll
  for (int n = 0; n < 16; n++) {
    x[n] = n >= first && n < end ? x[n] : -kInf;
    if (n & 1) __builtin_amdgcn_sched_barrier(0);
  }
}

// What a wave's lanes have written to LDS is there for its other lanes: the hardware keeps a wave's
// LDS instructions in order, and the compiler may not move them past this.
__device__ inline void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

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

// A tile in LDS: dense rows, whose 16-byte words are permuted among themselves: word c of a row lies
// at c ^ swizzle(row).  Sixteen lanes that read one word of the sixteen rows 4 g + a and 32 + 4 g + a
// (g = 0, 1, a = 0 .. 3) meet all 64 banks once, and so do those that read four words of four rows.
template <typename T, int DP> constexpr int words() { return DP * (int)sizeof(T) / 16; }
template <typename T, int DP> __device__ inline int swizzle(int row) {
  const int low = ((row >> 1) & 2) | ((row >> 5) & 1);
  if (words<T, DP>() % 16 == 0) return ((row & 3) << 2) | low;
  if (words<T, DP>() % 8 == 0) return ((row & 2) << 1) | low;
  return low;
}
// Word c of row `row`.
template <typename T, int DP> __device__ inline int word_at(int row, int c) {
  return row * words<T, DP>() + (c ^ swizzle<T, DP>(row));
}

// Operand whose summed axis runs along the rows of a tile: row `row`, values 16 chunk + ...
template <typename T, int DP>
__device__ inline Frag<T> row_frag(const Word *tile, int row, int chunk, int half) {
  constexpr int N = sizeof(T) / 2;
  struct { Word w[N]; } f;
#pragma unroll
  for (int n = 0; n < N; n++) f.w[n] = tile[word_at<T, DP>(row, N * (2 * chunk + half) + n)];
  return __builtin_bit_cast(Frag<T>, f);
}

// Operand whose summed axis runs down the rows: column 32 block + (lane & 31), rows r0 + 0 .. 7 in
// the lower half-wave, r0 + Half + 0 .. 7 in the upper.
template <typename T, int DP, int Half> struct Column;
template <int DP, int Half> struct Column<float, DP, Half> {
  static __device__ inline Frag<float> get(const Word *tile, int r0, int block, int lane) {
    const int column = 32 * block + (lane & 31);
    Frag<float> f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int row = r0 + Half * (lane >> 5) + e;
      f.v[e] = ((const float *)&tile[word_at<float, DP>(row, column >> 2)])[column & 3];
    }
    return f;
  }
};
// (the transposing load: of 16 lanes, four address a row's 16 values and lane c gets column c of
// the four rows)
template <int DP, int Half> struct Column<__bf16, DP, Half> {
  static __device__ inline Frag<__bf16> get(const Word *tile, int r0, int block, int lane) {
    const int row = r0 + Half * (lane >> 5) + ((lane & 15) >> 2);
    const int word = 4 * block + ((lane >> 3) & 2) + ((lane >> 1) & 1);
    typedef __attribute__((address_space(3))) shortx4 *lds4;
    struct { shortx4 lo, hi; } f;
    f.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds4)&tile[word_at<__bf16, DP>(row, word)] + (lane & 1));
    f.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds4)&tile[word_at<__bf16, DP>(row + 4, word)] + (lane & 1));
    return __builtin_bit_cast(Frag<__bf16>, f);
  }
};

// 16 bytes of a row: values d0 .., zeros behind the row's end.
template <bool Wide, typename T>
__device__ inline Word load16(const T *row, int d0, int D) {
  constexpr int E = 16 / (int)sizeof(T);
  if (Wide) return d0 < D ? *(const Word *)(row + d0) : Word{0, 0, 0, 0};
  T x[E];
#pragma unroll
  for (int e = 0; e < E; e++) x[e] = d0 + e < D ? row[d0 + e] : (T)0.f;
  return __builtin_bit_cast(Word, *(const __attribute__((ext_vector_type(E))) T *)x);
}

// Column operand straight from memory: row `row` (null: zeros) of this lane, values 16 chunk + ...
template <bool Wide, typename T>
__device__ inline Frag<T> global_frag(const T *row, int chunk, int half, int D) {
  constexpr int E = 16 / (int)sizeof(T), N = 8 / E;
  struct { Word w[N]; } f;
#pragma unroll
  for (int n = 0; n < N; n++)
    f.w[n] = row ? load16<Wide>(row, 16 * chunk + 8 * half + n * E, D) : Word{0, 0, 0, 0};
  return __builtin_bit_cast(Frag<T>, f);
}

// kTile rows of a matrix on their way from memory to LDS.  Whole words go there directly, without
// registers: a wave's instruction fills 64 consecutive words of the tile, so the permutation of a
// row's words is made on the side of the addresses.  Else through registers.
//   Where there are fewer rows, the last one stands for the missing ones, and a row's first word for
// those behind its end: finite values that meet zeros in the product (the other operand is padded
// with zeros, and a pair that is not there has probability zero), so no load is under a condition.
template <typename T, int DP, bool Wide> struct Feed {
  static constexpr int E = 16 / (int)sizeof(T), PerRow = words<T, DP>();
  static constexpr int N = kTile * PerRow / (64 * kWaves);
  Word r[Wide ? 1 : N];
  unsigned offset[Wide ? N : 1];
  unsigned step;  // bytes from row to row

  // the lane's n-th word: its row, and its first value
  static __device__ inline int row_of_word(int n, int tid) {
    return Wide ? ((tid & ~63) * N + n * 64 + (tid & 63)) / PerRow : (tid + n * 64 * kWaves) / PerRow;
  }
  static __device__ inline int first_value(int n, int tid, int D) {
    if (!Wide) return (tid + n * 64 * kWaves) % PerRow * E;
    const int id = (tid & ~63) * N + n * 64 + (tid & 63), row = id / PerRow;
    const int d0 = ((id % PerRow) ^ swizzle<T, DP>(row)) * E;
    return d0 < D ? d0 : 0;
  }
  __device__ inline Feed(int64_t stride, int D, int tid) {
    step = (unsigned)stride * (unsigned)sizeof(T);
    if (Wide) {
#pragma unroll
      for (int n = 0; n < N; n++)
        offset[n] = row_of_word(n, tid) * step + first_value(n, tid, D) * (unsigned)sizeof(T);
    }
  }
  static __device__ inline void to_lds(const T *base, unsigned at, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 : : "s"(to), "v"(at), "s"(base) : "memory", "m0");
  }
  // starts on rows [0, rows) of `base`, rows > 0; `tile` is where they go
  __device__ inline void start(const T *base, int64_t stride, int rows, Word *tile, int D, int tid) {
    if (Wide) {
      const unsigned to =
          __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) Word *)tile +
                                         (tid >> 6) * N * 1024);
      if (rows >= kTile) {
#pragma unroll
        for (int n = 0; n < N; n++) to_lds(base, offset[n], to + n * 1024);
      } else {
#pragma unroll
        for (int n = 0; n < N; n++)
          to_lds(base, min(row_of_word(n, tid), rows - 1) * step +
                           first_value(n, tid, D) * (unsigned)sizeof(T), to + n * 1024);
      }
    } else {
#pragma unroll
      for (int n = 0; n < N; n++)
        r[n] = load16<false>(base + min(row_of_word(n, tid), rows - 1) * stride,
                             first_value(n, tid, D), D);
    }
  }
  // what was started is in the tile, for this wave: before a barrier
  __device__ inline void finish(Word *tile, int tid) const {
    if (Wide) {
      asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    } else {
#pragma unroll
      for (int n = 0; n < N; n++) {
        const int id = tid + n * 64 * kWaves;
        tile[word_at<T, DP>(id / PerRow, id % PerRow)] = r[n];
      }
    }
  }
};

// ---- the bias of a tile of pairs -----------------------------------------------------------
// A tile of kTile rows and kBlock columns has kTile + kBlock - 1 differences; one more, below them,
// is the last of the tile before.  A lane wants eight
// consecutive ones from any place on: four copies, each shifted by one value, let it read them as
// two aligned 16-byte words.  The copies lie 16 banks apart, which keeps the four lanes of one
// word's neighbourhood out of each other's banks.
constexpr int kWindow = kTile + kBlock;  // 192
constexpr int kCopy = 208;
struct Window {
  float copy[4][kCopy];  // value t of copy s at t - s + 4
  __device__ inline void put(int t, float x) {
#pragma unroll
    for (int s = 0; s < 4; s++) copy[s][t - s + 4] = x;
  }
  // differences at .. at + 7, `shift` = at & 3
  __device__ inline floatx8 get(int at, int shift) const {
    const floatx4 *w = (const floatx4 *)&copy[shift][at - shift + 4];
    const floatx4 a = w[0], b = w[1];
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// Without a bias: the two windows are zeros from the start.
__device__ inline void clear(Window *windows, int tid) {
  float *x = &windows[0].copy[0][0];
  for (int n = tid; n < 2 * 4 * kCopy; n += 64 * kWaves) x[n] = 0.f;
}

__device__ inline int bucket_of(const Params &p, int difference) {
  return p.buckets[min(max(difference + p.zero, 0), p.R - 1)];
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

// A lane's column of a transposed result ([DP] values in blocks of 32) to a row of memory, and what
// rounding to T took from it to `rest`, where that is wanted.
template <bool Wide, typename T, int NBlocks>
__device__ inline void store_column(T *row, const floatx16 *acc, float factor, int D, int half,
                                    T *rest = nullptr) {
#pragma unroll
  for (int blk = 0; blk < NBlocks; blk++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int d0 = 32 * blk + 8 * g + 4 * half;
      typedef __attribute__((ext_vector_type(4))) T T4;
      floatx4 x = {acc[blk][4 * g] * factor, acc[blk][4 * g + 1] * factor,
                   acc[blk][4 * g + 2] * factor, acc[blk][4 * g + 3] * factor};
      const T4 y = __builtin_convertvector(x, T4);
      const T4 z = __builtin_convertvector(x - __builtin_convertvector(y, floatx4), T4);
      if (Wide) {
        if (d0 < D) *(T4 *)(row + d0) = y;
        if (rest && d0 < D) *(T4 *)(rest + d0) = z;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (d0 + e < D) {
            row[d0 + e] = y[e];
            if (rest) rest[d0 + e] = z[e];
          }
      }
    }
}

// One value of the output, and what rounding took from it.
template <typename T> __device__ inline void store_value(T *out, T *rest, int64_t at, float x) {
  const T y = (T)x;
  out[at] = y;
  if (rest) rest[at] = (T)(x - (float)y);
}

// Eight of the sixteen values of a product, s = 0, 1; and two eights as the start of one.
__device__ inline floatx8 eight(const floatx16 &x, int s) {
  return s == 0 ? __builtin_shufflevector(x, x, 0, 1, 2, 3, 4, 5, 6, 7)
                : __builtin_shufflevector(x, x, 8, 9, 10, 11, 12, 13, 14, 15);
}
__device__ inline floatx16 sixteen(const floatx8 &lo, const floatx8 &hi) {
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15);
}

// The loads issued so far have arrived: said before a loop, it keeps the compiler from waiting in
// the loop for what was loaded before it, and so for the loop's own loads.
__device__ inline void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

inline bool aligned16(const void *p) { return (uintptr_t)p % 16 == 0; }

// Calls f with the padded head size and whether rows are whole words, as constants.
#define MCX_ATTENTION_DISPATCH(D, wide, F)   \
  do {                                       \
    if (wide) {                              \
      if ((D) <= 32) F(32, true);            \
      else if ((D) <= 64) F(64, true);       \
      else if ((D) <= 96) F(96, true);       \
      else F(128, true);                     \
    } else {                                 \
      if ((D) <= 32) F(32, false);           \
      else if ((D) <= 64) F(64, false);      \
      else if ((D) <= 96) F(96, false);      \
      else F(128, false);                    \
    }                                        \
  } while (0)

// A launch has at most 2^32 threads: more than a quarter of them go into launches of their own.
// Calls f(the launch's parameters, its workgroups).
constexpr int64_t kMostGroups = (int64_t)1 << 22;
template <typename F> int launch_in_pieces(const Params &p, int64_t groups, F f) {
  Params piece = p;
  for (int64_t first = 0; first < groups; first += kMostGroups) {
    piece.first = (int)first;
    f(piece, dim3((unsigned)std::min(groups - first, kMostGroups)));
    MCX_HIP_CHECK_LAUNCH();
  }
  return MCX_OK;
}
// The workgroup of the call that this one is.
__device__ inline int group_of_call(const Params &p) {
  return p.first + xcd_contiguous_tile(blockIdx.x, gridDim.x);
}

// Checks the arguments of an entry point and fills in `p`: MCX_OK, or what is wrong with them.
int make_params(Params &p, const void *q, const void *k, const void *v, const void *table,
                const int32_t *buckets, const int32_t *query_start, const int32_t *key_lengths,
                const mcx_attention_desc *desc, int dtype);

// Work for fewer workgroups than there are compute units is split along the walked axis, in parts
// of four tiles at least, whose results are joined afterwards: into how many parts.
// 384 workgroups in all: gradients and output of 2 x 1250 float32 rows of 6 heads of 48 sharing 2
// take 831 us with no parts, and 349, 286, 299, 324 us with 256, 384, 512, 1024; of 2562 bf16 rows
// of 4 heads of 128 sharing one 236, 208, 249, 261 us.
int parts_of(int64_t units, int64_t tiles);

// The form for few queries against many keys (mcx_attention_split.hip): over how many parts of the
// keys (0: not the form for these sizes), its workspace, and its launch.
int split_parts(const Params &p, int dtype);
size_t split_bytes(const Params &p, int parts);
int launch_split(const Params &p, int parts, void *out, float *stats, void *rest, void *workspace,
                 int dtype, hipStream_t stream);

}  // namespace attention
}  // namespace mcx
