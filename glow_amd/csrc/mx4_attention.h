// Attention over a cache of microscaled rows: what a wave does with sixteen rows of queries.
//
// For a head of the cache, "rows" are (row of the batch, query head of the group) pairs, the group's
// heads of a row next to each other. With S = Q K^T, a softmax over tokens and O = P V, everything is
// kept transposed, tokens and columns of values being the matrix instructions' rows, the sixteen
// queries their columns, lane % 16 in what follows; q is lane / 16:
//
//   S   16 tokens x 16 queries by the scaled instruction over 128 columns: codes and scale bytes of
//       the keys as they lie in memory (a lane has one block of a token), queries as sums of 6-bit
//       floats (E2M3) with a power of two for each block of 32: 3 terms and a 4-bit one (E2M1) for 16-bit types,
//       6 for fp32. Nothing of a key is ever converted. A lane gets tokens 4 q .. 4 q + 3. 8-bit terms
//       (E4M3) have as many bits and take twice the time each, and the instruction cuts small products off
//       where exponents lie far apart (2^-17 of the sum; 6-bit products come out exact).
//   P   is what the lane then holds of two tiles of tokens: eight weights of its query, which is what the
//       16x16x32 instruction wants of its second operand, tokens in the order 4 q + i of the first
//       tile, then of the second. No lane needs another's weights.
//   O   values [32 tokens x D] are that instruction's first operand. A lane needs, of its eight tokens, D /
//       16 columns: those next to each other, a word of codes for D = 128; the instruction of
//       number m then has column m of each lane's.  Codes are converted to pairs of neighbouring columns and
//       transposed to pairs of tokens by byte permutes. Results: lane q has columns 32 q .. 32 q + 31 for
//       D = 128, a block of a microscaled result.
//
// The running maximum moves only when a score passes it by more than 2^8: weights stay below 2^8 times what they are
// shifted by then, and most steps have no rescaling. fp16's are shifted up by 2^7, so that small ones stay normal
// numbers; the others' down by 2^39: 2^31 of them are no more than 1, and their sum with values of any size stays in
// the range of 32 bits, as the mean does.
#ifndef GLOW_MI355X_MX4_ATTENTION_H
#define GLOW_MI355X_MX4_ATTENTION_H

#include "mx4_cache.h"

namespace mi355x {

typedef int at_v4i __attribute__((ext_vector_type(4)));
typedef int at_v8i __attribute__((ext_vector_type(8)));
typedef uint32_t at_v6u __attribute__((ext_vector_type(6)));
typedef float at_v4f __attribute__((ext_vector_type(4)));
typedef float at_v16f __attribute__((ext_vector_type(16)));
typedef float at_v32f __attribute__((ext_vector_type(32)));
typedef _Float16 at_v2h __attribute__((ext_vector_type(2)));
typedef _Float16 at_v8h __attribute__((ext_vector_type(8)));
typedef __bf16 at_v2b __attribute__((ext_vector_type(2)));
typedef __bf16 at_v8b __attribute__((ext_vector_type(8)));

struct Attention {
  MxCache c;
  const uint8_t *q;
  uint8_t *out;
  float *part;                    // what splits leave for the joining launch
  size_t q_row_bytes, out_row_bytes;
  int kv_heads, group;            // heads of queries to one of the cache
  int most;                       // tokens of a sequence
  int window, sinks;
  int slots, splits;              // splits: shares of a slot's tokens at most
  int target;                     // shares in all that are to run at once; 0: every slot has all of its shares
  int out_groups;                 // of a microscaled result's row
  float scale;                    // |scale| * log2(e)
  int negative;                   // of the scale
};

constexpr float kAtSlack = 8.0f;
constexpr float kAtNone = -__builtin_inff();

// 6-bit terms of a query, whether a 4-bit one follows, terms of a weight, what weights are shifted up by, the least scale byte of values that count as NaN
// (2^14 times 4 is past fp16's range), and what values are shifted down by until they are divided by the sum of the
// weights: 6 times 2^127 is past bf16's range, and an infinity would make NaN of the rows that do not see it, whose weight is 0.
template <class E> struct AtKind {
  static constexpr int kQ = 6, kP = 3, kNan = 255, kDown = 3;
  static constexpr bool kLast = false;
  static constexpr float kUp = -39;
};
template <> struct AtKind<F16> {
  static constexpr int kQ = 3, kP = 1, kNan = 141, kDown = 0;
  static constexpr bool kLast = true;
  static constexpr float kUp = 7;
};
template <> struct AtKind<BF16> {
  static constexpr int kQ = 3, kP = 1, kNan = 255, kDown = 3;
  static constexpr bool kLast = true;
  static constexpr float kUp = -39;
};
// Queries in fp16 whose result is microscaled: that holds numbers fp16 does not, as the values may be, and so these are bf16
// and weights two terms. us, with them / with fp16: four long sequences 150 / 132, a prompt of 16384 through a window of 1024 528 / 441.
struct AtWide : F16 {};
template <> struct AtKind<AtWide> : AtKind<BF16> { static constexpr int kP = 2; };

// Which rows a slot of sixteen has. Slots of a sequence begin at floor(start * group / 16) + its number, which leaves
// each as many as it needs.
struct AtRows {
  int sequence, begin, count;     // of the sequence's rows in the batch
  int first, last;                // its rows (row, head) of this slot: [first, last)
  int length;
};
template <int ROWS> __device__ __forceinline__ long long at_first_slot(const Attention &p, int s) {
  return (long long)batch_start(p.c, s) * p.group / ROWS + s;
}
template <int ROWS> __device__ __forceinline__ bool at_rows(const Attention &p, int slot, AtRows &r) {
  int length;
  if (p.c.sequences < 64) {                       // one round of loads, a sequence a lane
    const int lane = threadIdx.x & 63, s = min(lane, p.c.sequences);
    const int start = batch_start(p.c, s), tokens = p.c.lengths[min(s, p.c.sequences - 1)];
    const unsigned long long fits = __ballot(lane < p.c.sequences && (long long)start * p.group / ROWS + lane <= slot);
    r.sequence = fits ? 63 - __clzll((long long)fits) : 0;
    r.begin = __builtin_amdgcn_readlane(start, r.sequence);
    r.count = max(__builtin_amdgcn_readlane(start, r.sequence + 1) - r.begin, 0);
    length = __builtin_amdgcn_readlane(tokens, r.sequence);
  } else {
    r.sequence = __builtin_amdgcn_readfirstlane(
        find_sequence<64>(p.c.sequences, slot, [&](int s) { return at_first_slot<ROWS>(p, s); }));
    r.begin = batch_start(p.c, r.sequence);
    r.count = max(batch_start(p.c, r.sequence + 1) - r.begin, 0);
    length = p.c.lengths[r.sequence];
  }
  const long long at = (slot - ((long long)r.begin * p.group / ROWS + r.sequence)) * ROWS;
  const int all = r.count * p.group;
  if (at < 0 || at >= all) return false;
  r.first = (int)at;
  r.last = min(all, r.first + ROWS);
  r.length = min(max(length, 0), p.most);
  return true;
}
// The tiles of tokens that rows at `low` to `high` see some of: those of the first `sinks`, then [from, ..).
struct AtTiles {
  int sinks, from, all;
  __device__ __forceinline__ int at(int u) const { return u < sinks ? u : u - sinks + from; }
};
__device__ __forceinline__ AtTiles at_tiles(const Attention &p, int low, int high) {
  AtTiles t;
  t.from = max(0, low - p.window + 1) / kCacheTile;     // (low >= -1, window <= 2^31 - 1)
  t.sinks = min((int)(((unsigned)p.sinks + kCacheTile - 1) / kCacheTile), t.from);
  t.all = t.sinks + high / kCacheTile + 1 - t.from;
  if (high < 0) t.all = 0;
  return t;
}

// Steps of 32 tokens in a share of a slot that has `steps`: what gives all sequences together `target` shares, so that long
// and short ones have shares of a size, but `least` steps at least and no more than `splits` shares. (There is a target
// for a few hundred sequences at most: more need no shares.)
__device__ __forceinline__ int at_share_steps(const Attention &p, int steps, int least) {
  int chunk = max((int)(((long long)steps + p.splits - 1) / p.splits), least);
  if (p.target) {
    float all = 0;                                  // (in steps; equal in all waves of all launches)
    const long long most = (long long)p.window + p.sinks;
    for (int i = threadIdx.x & 63; i < p.c.sequences; i += 64)
      all += (float)((min((long long)min(max(p.c.lengths[i], 0), p.most), most) + 31) / 32);
    chunk = max(chunk, (int)fminf(__builtin_ceilf(wave_sum(all) / (float)p.target), 1e9f));
  }
  return __builtin_amdgcn_readfirstlane(chunk);
}

// ---- queries -----------------------------------------------------------------------

// Sixteen rows of queries of D columns as sums of small floats: 32 q to 32 q + 31 of 128 columns are lane q's, a block
// with a power of two of its own. The largest is scaled to [2, 4); a 6-bit term rounds to an eighth at most, and the next has
// a thirty-second of its scale, in which that is 4 at most: after T terms what is left is 2^(1 - 5T) of the largest at most,
// 2^-29 after six. Behind three terms (2^-14) a 4-bit one rounds to a half what is up to 4, which leaves 2^-17: rotary
// queries have columns that stand out, next to which the others' bits would be lost. It lies in LDS: where four waves share a SIMD's
// registers, or two with 32 rows each, a term more in registers had 7 to 49 of them in memory, in LDS 3 to 9, as with three
// terms. With / without it, us: four long sequences 134 / 130, two prompts of 4096 411 / 393.
template <class E, int D> struct AtQueries {
  static constexpr int kTerms = AtKind<E>::kQ, kAll = kTerms + AtKind<E>::kLast, kChunks = (D + 127) / 128, kWords = (kAll + 3) / 4;
  static constexpr int kLds = AtKind<E>::kLast ? kChunks * 1024 : 0;      // bytes of a wave
  at_v6u codes[kChunks][kTerms];
  int scale[kChunks][kWords];                    // a byte a term
  const at_v4i *last;                            // of this lane, 64 apart

  // `lds`: this wave's.
  __device__ __forceinline__ void load(const typename E::T *row, bool negative, uint8_t *lds) {
    const int q = (threadIdx.x & 63) >> 4;
    last = reinterpret_cast<const at_v4i *>(lds) + (threadIdx.x & 63);
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      at_v16f even, odd;               // the conversion takes every second column in either
      uint32_t most = 0;
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        float y[8];
        load8<E>(y, row + c * 128 + 32 * (D == 64 ? q & 1 : q) + e);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if (D == 64) y[j] = q < 2 ? y[j] : 0.0f;
          most = max(most, magnitude_bits(y[j]));
          y[j] = negative ? -y[j] : y[j];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) even[e / 2 + j] = y[2 * j], odd[e / 2 + j] = y[2 * j + 1];
      }
      const int exponent = (int)(most >> 23);
      auto byte_of = [&](int t) { return max(exponent - 1 - 5 * t, 1); };
#pragma unroll
      for (int w = 0; w < kWords; w++) scale[c][w] = 0;
#pragma unroll
      for (int t = 0; t < kAll; t++) scale[c][t / 4] |= (exponent == 255 ? 255 : byte_of(t)) << (8 * (t % 4));
#pragma unroll
      for (int t = 0; t < kTerms; t++) {
        const float s = __uint_as_float((uint32_t)byte_of(t) << 23);
        const at_v6u six = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, s);
        // (the conversion writes words of its result before it has read all operands: they have to live on)
        asm volatile("" ::"v"(even), "v"(odd), "v"(s), "v"(six));
        if (t + 1 < kAll) {
          const at_v32f back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(six, s);
#pragma unroll
          for (int j = 0; j < 16; j++) even[j] -= back[2 * j], odd[j] -= back[2 * j + 1];    // (exact)
        }
        codes[c][t] = six;
      }
      if constexpr (AtKind<E>::kLast) {
        at_v4i four;
#pragma unroll
        for (int w = 0; w < 4; w++) {
          float y[8];
#pragma unroll
          for (int j = 0; j < 4; j++) y[2 * j] = even[4 * w + j], y[2 * j + 1] = odd[4 * w + j];
          four[w] = (int)mx4_codes8(y, (uint32_t)byte_of(kTerms));
        }
        reinterpret_cast<at_v4i *>(lds)[c * 64 + (threadIdx.x & 63)] = four;
      }
    }
  }
};

// Scores of sixteen tokens of all terms of 128 columns, 4 bits by 6 and by 4.
template <int T, int TERMS, int WORDS>
__device__ __forceinline__ at_v4f at_terms(at_v4i keys, int key_scale, const at_v6u (&q)[TERMS], const int (&scale)[WORDS], at_v4f acc) {
  if constexpr (T == TERMS) return acc;
  else {
    const at_v4f sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
        at_v8i{keys[0], keys[1], keys[2], keys[3], 0, 0, 0, 0},
        at_v8i{(int)q[T][0], (int)q[T][1], (int)q[T][2], (int)q[T][3], (int)q[T][4], (int)q[T][5], 0, 0}, acc, 4, 2, 0, key_scale,
        T % 4, scale[T / 4]);
    return at_terms<T + 1>(keys, key_scale, q, scale, sum);
  }
}
template <class E, int D>
__device__ __forceinline__ at_v4f at_scores(at_v4i keys, int key_scale, const AtQueries<E, D> &q, int c, at_v4f acc) {
  const at_v4f sum = at_terms<0>(keys, key_scale, q.codes[c], q.scale[c], acc);
  if constexpr (AtKind<E>::kLast) {
    constexpr int T = AtKind<E>::kQ;
    const at_v4i four = q.last[c * 64];
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(at_v8i{keys[0], keys[1], keys[2], keys[3], 0, 0, 0, 0},
                                                            at_v8i{four[0], four[1], four[2], four[3], 0, 0, 0, 0}, sum, 4, 4, 0,
                                                            key_scale, T % 4, q.scale[c][T / 4]);
  }
  return sum;
}

// ---- weights and values --------------------------------------------------------------

// The power of two that a block of values is multiplied by, 2^-127 at least: what that makes too large is below 2^-124, nothing
// once it is multiplied by a weight of up to 2^-31.
template <class E> __device__ __forceinline__ float at_value_scale(uint32_t byte) {
  return __uint_as_float((uint32_t)max((int)(byte << 23) - (AtKind<E>::kDown << 23), 0x00400000));
}
// What results are divided by.
template <class E> __device__ __forceinline__ float at_divisor(float sum) {
  return AtKind<E>::kDown ? sum * (1.0f / (1 << AtKind<E>::kDown)) : sum;
}

// Pairs of values, and the product with weights, in the type that weights are rounded to: bf16 but for fp16's.
template <class E> struct AtValues {
  typedef at_v2b Two;
  static __device__ __forceinline__ Two two(uint32_t codes, float s, std::integral_constant<int, 0>) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0);
  }
  static __device__ __forceinline__ Two two(uint32_t codes, float s, std::integral_constant<int, 1>) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1);
  }
  static __device__ __forceinline__ Two two(uint32_t codes, float s, std::integral_constant<int, 2>) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2);
  }
  static __device__ __forceinline__ Two two(uint32_t codes, float s, std::integral_constant<int, 3>) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3);
  }
  static __device__ __forceinline__ Two pack(float a, float b) { return Two{(__bf16)a, (__bf16)b}; }
  static constexpr int kOnes = 0x3f803f80;
  static __device__ __forceinline__ at_v4f multiply(at_v4i values, at_v4i weights, at_v4f acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(at_v8b, values), __builtin_bit_cast(at_v8b, weights),
                                                   acc, 0, 0, 0);
  }
};
template <> struct AtValues<F16> {
  typedef at_v2h Two;
  static __device__ __forceinline__ Two two(uint32_t codes, float s, std::integral_constant<int, 0>) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 0);
  }
  static __device__ __forceinline__ Two two(uint32_t codes, float s, std::integral_constant<int, 1>) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 1);
  }
  static __device__ __forceinline__ Two two(uint32_t codes, float s, std::integral_constant<int, 2>) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 2);
  }
  static __device__ __forceinline__ Two two(uint32_t codes, float s, std::integral_constant<int, 3>) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 3);
  }
  static __device__ __forceinline__ Two pack(float a, float b) { return Two{(_Float16)a, (_Float16)b}; }
  static constexpr int kOnes = 0x3c003c00;
  static __device__ __forceinline__ at_v4f multiply(at_v4i values, at_v4i weights, at_v4f acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(at_v8h, values), __builtin_bit_cast(at_v8h, weights),
                                                  acc, 0, 0, 0);
  }
};

// Eight weights of a lane as sums of kP terms.
template <class E> __device__ __forceinline__ void at_pack(at_v4i (&w)[AtKind<E>::kP], float (&p)[8]) {
  typedef AtValues<E> V;
#pragma unroll
  for (int t = 0; t < AtKind<E>::kP; t++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const typename V::Two two = V::pack(p[2 * j], p[2 * j + 1]);
      w[t][j] = __builtin_bit_cast(int, two);
      if (t + 1 < AtKind<E>::kP) p[2 * j] -= (float)two[0], p[2 * j + 1] -= (float)two[1];
    }
}

// Eight tokens' words of codes (eight neighbouring columns each; COLS = 4: the low half) -> for each column the
// eight tokens' values, in the matrix instruction's order: use(column, values).
template <class E, int COLS, class USE>
__device__ __forceinline__ void at_transpose(const uint32_t (&codes)[8], const float (&scale)[8], USE &&use) {
  typedef AtValues<E> V;
  auto columns = [&](auto pair) {
    at_v4i even, odd;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t a = __builtin_bit_cast(uint32_t, V::two(codes[2 * j], scale[2 * j], pair));
      const uint32_t b = __builtin_bit_cast(uint32_t, V::two(codes[2 * j + 1], scale[2 * j + 1], pair));
      even[j] = (int)__builtin_amdgcn_perm(b, a, 0x05040100);
      odd[j] = (int)__builtin_amdgcn_perm(b, a, 0x07060302);
    }
    use(2 * decltype(pair)::value, even);
    use(2 * decltype(pair)::value + 1, odd);
  };
  columns(std::integral_constant<int, 0>());
  columns(std::integral_constant<int, 1>());
  if constexpr (COLS == 8) {
    columns(std::integral_constant<int, 2>());
    columns(std::integral_constant<int, 3>());
  }
}

// The same of four tokens, half of an operand.
template <class E, int COLS, class HALF>
__device__ __forceinline__ void at_transpose4(HALF (&out)[COLS], const uint32_t (&codes)[4], const float (&scale)[4]) {
  typedef AtValues<E> V;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    auto columns = [&](auto pair) {
      constexpr int P = decltype(pair)::value;
      const uint32_t a = __builtin_bit_cast(uint32_t, V::two(codes[2 * j], scale[2 * j], pair));
      const uint32_t b = __builtin_bit_cast(uint32_t, V::two(codes[2 * j + 1], scale[2 * j + 1], pair));
      out[2 * P][j] = (int)__builtin_amdgcn_perm(b, a, 0x05040100);
      out[2 * P + 1][j] = (int)__builtin_amdgcn_perm(b, a, 0x07060302);
    };
    columns(std::integral_constant<int, 0>());
    columns(std::integral_constant<int, 1>());
    if constexpr (COLS == 8) {
      columns(std::integral_constant<int, 2>());
      columns(std::integral_constant<int, 3>());
    }
  }
}

// 2^x, 0 of minus infinity.
__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// The largest of a query's scores over the four lanes that hold it.
__device__ __forceinline__ float at_max(float x) {
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __builtin_elementwise_maximum(__uint_as_float(s[0]), __uint_as_float(s[1]));
  s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// A row at `position` sees the token.
__device__ __forceinline__ bool at_sees(const Attention &p, int position, int token) {
  return token <= position && (token > position - p.window || token < p.sinks);
}
// Whether rows at `low` to `high` see all of a tile's tokens, and whether they see none.
__device__ __forceinline__ bool at_sees_all(const Attention &p, int low, int high, int first) {
  return first >= 0 && first + kCacheTile - 1 <= low && first > high - p.window;
}
__device__ __forceinline__ bool at_sees_none(const Attention &p, int low, int high, int first) {
  return first < 0 || first > high || (first + kCacheTile - 1 <= low - p.window && first >= p.sinks);
}

// Whether lanes of `bad`, values of a team's token, hold a bad block of which this lane has columns: 4 of the team's 16
// lanes, or 8 where it has two blocks.
template <int D> __device__ __forceinline__ bool at_bad_block(unsigned long long bad, int team, int q) {
  return D == 64 ? (bad >> (16 * team + 8 * (q >> 1)) & 0xff) != 0 : (bad >> (16 * team + 4 * q) & 0xf) != 0;
}

// The largest of a lane's query's scores, scaled. (maximum gives NaN as soon as one is NaN, which max would have to be kept
// from by another instruction for each.)
template <int N> __device__ __forceinline__ float at_top(const float (&score)[N], float scale) {
  float top[N];
#pragma unroll
  for (int j = 0; j < N; j++) top[j] = score[j];
#pragma unroll
  for (int half = N / 2; half > 0; half /= 2)
#pragma unroll
    for (int j = 0; j < half; j++) top[j] = __builtin_elementwise_maximum(top[j], top[j + half]);
  return at_max(top[0]) * scale;
}
// Scores of a lane's query (tokens that it does not see: minus infinity, and not in `seen`, which counts unless `whole`)
// become weights; the results so far are rescaled where the largest score moves.
template <class E, int N, int M>
__device__ __forceinline__ void at_weigh(float (&score)[N], float &most, float &sum, at_v4f (&acc)[M], float scale, bool whole,
                                         unsigned seen) {
  const float top = at_top(score, scale);
  const bool up = top > most + kAtSlack;
  if (__ballot(up)) {
    const float factor = up ? at_exp2(most - top) : 1.0f;
    most = up ? top : most;
    sum *= factor;
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[m][i] *= factor;
  }
  const float off = AtKind<E>::kUp - most;
#pragma unroll
  for (int j = 0; j < N; j++) score[j] = at_exp2(fmaf(score[j], scale, off));
  if (!whole) {
#pragma unroll
    for (int j = 0; j < N; j++) score[j] = seen >> j & 1 ? score[j] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < N; j++) sum += score[j];
}

// ---- results -------------------------------------------------------------------------

// Stores the results of quarter `i` of a slot's columns: those that component i of the results has, lane q's
// 4 q + i. D = 128 and 256: columns 128 c + 8 (4 q + i) + 0 .. 7; D = 64: 4 (4 q + i) + 0 .. 3. Where the
// result is microscaled, all waves of a workgroup call this together, four of them with results (`mine`) and i of their
// own (`most`: words of LDS for [4][64]).
template <class E, class OUT, int D>
__device__ __forceinline__ void at_store(const Attention &p, const AtRows &r, int h, int i, float (&x)[D / 16],
                                         uint32_t (*most)[64], bool mine) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
  const int at = r.first + l16, token = at / p.group, head = h * p.group + (at - token * p.group);
  uint8_t *row = p.out + (size_t)(r.begin + token) * p.out_row_bytes;
  constexpr int kChunks = (D + 127) / 128, COLS = D == 64 ? 4 : 8;
  if constexpr (OUT::kSize != 0) {
    if (at < r.last) {
      typename OUT::T *o = reinterpret_cast<typename OUT::T *>(row) + (size_t)head * D;
#pragma unroll
      for (int c = 0; c < kChunks; c++) {
        if constexpr (COLS == 8) {
          float y[8];
#pragma unroll
          for (int m = 0; m < 8; m++) y[m] = x[c * 8 + m];
          store8<OUT>(o + c * 128 + 8 * (4 * q + i), y);
        } else {
#pragma unroll
          for (int m = 0; m < 4; m++) o[4 * (4 * q + i) + m] = OUT::from(x[m]);
        }
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < COLS; j++) m = max(m, magnitude_bits(x[c * 8 + j]));
      if (COLS == 4) m = max_across16(m);           // (a block is two lanes')
      __syncthreads();
      if (mine) most[i][lane] = m;
      __syncthreads();
      m = max(max(most[0][lane], most[1][lane]), max(most[2][lane], most[3][lane]));
      const uint32_t byte = mx4_scale_byte(m);
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = j < COLS ? x[c * 8 + (j < COLS ? j : 0)] : 0.0f;
      const uint32_t codes = mx4_codes8(y, byte);
      if (mine && at < r.last) {
        const size_t column = (size_t)head * D + c * 128 + COLS * (4 * q + i);
        uint8_t *scales = row + (size_t)p.out_groups * kMxGroupBytes;
        if constexpr (COLS == 8) *reinterpret_cast<uint32_t *>(row + column / 2) = codes;
        else *reinterpret_cast<uint16_t *>(row + column / 2) = (uint16_t)codes;
        if (column % 32 == 0) scales[column / 32] = (uint8_t)byte;
        // the last head fills its group and the row up with zeros
        if (c == kChunks - 1 && head == p.kv_heads * p.group - 1) {
          const int heads = p.kv_heads * p.group;
          if (D == 64 && (heads & 1)) {
            reinterpret_cast<uint16_t *>(row + (size_t)heads * 32)[4 * q + i] = 0;
            if (i == 0 && q < 2) scales[heads * 2 + q] = 0;
          }
          if (i == 1 && q < ((-p.out_groups) & 3)) reinterpret_cast<uint32_t *>(scales)[p.out_groups + q] = 0;
        }
      }
    }
  }
}

// What a share of a slot of sixteen rows leaves: its results, component by component, then the largest score and the sum
// of each query; the first share how many there are, too.
template <int D> __device__ __forceinline__ constexpr size_t at_part_floats() { return 16 * D + 48; }

// The whole of a slot's results by one wave: a lane has the components of its query side by side.
template <class E, class OUT, int D, int M>
__device__ __forceinline__ void at_store_whole(const Attention &p, const AtRows &r, int h, const at_v4f (&acc)[M], float sum) {
  static_assert(M >= D / 16, "results");
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
  const int at = r.first + l16, token = at / p.group, head = h * p.group + (at - token * p.group);
  const bool there = at < r.last;
  uint8_t *row = p.out + (size_t)(r.begin + token) * p.out_row_bytes;
  constexpr int kChunks = (D + 127) / 128, COLS = D == 64 ? 4 : 8;
  const float by = sum == 0 ? 0.0f : 1.0f / at_divisor<E>(sum);
#pragma unroll
  for (int c = 0; c < kChunks; c++) {
    float x[4][8];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int m = 0; m < 8; m++) x[i][m] = m < COLS ? acc[c * 8 + (m < COLS ? m : 0)][i] * by : 0.0f;
    const size_t column = (size_t)head * D + c * 128 + 4 * COLS * q;
    if constexpr (OUT::kSize != 0) {
      typename OUT::T *o = reinterpret_cast<typename OUT::T *>(row) + column;
      if (there) {
        if constexpr (COLS == 8) {
#pragma unroll
          for (int i = 0; i < 4; i++) store8<OUT>(o + 8 * i, x[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float y[8] = {x[i][0], x[i][1], x[i][2], x[i][3], x[i + 1][0], x[i + 1][1], x[i + 1][2], x[i + 1][3]};
            store8<OUT>(o + 4 * i, y);
          }
        }
      }
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < COLS; j++) m = max(m, magnitude_bits(x[i][j]));
      if (COLS == 4) m = max_across16(m);           // (a block is two lanes')
      const uint32_t byte = mx4_scale_byte(m);
      uint32_t codes[4];
#pragma unroll
      for (int i = 0; i < 4; i++) codes[i] = mx4_codes8(x[i], byte);
      if (there) {
        uint8_t *scales = row + (size_t)p.out_groups * kMxGroupBytes;
        if constexpr (COLS == 8) *reinterpret_cast<uint4 *>(row + column / 2) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
        else *reinterpret_cast<uint2 *>(row + column / 2) = make_uint2((codes[0] & 0xffff) | codes[1] << 16, (codes[2] & 0xffff) | codes[3] << 16);
        if (column % 32 == 0) scales[column / 32] = (uint8_t)byte;
        // the last head fills its group and the row up with zeros
        const int heads = p.kv_heads * p.group;
        if (c == kChunks - 1 && head == heads - 1) {
          if (D == 64 && (heads & 1)) {
            *reinterpret_cast<uint2 *>(row + (size_t)heads * 32 + 8 * q) = make_uint2(0, 0);
            if (q < 2) scales[heads * 2 + q] = 0;
          }
          if (q < ((-p.out_groups) & 3)) reinterpret_cast<uint32_t *>(scales)[p.out_groups + q] = 0;
        }
      }
    }
  }
}

// Launches the kernel for many rows of queries (mx4_attention_prompt.hip).
int at_prompt_launch(const Attention &p, int type, bool mx4, int dim, hipStream_t st);
constexpr int kPromptWaves = 4;
// Sixteens of rows that a wave of that kernel has: as many as its registers hold.
constexpr int at_prompt_sixteens(int type, int dim) { return type == MI355X_F32 || dim == 256 ? 1 : 2; }

} // namespace mi355x

#endif
