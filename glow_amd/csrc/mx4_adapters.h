// Low-rank adapters beside a product of microscaled rows: out[m] += up[a] (scale[a] down[a] x[m]), a the row's own.
//
// A launch in front makes low[m] = scale[a] down[a] x[m], 32-bit sums, in parts of K where rows are few: the product's
// tiles add the parts, split them into three bf16 terms (24 bits) and add up[a] low[m] to their sums before bias and
// activation, by 16x16x32 instructions over 32 ranks. up is one (bf16), two (fp16) or three terms. Rows of a subtile may have adapters of their own: one after the other is
// multiplied by all sixteen rows, and each row takes what its own gives, so that what is in one adapter
// stays with its rows.
//
// What this adds to a product, us: 64 rows of 64 adapters of rank 16, 4096 x 4096, bf16: 19 for 10 (four adapters a wave, a load's
// latency each); 4096 rows of six of rank 64, fp16: 72 for 48 (three rounds of loads at the end of each tile, and 5 matrix
// instructions for 32 ranks of a subtile).
#ifndef GLOW_MI355X_MX4_ADAPTERS_H
#define GLOW_MI355X_MX4_ADAPTERS_H

#include "mx4_fc.h"

namespace mi355x {

typedef __bf16 ad_v8b __attribute__((ext_vector_type(8)));
typedef __bf16 ad_v2b __attribute__((ext_vector_type(2)));

// Eight floats as a sum of TERMS bf16.
template <int TERMS> __device__ __forceinline__ void ad_split(v4i (&t)[TERMS], float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < TERMS; k++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const ad_v2b two = {(__bf16)x[2 * j], (__bf16)x[2 * j + 1]};
      t[k][j] = __builtin_bit_cast(int, two);
      if (k + 1 < TERMS) x[2 * j] -= (float)two[0], x[2 * j + 1] -= (float)two[1];
    }
}
__device__ __forceinline__ mx_v4f ad_multiply(v4i a, v4i b, mx_v4f acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ad_v8b, a), __builtin_bit_cast(ad_v8b, b), acc, 0, 0, 0);
}

constexpr int kLowTerms = 3, kMostParts = 4;

struct MxAdapters {
  const uint8_t *up;
  const float *low;                // [parts][M][ranks]
  const int32_t *of_row;
  int type, rank, ranks, count;    // ranks: rank up to a multiple of 32, the rest zeros
  int parts;

  // Eight ranks of a row of up, q's of those from r0 on; zeros behind the last.
  template <class E> __device__ __forceinline__ typename E::Eight load_up(size_t row, int r0, int q) const {
    const typename E::T *at = reinterpret_cast<const typename E::T *>(up) + row * rank;
    const int r = r0 + 8 * q;
    // (no condition of each lane's where it can be done without: loads behind one are not asked for together)
    if (r0 + 32 <= rank) return load_eight<E>(at + r);
    if (rank % 8 == 0) {
      const typename E::Eight e = load_eight<E>(at + min(r, rank - 8));
      return r < rank ? e : typename E::Eight{};
    }
    return r + 8 <= rank ? load_eight<E>(at + r) : load_eight_end<E>(at + r, rank - r);
  }
  template <class E, int TERMS> static __device__ __forceinline__ void split(v4i (&u)[TERMS], const typename E::Eight &e) {
    if constexpr (std::is_same<E, BF16>::value) u[0] = __builtin_bit_cast(v4i, e);
    else {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = E::get(e, j);
      ad_split<TERMS>(u, x);
    }
  }

  // Adds to the results acc(i, j) of 16 columns by 16 rows: columns column(i) of this lane (lane % 16 of a subtile), rows from
  // m0. Of the adapters that these rows have, number k * share + mine are this wave's.
  template <int TN, int TM, class ACC, class COLUMN>
  __device__ __forceinline__ void add(ACC &&acc, COLUMN &&column, int m0, int M, int N, int mine = 0, int share = 1) const {
    const int lane = threadIdx.x & 63;
    const int id = lane < 16 * TM && m0 + lane < M ? of_row[m0 + lane] : -1;
    const unsigned long long rows = __ballot(id >= 0 && id < count);
    if (!rows) return;
    if (type == MI355X_BF16) add_of<BF16, TN, TM>(acc, column, m0, M, N, mine, share, id, rows);
    else if (type == MI355X_F16) add_of<F16, TN, TM>(acc, column, m0, M, N, mine, share, id, rows);
    else add_of<F32, TN, TM>(acc, column, m0, M, N, mine, share, id, rows);
  }
  // The columns of several subtiles are asked for at once, and those of the next adapter, or of the next subtiles, while the
  // ones in front are multiplied: a load takes as long as ten such products.
  template <class E, int TN, int TM, class ACC, class COLUMN>
  __device__ __forceinline__ void add_of(ACC &acc, COLUMN &column, int m0, int M, int N, int mine, int share, int id,
                                         unsigned long long all) const {
    static_assert(TM <= 4, "rows are held a lane each");
    constexpr int TERMS = std::is_same<E, F32>::value ? 3 : std::is_same<E, F16>::value ? 2 : 1;
    constexpr int AT_ONCE = TN < (E::kSize == 4 ? 2 : 4) ? TN : (E::kSize == 4 ? 2 : 4), PARTS = TN / AT_ONCE;
    static_assert(TN % AT_ONCE == 0, "subtiles");
    const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
    for (int r0 = 0; r0 < ranks; r0 += 32) {
      v4i low_terms[TM][kLowTerms];
#pragma unroll
      for (int j = 0; j < TM; j++) {
        const float *at = low + (size_t)min(m0 + j * 16 + l16, M - 1) * ranks + r0 + 8 * q;
        float x[8];
        load8<F32>(x, at);
        if (parts > 1) {                           // (all asked for before the first is added)
          float y[kMostParts - 1][8];
#pragma unroll
          for (int k = 1; k < kMostParts; k++) load8<F32>(y[k - 1], at + (size_t)min(k, parts - 1) * M * ranks);
#pragma unroll
          for (int k = 1; k < kMostParts; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] += k < parts ? y[k - 1][e] : 0.0f;
        }
        ad_split<kLowTerms>(low_terms[j], x);
      }
      // this wave's adapters one after the other: `a` and its rows
      unsigned long long left = all;
      int k = 0;
      auto following = [&](int &a, unsigned long long &rows) {
        while (left) {
          a = __builtin_amdgcn_readlane(id, __ffsll(left) - 1);
          rows = __ballot(id == a);
          left &= ~rows;
          if (k++ % share == mine) return true;
        }
        return false;
      };
      typename E::Eight coming[AT_ONCE];
      auto ask = [&](int a, int part) {
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) coming[i] = load_up<E>((size_t)a * N + min(column(part * AT_ONCE + i), N - 1), r0, q);
      };
      int a = 0, next_a = 0;
      unsigned long long rows = 0, next_rows = 0;
      bool more = following(a, rows);
      if (more) ask(a, 0);
      while (more) {
        more = following(next_a, next_rows);
#pragma unroll
        for (int part = 0; part < PARTS; part++) {
          typename E::Eight now[AT_ONCE];
#pragma unroll
          for (int i = 0; i < AT_ONCE; i++) now[i] = coming[i];
          if (part + 1 < PARTS) ask(a, part + 1);
          else if (more) ask(next_a, 0);
#pragma unroll
          for (int i = 0; i < AT_ONCE; i++) {
            v4i u[TERMS];
            split<E, TERMS>(u, now[i]);
#pragma unroll
            for (int j = 0; j < TM; j++) {
              if (!(rows >> (16 * j) & 0xffff)) continue;
              mx_v4f sum = {0, 0, 0, 0};
              // the smallest products first; a third term by a third one is below the 32-bit sum's own steps
#pragma unroll
              for (int order = TERMS + kLowTerms - 2; order >= 0; order--)
#pragma unroll
                for (int t = 0; t < TERMS; t++)
                  if (order - t >= 0 && order - t < kLowTerms && order <= 3) sum = ad_multiply(u[t], low_terms[j][order - t], sum);
              const bool own = rows >> (16 * j + l16) & 1;
#pragma unroll
              for (int e = 0; e < 4; e++) acc(part * AT_ONCE + i, j)[e] += own ? sum[e] : 0.0f;
            }
          }
        }
        a = next_a, rows = next_rows;
      }
    }
  }
};

struct MxFcAdapted : MxFc {
  static constexpr bool kAdapters = true;
  MxAdapters ad;
};

} // namespace mi355x

#endif
