// Low-rank adapters beside a product of microscaled rows: out[m] += up[a] (scale[a] down[a] x[m]), a the row's own.
//
// A launch in front makes low[m] = scale[a] down[a] x[m], 32-bit sums, and keeps it as three bf16 terms (24 bits): the
// product's tiles add up[a] low[m] to their sums before bias and activation, by 16x16x32 instructions over 32 ranks. up
// is one (bf16), two (fp16) or three terms. Rows of a subtile may have adapters of their own: one after the other is
// multiplied by all sixteen rows, and each row takes what its own gives, so that what is in one adapter
// stays with its rows.
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

constexpr int kLowTerms = 3;

struct MxAdapters {
  const uint8_t *up;
  const uint16_t *low;             // [M][kLowTerms][ranks]
  const int32_t *of_row;
  int type, rank, ranks, count;    // ranks: rank up to a multiple of 32, the rest zeros

  // Eight ranks of a row of up, as terms.
  template <class E, int TERMS> __device__ __forceinline__ void load_up(v4i (&u)[TERMS], size_t row, int r) const {
    const typename E::T *at = reinterpret_cast<const typename E::T *>(up) + row * rank + r;
    float x[8];
    if (r + 8 <= rank) load8<E>(x, at);
    else load8_end<E>(x, at, rank - r);
    ad_split<TERMS>(u, x);
  }

  // Adds to the results acc(i, j) of 16 columns by 16 rows: columns column(i) of this lane (lane % 16 of a subtile), rows from
  // m0. Of the adapters that these rows have, number k * share + mine are this wave's.
  template <int TN, int TM, class ACC, class COLUMN>
  __device__ __forceinline__ void add(ACC &&acc, COLUMN &&column, int m0, int M, int N, int mine = 0, int share = 1) const {
    static_assert(TM <= 4, "rows are held a lane each");
    const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
    const int id = lane < 16 * TM && m0 + lane < M ? of_row[m0 + lane] : -1;
    unsigned long long left = __ballot(id >= 0 && id < count);
    for (int k = 0; left; k++) {
      const int a = __builtin_amdgcn_readlane(id, __ffsll(left) - 1);
      const unsigned long long rows = __ballot(id == a);
      left &= ~rows;
      if (k % share != mine) continue;
      for (int r0 = 0; r0 < ranks; r0 += 32) {
        v4i low_terms[TM][kLowTerms];
#pragma unroll
        for (int j = 0; j < TM; j++) {
          const uint16_t *at = low + (size_t)min(m0 + j * 16 + l16, M - 1) * kLowTerms * ranks + r0 + 8 * q;
#pragma unroll
          for (int t = 0; t < kLowTerms; t++) low_terms[j][t] = *reinterpret_cast<const v4i *>(at + t * ranks);
        }
#pragma unroll
        for (int i = 0; i < TN; i++) {
          const size_t row = (size_t)a * N + min(column(i), N - 1);
          auto products = [&](auto kind) {
            typedef decltype(kind) E;
            constexpr int TERMS = std::is_same<E, F32>::value ? 3 : std::is_same<E, F16>::value ? 2 : 1;
            v4i u[TERMS];
            load_up<E, TERMS>(u, row, r0 + 8 * q);
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
              for (int e = 0; e < 4; e++) acc(i, j)[e] += own ? sum[e] : 0.0f;
            }
          };
          if (type == MI355X_BF16) products(BF16());
          else if (type == MI355X_F16) products(F16());
          else products(F32());
        }
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
