// Products of microscaled rows with few results, or few columns: one launch that is as long as
// its longest chain of dependent steps.
//
// A workgroup multiplies 16 weight rows (or 32) by 16 or 32 input rows, its eight waves each a
// share of K. Fragments go from memory straight into registers in the matrix cores' layout: a
// lane feeds one block of 32 columns, row lane % 16, block lane / 16 of a group. A float input
// is quantised there and then: a lane has its whole block, so that no lane needs another one's
// values, and no launch in front is needed. Partial results meet in LDS.
//
// Up to four rows are quantised by the workgroup as a whole, a thread a block, into LDS, while
// the weights are on their way: left to the waves, each lane would load and convert the row that
// its number modulo sixteen stands for, the last one again and again.
//
// What bounds it: the launch (3 us), one round of loads of every wave, and the rate at which a CU
// pulls rows from L2. One row, 4096 x 4096: 4.4 us from a microscaled row (9 MB of weights, 1.7 us at
// the rate of a large copy), 4.8 from fp16 (6.1 converted by the waves). 128 x 1024 x
// 1024 of bf16 4.9, 61 x 415 x 509 of fp32 3.5 (rows x K x columns). Other splits of the eight waves,
// over input rows as well as K, are slower wherever K has a group for each.
#ifndef GLOW_MI355X_MX4_SMALL_H
#define GLOW_MI355X_MX4_SMALL_H

#include "mx4_tiles.h"

namespace mi355x {

// What a lane holds of a block of an input row before it is multiplied.
template <class IN> struct SmallBlock {
  typename IN::Eight v[4];
  __device__ __forceinline__ void load(const uint8_t *row, int groups, int g, int b, int K) {
    const int k = g * kMxGroup + b * 32;
    const typename IN::T *at = reinterpret_cast<const typename IN::T *>(row) + k;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int left = K - k - q * 8;
      if (left >= 8) v[q] = load_eight<IN>(at + q * 8);
      else v[q] = load_eight_end<IN>(at + q * 8, left);
    }
  }
  __device__ __forceinline__ void codes(v4i &c, int &byte) const {
    uint32_t most = 0;
#pragma unroll
    for (int q = 0; q < 4; q++) most = max(most, largest8<IN>(v[q]));
    byte = (int)mx4_scale_byte(largest_bits<IN>(most));
#pragma unroll
    for (int q = 0; q < 4; q++) c[q] = (int)mx4_codes8_of<IN>(v[q], (uint32_t)byte);
  }
};
template <> struct SmallBlock<MX4> {
  v4i v;
  int s;
  __device__ __forceinline__ void load(const uint8_t *row, int groups, int g, int b, int) {
    v = *reinterpret_cast<const v4i *>(row + (size_t)g * kMxGroupBytes + b * 16);
    s = reinterpret_cast<const int *>(row + (size_t)groups * kMxGroupBytes)[g] >> (8 * b);
  }
  __device__ __forceinline__ void codes(v4i &c, int &byte) const { c = v, byte = s; }
};

constexpr int kSmallWaves = 8;

constexpr int kSharedRows = 4;
// Bytes from one shared row to the next in LDS: its codes, its scales, and 16 so that rows of a power of
// two do not lie on the same banks.
__host__ __device__ constexpr int mx4_shared_row(int groups) { return (groups * (kMxGroupBytes + 4) + 15) / 16 * 16 + 16; }

template <class IN, class OUT, int MT, int NT, bool SHARED>
__global__ __launch_bounds__(kSmallWaves * 64, 2) void mx4_fc_small_kernel(MxFc p, int K, int tiles_n) {
  // groups in flight: as many as their registers allow
  static_assert(!SHARED || (MT == 1 && IN::kSize), "shared rows");
  constexpr int kRegs = IN::kSize == 0 || SHARED ? 5 : IN::kSize * 8;
  constexpr int D = kRegs * MT <= 20 ? 4 : kRegs * MT <= 32 ? 2 : 1;
  constexpr int kTiles = MT * NT;
  __shared__ float s_part[kSmallWaves][kTiles * 4][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, b = lane >> 4;
  const int n0 = (int)(blockIdx.x % (unsigned)tiles_n) * (16 * NT);
  const int m0 = (int)(blockIdx.x / (unsigned)tiles_n) * (16 * MT);

  mx_v4f acc[MT][NT];
#pragma unroll
  for (int a = 0; a < MT; a++)
#pragma unroll
    for (int c = 0; c < NT; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[a][c][i] = 0.0f;

  const int per = (p.groups + kSmallWaves - 1) / kSmallWaves;
  const int g_begin = wave * per, g_end = min(p.groups, g_begin + per);
  // rows past the end re-read the last one; what they give is not stored
  const uint8_t *w[NT];
#pragma unroll
  for (int c = 0; c < NT; c++) w[c] = p.weights + (size_t)min(n0 + c * 16 + row, p.N - 1) * p.weights_row_bytes;
  SmallBlock<MX4> wf[D][NT];
  auto load_weights = [&](int g0) {
#pragma unroll
    for (int d = 0; d < D; d++)
      if (g0 + d < g_end) {
#pragma unroll
        for (int c = 0; c < NT; c++) wf[d][c].load(w[c], p.groups, g0 + d, b, 0);
      }
  };
  auto multiply = [&](int d, int a, v4i codes, int byte) {
#pragma unroll
    for (int c = 0; c < NT; c++)
      acc[a][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(wf[d][c].v), fp4_operand(codes),
                                                                   acc[a][c], 4, 4, 0, wf[d][c].s, 0, byte);
  };
  if constexpr (SHARED) {
    extern __shared__ __attribute__((aligned(16))) uint8_t s_rows[];
    const int row_bytes = mx4_shared_row(p.groups), blocks = 4 * p.groups;
    load_weights(g_begin);
    for (int m = 0; m < min(kSharedRows, p.M - m0); m++)
      for (int u = tid; u < blocks; u += kSmallWaves * 64) {
        SmallBlock<IN> x;
        x.load(p.in + (size_t)(m0 + m) * p.in_row_bytes, p.groups, u >> 2, u & 3, K);
        v4i codes;
        int byte;
        x.codes(codes, byte);
        *reinterpret_cast<v4i *>(s_rows + m * row_bytes + u * 16) = codes;
        s_rows[m * row_bytes + blocks * 16 + u] = (uint8_t)byte;
      }
    __syncthreads();
    const uint8_t *mine = s_rows + min(row, min(kSharedRows, p.M - m0) - 1) * row_bytes;
    for (int g0 = g_begin; g0 < g_end; g0 += D) {
      if (g0 != g_begin) load_weights(g0);
#pragma unroll
      for (int d = 0; d < D; d++)
        if (g0 + d < g_end) {
          const int u = (g0 + d) * 4 + b;
          multiply(d, 0, *reinterpret_cast<const v4i *>(mine + u * 16), mine[blocks * 16 + u]);
        }
    }
  } else {
    const uint8_t *x[MT];
#pragma unroll
    for (int a = 0; a < MT; a++) x[a] = p.in + (size_t)min(m0 + a * 16 + row, p.M - 1) * p.in_row_bytes;
    for (int g0 = g_begin; g0 < g_end; g0 += D) {
      SmallBlock<IN> xf[D][MT];
      load_weights(g0);
#pragma unroll
      for (int d = 0; d < D; d++)
        if (g0 + d < g_end) {
#pragma unroll
          for (int a = 0; a < MT; a++) xf[d][a].load(x[a], p.groups, g0 + d, b, K);
        }
#pragma unroll
      for (int d = 0; d < D; d++)
        if (g0 + d < g_end) {
#pragma unroll
          for (int a = 0; a < MT; a++) {
            v4i codes;
            int byte;
            xf[d][a].codes(codes, byte);
            multiply(d, a, codes, byte);
          }
        }
    }
  }
  // register i of a lane: column 4 * (lane / 16) + i, row lane % 16
#pragma unroll
  for (int a = 0; a < MT; a++)
#pragma unroll
    for (int c = 0; c < NT; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) s_part[wave][(a * NT + c) * 4 + i][lane] = acc[a][c][i];
  __syncthreads();
  // a wave finishes 16 rows of all columns at a time
  if (wave < MT) {
    const int a = wave, m = m0 + a * 16 + row;
    float y[NT][4];
#pragma unroll
    for (int c = 0; c < NT; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float t = 0;
#pragma unroll
        for (int k = 0; k < kSmallWaves; k++) t += s_part[k][(a * NT + c) * 4 + i][lane];
        const int n = n0 + c * 16 + 4 * b + i;
        y[c][i] = n < p.N ? t + (p.bias ? p.bias[n] : 0.0f) : 0.0f;
      }
    with_activation(p.act, [&](auto act) {         // (all of them make 0 of 0)
#pragma unroll
      for (int c = 0; c < NT; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) y[c][i] = activate<decltype(act)::value>(y[c][i]);
    });
    uint8_t *out = p.out + (size_t)m * p.out_row_bytes;
    if constexpr (OUT::kSize == 0) {
      static_assert(NT == 2, "a block of columns");
      uint32_t most = 0;
#pragma unroll
      for (int c = 0; c < NT; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) most = max(most, magnitude_bits(y[c][i]));
      most = max_across32(max_across16(most));
      const uint32_t byte = mx4_scale_byte(most);
      const float x8[8] = {y[0][0], y[0][1], y[0][2], y[0][3], y[1][0], y[1][1], y[1][2], y[1][3]};
      const uint32_t codes = mx4_codes8(x8, byte);
      if (m < p.M) {
        uint16_t *at = reinterpret_cast<uint16_t *>(out + n0 / 2 + 2 * b);
        at[0] = (uint16_t)codes;
        at[4] = (uint16_t)(codes >> 16);
        uint8_t *scales = out + (size_t)p.out_groups * kMxGroupBytes;
        if (b == 0) scales[n0 / 32] = (uint8_t)byte;
        // the zeros behind the last group's scales
        else if (n0 / 32 == 4 * p.out_groups - 1 && b <= ((-p.out_groups) & 3))
          reinterpret_cast<uint32_t *>(scales)[p.out_groups + b - 1] = 0;
      }
    } else if (m < p.M) {
      typedef typename OUT::T E;
      typedef E Four __attribute__((ext_vector_type(4)));
      typedef Four Four1 __attribute__((aligned(OUT::kSize)));
#pragma unroll
      for (int c = 0; c < NT; c++) {
        const int n = n0 + c * 16 + 4 * b;
        E *at = reinterpret_cast<E *>(out) + n;
        if (n + 4 <= p.N)
          *reinterpret_cast<Four1 *>(at) = Four{OUT::from(y[c][0]), OUT::from(y[c][1]), OUT::from(y[c][2]), OUT::from(y[c][3])};
        else
          for (int i = 0; i < 4; i++)
            if (n + i < p.N) at[i] = OUT::from(y[c][i]);
      }
    }
  }
}

template <class IN, class OUT, int MT, int NT>
static int mx4_fc_small_launch(const MxFc &p, int K, hipStream_t st) {
  const long long columns = OUT::kSize ? p.N : (long long)p.out_groups * kMxGroup;
  const long long tiles_n = (columns + 16 * NT - 1) / (16 * NT);
  const long long blocks = tiles_n * (((long long)p.M + 16 * MT - 1) / (16 * MT));
  if (blocks > (1 << 22)) return fail(MI355X_ERR_NOT_SUPPORTED, "mx4_fc: %d x %d results", p.M, p.N);
  if constexpr (IN::kSize && MT == 1) {
    if (p.M <= kSharedRows) {
      // (at most 96 KB of values are quantised here: a quarter of that and the pads)
      const size_t lds = (size_t)p.M * mx4_shared_row(p.groups);
      mx4_fc_small_kernel<IN, OUT, MT, NT, true><<<(unsigned)blocks, kSmallWaves * 64, lds, st>>>(p, K, (int)tiles_n);
      return check_launch("mx4_fc");
    }
  }
  mx4_fc_small_kernel<IN, OUT, MT, NT, false><<<(unsigned)blocks, kSmallWaves * 64, 0, st>>>(p, K, (int)tiles_n);
  return check_launch("mx4_fc");
}

} // namespace mi355x

#endif
