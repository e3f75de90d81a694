// Products of microscaled rows over up to 512 columns, with many results: no ring, all of a
// tile's codes and scales are asked for at once and multiplied when they have arrived. A
// float input is quantised on its way into LDS, a thread a block of 32 columns, which saves the
// launch in front and the rows' way through memory.
#ifndef GLOW_MI355X_MX4_SHORT_H
#define GLOW_MI355X_MX4_SHORT_H

#include "mx4_small.h"
#include "mx4_tiles.h"

namespace mi355x {

constexpr int kShortGroups = 4;

template <class OUT, int BN, int BM, int WN, int WM>
constexpr int mx4_short_bias(int groups) {
  typedef MxTile<OUT, BN, BM, WN, WM> T;
  return groups * T::kStep + T::kScales > T::kStaging ? groups * T::kStep + T::kScales : T::kStaging;
}

template <class IN, class OUT, int BN, int BM, int WN, int WM, int BLOCKS>
__global__ __launch_bounds__((BN / WN) * (BM / WM) * 64, BLOCKS *(BN / WN) * (BM / WM) / 4) void mx4_fc_short_kernel(
    MxFc p, int K, int tiles_n, int tiles_m) {
  typedef MxTile<OUT, BN, BM, WN, WM> T;
  constexpr int WAVES = T::kWaves, TN = T::TN, TM = T::TM, THREADS = T::kThreads, kStep = T::kStep;
  constexpr int A_LOADS = BN / 16 / WAVES, B_LOADS = IN::kSize ? 0 : BM / 16 / WAVES;
  static_assert(BN / 16 % WAVES == 0 && BM / 16 % WAVES == 0 && BN % 64 == 0 && BM % 64 == 0, "tile");
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % T::kWavesN, wm = wave / T::kWavesN;
  const int l16 = lane & 15, q = lane >> 4;
  int tm, tn;
  tile_of_block(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN, KT = p.groups;
  int8_t *scales = lds + KT * kStep;

  // rows past the end re-read the last one; their results are not used
  auto weight_row = [&](int s) {
    return p.weights + (size_t)min(n0 + mx4_weight_column<T::S>(s), p.N - 1) * p.weights_row_bytes;
  };
  auto input_row = [&](int s) { return p.in + (size_t)min(m0 + s, p.M - 1) * p.in_row_bytes; };
  float bias = 0.0f;
  if (tid < BN && p.bias && n0 + tid < p.N) bias = p.bias[n0 + tid];

  if (KT > 0) {
    const uint32_t lds0 = lds_address(lds);
    // (a row's end is rounded up to 16 bytes: four steps' scales are there in any case)
    constexpr int kScaleRows = IN::kSize ? BN : BN + BM;
    for (int s0 = wave * 64; s0 < kScaleRows; s0 += WAVES * 64) {
      const int s = s0 + lane;
      dma16((s < BN ? weight_row(s) : input_row(s - BN)) + (size_t)KT * kMxGroupBytes,
            lds0 + (uint32_t)(KT * kStep) + (uint32_t)s0 * 16);
    }
    const int kc = ((lane & 3) ^ mx4_swizzle(lane >> 2)) * 16;
#pragma unroll
    for (int i = 0; i < A_LOADS + B_LOADS; i++) {
      const int g = (i < A_LOADS ? i : i - A_LOADS) * WAVES + wave, s = g * 16 + (lane >> 2);
      const uint8_t *src = (i < A_LOADS ? weight_row(s) : input_row(s)) + kc;
      const uint32_t dst = lds0 + (i < A_LOADS ? 0 : BN * 64) + g * 1024;
      for (int t = 0; t < KT; t++) dma16(src + t * kMxGroupBytes, dst + (uint32_t)(t * kStep));
    }
    if constexpr (IN::kSize != 0) {
      // block u of the tile: row u / 4, block u % 4 of a step; two steps' values at a time
      constexpr int PER = BM * 4 / THREADS;
      for (int t = 0; t < KT; t += 2) {
        SmallBlock<IN> x[2][PER];
#pragma unroll
        for (int d = 0; d < 2; d++)
          if (t + d < KT)
#pragma unroll
            for (int i = 0; i < PER; i++) {
              const int u = i * THREADS + tid;
              x[d][i].load(input_row(u >> 2), KT, t + d, u & 3, K);
            }
#pragma unroll
        for (int d = 0; d < 2; d++)
          if (t + d < KT)
#pragma unroll
            for (int i = 0; i < PER; i++) {
              const int u = i * THREADS + tid, s = u >> 2, b = u & 3;
              v4i codes;
              int byte;
              x[d][i].codes(codes, byte);
              *reinterpret_cast<v4i *>(lds + (t + d) * kStep + (BN + s) * 64 + ((b ^ mx4_swizzle(s)) << 4)) = codes;
              scales[(BN + s) * 16 + (t + d) * 4 + b] = (int8_t)byte;
            }
      }
    }
    dma_wait<0>();
    __syncthreads();
  }

  mx_v4f acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; i++)
#pragma unroll
    for (int j = 0; j < TM; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) acc[i][j][r] = 0.0f;
  const int frag_off = l16 * 64 + ((q ^ mx4_swizzle(l16)) << 4), byte_off = l16 * 16 + q;
  for (int t = 0; t < KT; t++) {
    v4i frag[TN + TM];
    int scale[TN + TM];
#pragma unroll
    for (int f = 0; f < TN + TM; f++) {
      const int row = f < TN ? wn * WN + f * 16 : BN + wm * WM + (f - TN) * 16;
      frag[f] = *reinterpret_cast<const v4i *>(lds + t * kStep + row * 64 + frag_off);
      scale[f] = reinterpret_cast<const uint8_t *>(scales)[row * 16 + t * 4 + byte_off];
    }
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
      for (int j = 0; j < TM; j++)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(frag[i]), fp4_operand(frag[TN + j]),
                                                                     acc[i][j], 4, 4, 0, scale[i], 0, scale[TN + j]);
  }
  __syncthreads();
  mx4_tile_results<OUT, BN, BM, WN, WM>(acc, p, lds,
                                        reinterpret_cast<float *>(lds + mx4_short_bias<OUT, BN, BM, WN, WM>(KT)), bias,
                                        m0, n0);
}

template <class IN, class OUT, int BN, int BM, int WN, int WM, int BLOCKS>
static int mx4_fc_short_launch(const MxFc &p, int K, hipStream_t st) {
  auto kern = mx4_fc_short_kernel<IN, OUT, BN, BM, WN, WM, BLOCKS>;
  const auto lds = [](int groups) { return (size_t)mx4_short_bias<OUT, BN, BM, WN, WM>(groups) + BN * 4; };
  const long long columns = OUT::kSize ? p.N : (long long)p.out_groups * kMxGroup;
  const long long tiles_n = (columns + BN - 1) / BN, tiles_m = ((long long)p.M + BM - 1) / BM;
  constexpr int THREADS = MxTile<OUT, BN, BM, WN, WM>::kThreads;
  if (tiles_n * tiles_m > (1 << 22))
    return fail(MI355X_ERR_NOT_SUPPORTED, "mx4_fc: %d x %d results", p.M, p.N);
  static std::atomic<uint64_t> attr_set{0};
  if (int rc = set_lds_attr(kern, lds(kShortGroups), attr_set)) return rc;
  kern<<<(unsigned)(tiles_n * tiles_m), THREADS, lds(p.groups), st>>>(p, K, (int)tiles_n, (int)tiles_m);
  return check_launch("mx4_fc");
}

} // namespace mi355x

#endif
