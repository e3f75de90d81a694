// Products of microscaled rows with many results: output tiles of 64x64 to 256x256, K in
// steps of 128 columns through a ring in LDS.
//
// A step is 64 bytes of codes of every row of both operands, moved from global memory
// straight into LDS, and one scaled matrix instruction of 16x16 results for each pair of
// sixteen rows, whose lanes read one block (16 bytes) each. Scale bytes travel apart from the
// codes, with every fourth step: 16 bytes of a row are four steps' words. Weights are the
// first operand and their rows are permuted on the way into LDS: a lane ends with sixteen
// neighbouring columns of one output row (eight, where a wave has 32).
//
// 8192 x 4096 x 4096 of random codes to bf16: 80 us, 75 to 87 by card and load, 3.4 PFLOP/s. The
// matrix cores are busy for 47 % of the cycles. Random codes draw so much power that the
// instructions alone, from registers, reach 6.5 PFLOP/s in their 32x32 form and 7.5 in this one
// (zeros: 9.5); a step of a 256x256 tile takes 0.95 us where they need 0.46, and 0.8 without
// its loads; and the ends of a tile cost 8 us, where all CUs write (67 MB in all) or wait together.
// What gave most on the way, about 5 % each: the activation chosen once, 16x16 instructions, chunks
// placed so that reads meet no bank twice (the scales' single bytes still meet one another).
#ifndef GLOW_MI355X_MX4_TILES_H
#define GLOW_MI355X_MX4_TILES_H

#include "gemm_i8.h"
#include "mx4.h"

namespace mi355x {

typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef float mx_v4f __attribute__((ext_vector_type(4)));

__device__ __forceinline__ mx_v8i fp4_operand(v4i v) { return mx_v8i{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

struct MxFc {
  uint8_t *out;
  size_t out_row_bytes;
  const uint8_t *in, *weights;
  size_t in_row_bytes, weights_row_bytes;
  const float *bias;
  int M, N, groups;        // groups of 128 columns of K
  int out_groups;          // of a microscaled result's row
  int act;
};

// The place of weight rows in a tile's LDS: subtile t of the S that a group of 16 S columns has holds
// in its row 4 q + i the group's column 4 S q + 4 t + i. A matrix instruction gives a lane rows 4 q .. 4
// q + 3 (q = lane / 16) of each subtile: with these, 4 S neighbouring columns.
template <int S> __device__ __forceinline__ int mx4_weight_column(int slot) {
  const int in = slot & (16 * S - 1);
  return (slot - in) + 4 * S * ((in >> 2) & 3) + 4 * (in >> 4) + (in & 3);
}

// Chunk k of a row lies at k ^ this in LDS. Reads of sixteen bytes are served sixteen lanes at a time,
// 0-3, 12-15, 20-23 and 24-27 first: rows 0-3 and 12-15 of chunk 0, 4-11 of chunk 1. With these
// they meet no bank twice.
__device__ __forceinline__ int mx4_swizzle(int row) { return -(row >> 2) & 3; }

template <class OUT, int BN, int BM, int WN, int WM>
struct MxTile {
  static constexpr int kWavesN = BN / WN, kWaves = (BN / WN) * (BM / WM), kThreads = kWaves * 64;
  static constexpr int TN = WN / 16, TM = WM / 16;
  static constexpr int S = TN < 4 ? TN : 4;                 // subtiles of a group of columns
  static constexpr int kStep = (BN + BM) * 64;              // a step's codes
  static constexpr int kScales = (BN + BM) * 16;            // four steps' scales
  // a wave's results on their way out: 16 rows, 16 bytes apart from a whole number of banks
  static constexpr int kOutRow = WN * OUT::kSize + 16;
  static constexpr int kStaging = OUT::kSize ? kWaves * 16 * kOutRow : 0;
  static_assert(TN % S == 0 && S % 2 == 0 && kThreads >= BN, "tile");
};

// The end of a tile: biases, activation, and the results on their way out. `bias` is column
// tid's; a wave stages its results in LDS where nothing that is still needed lies.
template <class OUT, int BN, int BM, int WN, int WM>
__device__ __forceinline__ void mx4_tile_results(mx_v4f (&acc)[WN / 16][WM / 16], const MxFc &p, int8_t *lds,
                                                 float *s_bias, float bias, int m0, int n0) {
  typedef MxTile<OUT, BN, BM, WN, WM> T;
  constexpr int S = T::S, GROUPS = T::TN / S, COLS = 4 * S;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % T::kWavesN, wm = wave / T::kWavesN;
  const int l16 = lane & 15, q = lane >> 4;
  if (tid < BN) s_bias[tid] = bias;
  __syncthreads();

  const int nw = n0 + wn * WN;                     // first column of this wave
  with_activation(p.act, [&](auto act) {
    // column g * 16 S + 4 S q + r of row j * 16 + l16
    auto value = [&](int g, int j, int r) {
      return activate<decltype(act)::value>(acc[g * S + r / 4][j][r % 4] + s_bias[wn * WN + g * 16 * S + COLS * q + r]);
    };
    if constexpr (OUT::kSize == 0) {
      const int blocks = 4 * p.out_groups;
#pragma unroll
      for (int j = 0; j < T::TM; j++) {
        const int m = m0 + wm * WM + j * 16 + l16;
        uint8_t *row = p.out + (size_t)m * p.out_row_bytes;
        uint8_t *scales = row + (size_t)p.out_groups * kMxGroupBytes;
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
          float x[COLS / 8][8];
          uint32_t most = 0;
          const int n = nw + g * 16 * S + COLS * q;
#pragma unroll
          for (int r = 0; r < COLS; r++) {
            const float y = value(g, j, r);
            x[r / 8][r % 8] = n + r < p.N ? y : 0.0f;
            most = max(most, magnitude_bits(x[r / 8][r % 8]));
          }
          // a block of 32 columns is two lanes' or four lanes'
          most = max_across16(most);
          if constexpr (S == 2) most = max_across32(most);
          const uint32_t byte = mx4_scale_byte(most);
          if (m < p.M && n / 32 < blocks) {
            if constexpr (S == 4) {
              *reinterpret_cast<uint2 *>(row + n / 2) = make_uint2(mx4_codes8(x[0], byte), mx4_codes8(x[1], byte));
            } else {
              *reinterpret_cast<uint32_t *>(row + n / 2) = mx4_codes8(x[0], byte);
            }
            if (n % 32 == 0) scales[n / 32] = (uint8_t)byte;
          }
        }
        // the zeros behind the last group's scales
        if (m < p.M && nw / 32 <= blocks - 1 && blocks - 1 < (nw + WN) / 32 && q < ((-p.out_groups) & 3))
          reinterpret_cast<uint32_t *>(scales)[p.out_groups + q] = 0;
      }
    } else {
      // through LDS: a lane's columns are a piece of a line, a row's columns of a wave whole ones
      typedef typename OUT::T E;
      constexpr int PER = 16 / OUT::kSize, LPR = WN / PER;   // columns of a store, lanes of a row
      typedef E Chunk __attribute__((ext_vector_type(PER)));
      typedef Chunk Chunk1 __attribute__((aligned(OUT::kSize)));
      int8_t *stage = lds + wave * 16 * T::kOutRow;
#pragma unroll
      for (int j = 0; j < T::TM; j++) {
#pragma unroll
        for (int g = 0; g < GROUPS; g++)
#pragma unroll
          for (int k = 0; k < COLS / PER; k++) {
            Chunk c;
#pragma unroll
            for (int r = 0; r < PER; r++) c[r] = OUT::from(value(g, j, k * PER + r));
            *reinterpret_cast<Chunk *>(stage + l16 * T::kOutRow + (g * 16 * S + COLS * q + k * PER) * OUT::kSize) = c;
          }
        wave_fence();
        const int n = nw + (lane % LPR) * PER;
        constexpr int kPass = 64 / LPR < 16 ? 64 / LPR : 16;
#pragma unroll
        for (int r0 = 0; r0 < 16; r0 += kPass) {
          const int r = r0 + lane / LPR, m = m0 + wm * WM + j * 16 + r;
          if (r < 16 && m < p.M && n < p.N) {
            const Chunk c = *reinterpret_cast<const Chunk *>(stage + r * T::kOutRow + (lane % LPR) * 16);
            E *at = reinterpret_cast<E *>(p.out + (size_t)m * p.out_row_bytes) + n;
            if (n + PER <= p.N) *reinterpret_cast<Chunk1 *>(at) = c;
            else
#pragma unroll
              for (int e = 0; e < PER; e++)
                if (n + e < p.N) at[e] = c[e];
          }
        }
        wave_fence();
      }
    }
  });
}

template <class OUT, int BN, int BM, int WN, int WM, int STAGES>
struct MxRing : MxTile<OUT, BN, BM, WN, WM> {
  typedef MxTile<OUT, BN, BM, WN, WM> T;
  static constexpr int kRing = STAGES * T::kStep, kMain = kRing + 2 * T::kScales;
  static constexpr int kBias = kMain > T::kStaging ? kMain : T::kStaging;   // where the biases lie
  static constexpr size_t kLds = (size_t)kBias + BN * 4;
};

template <class OUT, int BN, int BM, int WN, int WM, int STAGES, int BLOCKS>
__global__ __launch_bounds__((BN / WN) * (BM / WM) * 64, BLOCKS *(BN / WN) * (BM / WM) / 4) void mx4_fc_tile_kernel(
    MxFc p, int tiles_n, int tiles_m) {
  typedef MxRing<OUT, BN, BM, WN, WM, STAGES> T;
  constexpr int WAVES = T::kWaves, TN = T::TN, TM = T::TM;
  constexpr int A_LOADS = BN / 16 / WAVES, B_LOADS = BM / 16 / WAVES;  // 16 rows an instruction
  constexpr int LOADS = A_LOADS + B_LOADS;
  constexpr int ROWS = (BN + BM) / WAVES;                              // whose scales a wave moves
  constexpr int SLOADS = (ROWS + 63) / 64, SLANES = ROWS < 64 ? ROWS : 64;
  static_assert(BN / 16 % WAVES == 0 && BM / 16 % WAVES == 0 && SLOADS * SLANES == ROWS, "tile");
  // (with another number of slots scales would be asked for while others read the ones they replace)
  static_assert(STAGES == 4 && (STAGES - 1) * LOADS + SLOADS < 64, "ring depth");

  extern __shared__ __attribute__((aligned(16))) int8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % T::kWavesN, wm = wave / T::kWavesN;
  const int l16 = lane & 15, q = lane >> 4;

  int tm, tn;
  tile_of_block(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int KT = p.groups;

  // rows past the end re-read the last one, and their results are not used
  auto weight_row = [&](int s) {
    return p.weights + (size_t)min(n0 + mx4_weight_column<T::S>(s), p.N - 1) * p.weights_row_bytes;
  };
  auto input_row = [&](int s) { return p.in + (size_t)min(m0 + s, p.M - 1) * p.in_row_bytes; };

  float bias = 0.0f;
  if (tid < BN && p.bias && n0 + tid < p.N) bias = p.bias[n0 + tid];

  // lane i of a load owns row i / 4 of its sixteen and the LDS chunk i % 4 of it
  const int kc = ((lane & 3) ^ mx4_swizzle(lane >> 2)) * 16;
  const uint32_t lds0 = lds_address(lds);
  const uint8_t *src[LOADS], *scale_src[SLOADS];
  uint32_t dst[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; i++) {
    const int g = (i < A_LOADS ? i : i - A_LOADS) * WAVES + wave, s = g * 16 + (lane >> 2);
    src[i] = (i < A_LOADS ? weight_row(s) : input_row(s)) + kc;
    dst[i] = lds0 + (i < A_LOADS ? 0 : BN * 64) + g * 1024;
  }
#pragma unroll
  for (int i = 0; i < SLOADS; i++) {
    const int s = wave * ROWS + i * 64 + (lane & (SLANES - 1));
    scale_src[i] = (s < BN ? weight_row(s) : input_row(s - BN)) + (size_t)KT * kMxGroupBytes;
  }
  const uint32_t scale_dst = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + T::kRing + wave * ROWS * 16));
  // the scales of steps 4 * group and on
  const int last_group = (KT - 1) >> 2;
  auto issue_scales = [&](int group) {
    const uint32_t slot = (uint32_t)(group & 1) * T::kScales;
    const int at = min(group, last_group) * 16;
#pragma unroll
    for (int i = 0; i < SLOADS; i++)
      if (SLANES == 64 || lane < SLANES) dma16(scale_src[i] + at, slot, scale_dst + i * 1024);
  };
  // Load x of a step, to ring offset `ring`; behind the last one of every fourth step the scales of
  // the four steps that follow: step 4 g + 3 is asked for while step 4 g is multiplied, when every wave
  // has read the last of the scales that these replace, those of steps up to 4 g - 1.
  auto issue = [&](int step, uint32_t ring, int x) {
    dma16(src[x] + (size_t)min(step, KT - 1) * 64, ring, dst[x]);
    if (x == LOADS - 1 && (step & 3) == 3) issue_scales((step >> 2) + 1);
  };
  constexpr int H0 = LOADS / 2;
  if (KT > 0) {
    issue_scales(0);
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++)
#pragma unroll
      for (int x = 0; x < LOADS; x++) issue(s, s * T::kStep, x);
#pragma unroll
    for (int x = 0; x < H0; x++) issue(STAGES - 1, (STAGES - 1) * T::kStep, x);
  }

  mx_v4f acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; i++)
#pragma unroll
    for (int j = 0; j < TM; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) acc[i][j][r] = 0.0f;

  // A lane reads block q of row l16 of a subtile and its scale byte. The weights' fragments are used
  // row by row: those of the first half are replaced during the second, the others during the
  // next step's first half; the input's next ones wait in registers of their own. (Two bodies that
  // swap the two sets would save the moves, but the loop's two exits make copies of all results.)
  const int frag_off = l16 * 64 + ((q ^ mx4_swizzle(l16)) << 4), byte_off = l16 * 16 + q;
  v4i wf[TN], xf[TM], xn[TM];
  int ws[TN], xs[TM], xsn[TM];
  auto read_weights = [&](const int8_t *stage, const int8_t *scales, int i) {
    wf[i] = *reinterpret_cast<const v4i *>(stage + (wn * WN + i * 16) * 64 + frag_off);
    ws[i] = reinterpret_cast<const uint8_t *>(scales)[(wn * WN + i * 16) * 16 + byte_off];
  };
  auto read_input = [&](const int8_t *stage, const int8_t *scales, int j) {
    xn[j] = *reinterpret_cast<const v4i *>(stage + (BN + wm * WM + j * 16) * 64 + frag_off);
    xsn[j] = reinterpret_cast<const uint8_t *>(scales)[(BN + wm * WM + j * 16) * 16 + byte_off];
  };
  auto scales_of = [&](int step) {
    return lds + T::kRing + ((step >> 2) & 1) * T::kScales + (step & 3) * 4;
  };
  constexpr int HALF = TN / 2, MFMAS = HALF * TM;
  // half a step's matrix instructions, memory operations spread between them: a wave issues in
  // order, so that a burst of them would hold back the instructions behind it
  auto multiply = [&](auto half, int reads, auto &&read, int loads, auto &&load) {
    constexpr int I0 = decltype(half)::value * HALF;
#pragma unroll
    for (int i = 0; i < HALF; i++)
#pragma unroll
      for (int j = 0; j < TM; j++) {
        const int t = i * TM + j;
        acc[I0 + i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            fp4_operand(wf[I0 + i]), fp4_operand(xf[j]), acc[I0 + i][j], 4, 4, 0, ws[I0 + i], 0, xs[j]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = t * reads / MFMAS; f < (t + 1) * reads / MFMAS; f++) read(f);
#pragma unroll
        for (int x = 0; x < loads; x++)
          if (min(MFMAS - 1, (2 * x + 1) * MFMAS / (2 * loads)) == t) load(x);
        __builtin_amdgcn_sched_barrier(0);
      }
  };

  if (KT > 0) {
    // Step 0 and the first scales have landed. (The counts leave out that scales may be among the
    // loads in flight: one of a step that need not have landed is waited for then.)
    dma_wait<(STAGES - 2) * LOADS + H0>();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TM; j++) read_input(lds, scales_of(0), j);
#pragma unroll
    for (int i = 0; i < HALF; i++) read_weights(lds, scales_of(0), i);
    uint32_t ring_cur = 0, ring_prev = (STAGES - 1) * T::kStep;
    for (int kt = 0; kt < KT; kt++) {
      const uint32_t ring_next = ring_cur + T::kStep == T::kRing ? 0u : ring_cur + T::kStep;
      const int8_t *cur = lds + ring_cur, *nxt = lds + ring_next;
      const int8_t *cur_scales = scales_of(kt), *nxt_scales = scales_of(kt + 1);
#pragma unroll
      for (int j = 0; j < TM; j++) xf[j] = xn[j], xs[j] = xsn[j];
      multiply(
          std::integral_constant<int, 0>(), HALF, [&](int f) { read_weights(cur, cur_scales, HALF + f); },
          LOADS - H0, [&](int x) { issue(kt + STAGES - 1, ring_prev, H0 + x); });
      // Step kt + 1 has landed once only the steps behind it are pending; past the barrier every
      // wave holds step kt in registers, so that its slot is free.
      dma_wait<(STAGES - 2) * LOADS>();
      __syncthreads();
      // (what is read past the last step is not used)
      multiply(
          std::integral_constant<int, 1>(), TM + HALF,
          [&](int f) {
            if (f < TM) read_input(nxt, nxt_scales, f);
            else read_weights(nxt, nxt_scales, f - TM);
          },
          H0, [&](int x) { issue(kt + STAGES, ring_cur, x); });
      ring_prev = ring_cur;
      ring_cur = ring_next;
    }
  }
  dma_wait<0>();                                   // the re-reads, before LDS is used again
  __syncthreads();
  mx4_tile_results<OUT, BN, BM, WN, WM>(acc, p, lds, reinterpret_cast<float *>(lds + T::kBias), bias, m0, n0);
}

template <class OUT, int BN, int BM, int WN, int WM, int STAGES, int BLOCKS>
static int mx4_fc_tile_launch(const MxFc &p, hipStream_t st) {
  typedef MxRing<OUT, BN, BM, WN, WM, STAGES> T;
  auto kern = mx4_fc_tile_kernel<OUT, BN, BM, WN, WM, STAGES, BLOCKS>;
  // a microscaled result has whole groups of columns, the ones past N zeros
  const long long columns = OUT::kSize ? p.N : (long long)p.out_groups * kMxGroup;
  const long long tiles_n = (columns + BN - 1) / BN, tiles_m = ((long long)p.M + BM - 1) / BM;
  if (tiles_n * tiles_m > (1 << 22))
    return fail(MI355X_ERR_NOT_SUPPORTED, "mx4_fc: %d x %d results", p.M, p.N);
  static std::atomic<uint64_t> attr_set{0};
  if (int rc = set_lds_attr(kern, T::kLds, attr_set)) return rc;
  kern<<<(unsigned)(tiles_n * tiles_m), T::kThreads, T::kLds, st>>>(p, (int)tiles_n, (int)tiles_m);
  return check_launch("mx4_fc");
}

} // namespace mi355x

#endif
