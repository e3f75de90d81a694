// Products of microscaled rows with many results: output tiles of 64x64 to 256x256, K in
// steps of 128 columns through a ring in LDS.
//
// A step is 64 bytes of codes of every row of both operands, moved from global memory
// straight into LDS, and two slices of 64 columns for the matrix cores, whose lanes read one
// block (16 bytes) each. Scale bytes travel apart from the codes, with every fourth step: 16
// bytes of a row are four steps' words. Weights are the first operand and their rows are permuted on the way
// into LDS: a lane ends with sixteen neighbouring columns of one output row.
#ifndef GLOW_MI355X_MX4_TILES_H
#define GLOW_MI355X_MX4_TILES_H

#include "gemm_i8.h"
#include "mx4.h"

namespace mi355x {

typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef float mx_v16f __attribute__((ext_vector_type(16)));

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

template <class OUT, int BN, int BM, int WN, int WM, int STAGES>
struct MxTile {
  static constexpr int kWavesN = BN / WN, kWaves = (BN / WN) * (BM / WM);
  static constexpr int kStage = (BN + BM) * 64;                       // a step's codes
  static constexpr int kRing = STAGES * kStage;
  static constexpr int kScales = (BN + BM) * 16;                      // four steps' scales
  // a wave's results on their way out: 32 rows, 16 bytes apart from a whole number of banks
  static constexpr int kOutRow = WN * OUT::kSize + 16;
  static constexpr int kStaging = OUT::kSize ? kWaves * 32 * kOutRow : 0;
  static constexpr int kMain = kRing + 2 * kScales;
  static constexpr int kBias = kMain > kStaging ? kMain : kStaging;   // where the biases lie
  static constexpr size_t kLds = (size_t)kBias + BN * 4;
};

// The end of a tile: biases, activation, and the results on their way out. `bias` is column
// tid's; a wave stages its results in LDS where nothing that is still needed lies.
template <class OUT, int BN, int BM, int WN, int WM>
__device__ __forceinline__ void mx4_tile_results(mx_v16f (&acc)[WN / 32][WM / 32], const MxFc &p, int8_t *lds,
                                                 float *s_bias, float bias, int m0, int n0) {
  constexpr int TN = WN / 32, TM = WM / 32, kWavesN = BN / WN, kOutRow = WN * OUT::kSize + 16;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % kWavesN, wm = wave / kWavesN;
  const int l32 = lane & 31, half = lane >> 5;
  if (tid < BN) s_bias[tid] = bias;
  __syncthreads();

  const int nw = n0 + wn * WN;                     // first column of this wave
  with_activation(p.act, [&](auto act) {
  auto value = [&](int i, int j, int r) {          // column i * 32 + 16 * half + r of row j * 32 + l32
    return activate<decltype(act)::value>(acc[i][j][r] + s_bias[wn * WN + i * 32 + 16 * half + r]);
  };
  if constexpr (OUT::kSize == 0) {
    const int blocks = 4 * p.out_groups;
#pragma unroll
    for (int j = 0; j < TM; j++) {
      const int m = m0 + wm * WM + j * 32 + l32;
      uint8_t *row = p.out + (size_t)m * p.out_row_bytes;
      uint32_t bytes = 0;
#pragma unroll
      for (int i = 0; i < TN; i++) {
        float x[2][8];
        uint32_t most = 0;
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const float y = value(i, j, r);
          x[r >> 3][r & 7] = nw + i * 32 + 16 * half + r < p.N ? y : 0.0f;
          most = max(most, magnitude_bits(x[r >> 3][r & 7]));
        }
        most = max_across32(most);
        const uint32_t byte = mx4_scale_byte(most);
        bytes |= byte << (8 * i);
        const uint32_t lo = mx4_codes8(x[0], byte), hi = mx4_codes8(x[1], byte);
        if (m < p.M && nw / 32 + i < blocks)
          *reinterpret_cast<uint2 *>(row + nw / 2 + i * 16 + 8 * half) = make_uint2(lo, hi);
      }
      // (a wave's columns are whole groups, or a part of one: all of its blocks exist or none)
      uint8_t *scales = row + (size_t)p.out_groups * kMxGroupBytes;
      if (m < p.M && half == 0 && nw / 32 < blocks) {
        if constexpr (TN == 4) *reinterpret_cast<uint32_t *>(scales + nw / 32) = bytes;
        else if constexpr (TN == 2) *reinterpret_cast<uint16_t *>(scales + nw / 32) = (uint16_t)bytes;
        else scales[nw / 32] = (uint8_t)bytes;
      }
      // the zeros behind the last group's scales
      if (m < p.M && half == 1 && nw / 32 <= blocks - 1 && blocks - 1 < nw / 32 + TN)
        for (int w = 0; w < ((-p.out_groups) & 3); w++) reinterpret_cast<uint32_t *>(scales)[p.out_groups + w] = 0;
    }
  } else {
    // through LDS: a lane's sixteen columns are a piece of a line, a row's columns of a wave whole ones
    typedef typename OUT::T E;
    constexpr int PER = 16 / OUT::kSize, LPR = WN / PER;   // columns of a store, lanes of a row
    typedef E Chunk __attribute__((ext_vector_type(PER)));
    typedef Chunk Chunk1 __attribute__((aligned(OUT::kSize)));
    int8_t *stage = lds + wave * 32 * kOutRow;
#pragma unroll
    for (int j = 0; j < TM; j++) {
#pragma unroll
      for (int i = 0; i < TN; i++)
#pragma unroll
        for (int q = 0; q < 16 / PER; q++) {
          Chunk c;
#pragma unroll
          for (int r = 0; r < PER; r++) c[r] = OUT::from(value(i, j, q * PER + r));
          *reinterpret_cast<Chunk *>(stage + l32 * kOutRow + (i * 32 + 16 * half + q * PER) * OUT::kSize) = c;
        }
      wave_fence();
      const int n = nw + (lane % LPR) * PER;
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += 64 / LPR) {
        const int r = r0 + lane / LPR, m = m0 + wm * WM + j * 32 + r;
        const Chunk c = *reinterpret_cast<const Chunk *>(stage + r * kOutRow + (lane % LPR) * 16);
        if (m < p.M && n < p.N) {
          E *at = reinterpret_cast<E *>(p.out + (size_t)m * p.out_row_bytes) + n;
          if (n + PER <= p.N) *reinterpret_cast<Chunk1 *>(at) = c;
          else
            for (int e = 0; e < PER; e++)
              if (n + e < p.N) at[e] = c[e];
        }
      }
      wave_fence();
    }
  }
  });
}

template <class OUT, int BN, int BM, int WN, int WM, int STAGES, int BLOCKS>
__global__ __launch_bounds__((BN / WN) * (BM / WM) * 64, BLOCKS *(BN / WN) * (BM / WM) / 4) void mx4_fc_tile_kernel(
    MxFc p, int tiles_n, int tiles_m) {
  typedef MxTile<OUT, BN, BM, WN, WM, STAGES> T;
  constexpr int WAVES = T::kWaves, TN = WN / 32, TM = WM / 32;
  constexpr int A_LOADS = BN / 16 / WAVES, B_LOADS = BM / 16 / WAVES;  // 16 rows an instruction
  constexpr int LOADS = A_LOADS + B_LOADS;
  constexpr int ROWS = (BN + BM) / WAVES;                              // whose scales a wave moves
  constexpr int SLOADS = (ROWS + 63) / 64, SLANES = ROWS < 64 ? ROWS : 64;
  static_assert(BN / 16 % WAVES == 0 && BM / 16 % WAVES == 0 && SLOADS * SLANES == ROWS, "tile");
  // (with more slots a group's scales would be asked for while others read the ones they replace)
  static_assert((STAGES == 3 || STAGES == 4) && (STAGES - 1) * LOADS < 64, "ring depth");

  extern __shared__ __attribute__((aligned(16))) int8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % T::kWavesN, wm = wave / T::kWavesN;
  const int l32 = lane & 31, half = lane >> 5;

  int tm, tn;
  tile_of_block(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int KT = p.groups;

  // slot s of the weights' part of a ring slot holds this row; rows past the end re-read the
  // last one, and their results are not used
  auto weight_row = [&](int s) { return p.weights + (size_t)min(n0 + (s & ~31) + perm_row16(s & 31), p.N - 1) * p.weights_row_bytes; };
  auto input_row = [&](int s) { return p.in + (size_t)min(m0 + s, p.M - 1) * p.in_row_bytes; };

  float bias = 0.0f;
  if (tid < BN && p.bias && n0 + tid < p.N) bias = p.bias[n0 + tid];

  // lane i of a load owns row i / 4 of its sixteen and the LDS chunk i % 4 of it; the chunk
  // stored there is swizzled, so that fragment reads meet no bank twice
  const int kc = ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
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
  // load x of a step, to ring offset `ring`; behind the last one of every fourth step the scales of
  // the four steps that come after its own
  auto issue = [&](int step, uint32_t ring, int x) {
    dma16(src[x] + (size_t)min(step, KT - 1) * 64, ring, dst[x]);
    if (x == LOADS - 1 && (step & 3) == 0) issue_scales((step >> 2) + 1);
  };
  constexpr int H0 = LOADS / 2;
  if (KT > 0) {
    issue_scales(0);
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++)
#pragma unroll
      for (int x = 0; x < LOADS; x++) issue(s, s * T::kStage, x);
#pragma unroll
    for (int x = 0; x < H0; x++) issue(STAGES - 1, (STAGES - 1) * T::kStage, x);
  }

  mx_v16f acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; i++)
#pragma unroll
    for (int j = 0; j < TM; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;

  const int swz = (lane >> 2) & 3;
  int frag_off[2];
#pragma unroll
  for (int ks = 0; ks < 2; ks++) frag_off[ks] = l32 * 64 + (((ks * 2 + half) ^ swz) << 4);
  const int a_base = wn * WN * 64, b_base = BN * 64 + wm * WM * 64;
  v4i frag[2][TN + TM];
  auto read_frag = [&](const int8_t *stage, int ks, int f) {
    const int8_t *at = f < TN ? stage + a_base + f * 2048 : stage + b_base + (f - TN) * 2048;
    frag[ks][f] = *reinterpret_cast<const v4i *>(at + frag_off[ks]);
  };
  // four steps' scale words of the rows a lane feeds, the current step's first
  v4i quad[TN + TM];
  int scale[TN + TM];
  auto read_quads = [&](int group) {
    const int8_t *at = lds + T::kRing + (group & 1) * T::kScales + l32 * 16;
#pragma unroll
    for (int f = 0; f < TN + TM; f++)
      quad[f] = *reinterpret_cast<const v4i *>(at + (f < TN ? wn * WN + f * 32 : BN + wm * WM + (f - TN) * 32) * 16);
  };
  auto take_scales = [&]() {
    // a lane of the upper half feeds blocks 1 and 3 of a step: bytes 0 and 2 from here
#pragma unroll
    for (int f = 0; f < TN + TM; f++) {
      scale[f] = (int)((uint32_t)quad[f][0] >> (8 * half));
      quad[f] = v4i{quad[f][1], quad[f][2], quad[f][3], 0};
    }
  };
  constexpr int MFMAS = TN * TM, FRAGS = TN + TM;
  // the matrix instructions of a slice, memory operations of the next one spread between them
  auto multiply = [&](auto ks, auto &&between) {
    constexpr int KS = decltype(ks)::value;
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
      for (int j = 0; j < TM; j++) {
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
            fp4_operand(frag[KS][i]), fp4_operand(frag[KS][TN + j]), acc[i][j], 4, 4, 2 * KS, scale[i], 2 * KS,
            scale[TN + j]);
        __builtin_amdgcn_sched_barrier(0);
        between(i * TM + j);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  auto frags_in_slot = [&](int t, const int8_t *stage, int ks) {
#pragma unroll
    for (int f = t * FRAGS / MFMAS; f < (t + 1) * FRAGS / MFMAS; f++) read_frag(stage, ks, f);
  };
  auto loads_in_slot = [&](int t, int step, uint32_t ring, int from, int n) {
#pragma unroll
    for (int x = 0; x < n; x++)
      if (min(MFMAS - 1, (2 * x + 1) * MFMAS / (2 * n)) == t) issue(step, ring, from + x);
  };

  if (KT > 0) {
    // Step 0 and the first scales have landed. (The counts leave out that scales may be among the
    // loads in flight: one of a step that need not have landed is waited for then.)
    dma_wait<(STAGES - 2) * LOADS + H0>();
    __syncthreads();
    read_quads(0);
#pragma unroll
    for (int f = 0; f < FRAGS; f++) read_frag(lds, 0, f);
    uint32_t ring_cur = 0, ring_prev = (STAGES - 1) * T::kStage;
    for (int kt = 0; kt < KT; kt++) {
      const uint32_t ring_next = ring_cur + T::kStage == T::kRing ? 0u : ring_cur + T::kStage;
      const int8_t *cur = lds + ring_cur, *nxt = lds + ring_next;
      take_scales();
      multiply(std::integral_constant<int, 0>(), [&](int t) {
        frags_in_slot(t, cur, 1);
        loads_in_slot(t, kt + STAGES - 1, ring_prev, H0, LOADS - H0);
      });
      // step kt + 1 has landed once only the steps behind it are pending; past the barrier every
      // wave holds step kt in registers, so that its slot is free
      dma_wait<(STAGES - 2) * LOADS>();
      __syncthreads();
      if ((kt & 3) == 3) read_quads((kt >> 2) + 1);
      multiply(std::integral_constant<int, 1>(), [&](int t) {
        frags_in_slot(t, nxt, 0);
        loads_in_slot(t, kt + STAGES, ring_cur, 0, H0);
      });
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
  typedef MxTile<OUT, BN, BM, WN, WM, STAGES> T;
  auto kern = mx4_fc_tile_kernel<OUT, BN, BM, WN, WM, STAGES, BLOCKS>;
  static std::atomic<uint64_t> attr_set{0};
  if (int rc = set_lds_attr(kern, T::kLds, attr_set)) return rc;
  // a microscaled result has whole groups of columns, the ones past N zeros
  const long long columns = OUT::kSize ? p.N : (long long)p.out_groups * kMxGroup;
  const long long tiles_n = (columns + BN - 1) / BN, tiles_m = ((long long)p.M + BM - 1) / BM;
  if (tiles_n * tiles_m > (1 << 22))
    return fail(MI355X_ERR_NOT_SUPPORTED, "mx4_fc: %d x %d results", p.M, p.N);
  kern<<<(unsigned)(tiles_n * tiles_m), T::kWaves * 64, T::kLds, st>>>(p, (int)tiles_n, (int)tiles_m);
  return check_launch("mx4_fc");
}

} // namespace mi355x

#endif
