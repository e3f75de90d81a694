// Attention over a cache of microscaled rows: few rows of queries a sequence.
#include "mx4_attention.h"
#include "mx4_tiles.h"

namespace mi355x {

// A workgroup has sixteen rows of queries and a share of the tokens that they see, its eight waves every
// eighth step of 32 tokens each; their results meet in LDS, those of several shares in a second launch.
//
// Rows go from memory to LDS without registers between, a step ahead, each wave into a ring of its own that no other
// reads: there is no barrier in the loop. A load moves 16 bytes a lane, 1 KB at once, and a lane picks the piece that
// makes the reads free of bank conflicts: keys' blocks in the order of the products' tiles (mx4_swizzle), token 4 q + i of
// the values in row q + 4 i, so that word i of a lane lies at 64 i + lane. What bounds it: the launch and four rounds of
// dependent loads (one token over 200, 8 heads of 64: 6.8 us), then memory.
template <int D> constexpr int kAtWaves = D == 256 ? 4 : 8;
constexpr int kAtStages = 2;
constexpr int kAtLeast = 8;            // steps of a share at least

template <int D> struct AtRing {
  static constexpr int kTile = 8 * D;                    // bytes of sixteen tokens' codes
  static constexpr int kKeys = 0, kValues = 2 * kTile, kScales = 4 * kTile;
  static constexpr int kWords = D <= 128 ? 1 : 2;        // of a token's scales
  static constexpr int kStage = kScales + 256 * kWords;
  static constexpr int kLoads = 4 * kTile / 1024 + kWords;
};

// Four bytes a lane from global memory straight into LDS at lds_addr + 4 * lane.
__device__ __forceinline__ void dma4(const void *gptr, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds_addr), "v"(gptr) : "memory");
}

// 32 tokens as a wave has them in registers: for each of two tiles a block of a token's keys and its scale byte, and
// then, when these have become weights, of the values eight tokens' words and their scales. (Both at once take 26
// registers, with which four waves no longer share a SIMD: 225 us for 137 over 4 x 115 000 tokens where some went to memory.)
template <int D> struct AtKeys {
  static constexpr int kChunks = (D + 127) / 128;
  at_v4i codes[2][kChunks];
  int scale[2][kChunks];
  int first[2];                        // token of each tile; -1: none
};
template <int D> struct AtWords {
  static constexpr int kChunks = (D + 127) / 128;
  uint32_t codes[kChunks][8], scale[kChunks][8];
};

template <int D> struct AtLoader {
  typedef AtRing<D> R;
  static constexpr int kChunks = (D + 127) / 128, COLS = D == 64 ? 4 : 8;
  const Attention &p;
  const AtTiles tiles;
  const int sequence, begin, stride, end;     // this wave's steps: begin, begin + stride, ..
  const int lane, l16, q;
  uint32_t key_at, value_at[D == 256 ? 2 : 1], scale_at, lds;
  int tile_of;                         // which rows the tile of this lane has, of 32 steps' 64

  __device__ __forceinline__ AtLoader(const Attention &p, const AtTiles &tiles, int sequence, int h, int begin, int stride, int end,
                                      uint32_t lds)
      : p(p), tiles(tiles), sequence(sequence), begin(begin), stride(stride), end(end), lane(threadIdx.x & 63), l16(lane & 15),
        q(lane >> 4), lds(lds) {
    const uint32_t row = (uint32_t)p.c.row_bytes, codes = (uint32_t)h * (D / 2);
    if constexpr (D == 64) {
      // a load has both tiles, rows of two pieces
      key_at = (lane >> 1 & 15) * row + codes + (lane & 1) * 16;
      const int r = lane >> 1 & 15;
      value_at[0] = (4 * (r & 3) + (r >> 2)) * row + codes + (lane & 1) * 16;
      scale_at = l16 * row + ((p.c.scales_at + (uint32_t)h * 2) & ~3u);
    } else {
      // (D = 256: two loads a tile, 128 columns each)
      key_at = (lane >> 2) * row + codes + ((lane & 3) ^ mx4_swizzle(lane >> 2)) * 16;
      const int r = lane >> 2;
      value_at[0] = (4 * (r & 3) + (r >> 2)) * row + codes + (lane & 3) * 16;
      scale_at = l16 * row + p.c.scales_at + (uint32_t)h * (D / 32);
    }
  }
  __device__ __forceinline__ int step_of(int n) const { return min(begin + n * stride, end - 1); }
  // Finds the rows of steps n to n + 31.
  __device__ __forceinline__ void locate(int n) {
    const long long step = begin + (long long)(n + (lane >> 1)) * stride;
    const int u = (int)min(2 * step + (lane & 1), (long long)tiles.all);
    tile_of = step < end && u < tiles.all ? cache_tile(p.c, sequence, (unsigned)tiles.at(u)) : -1;
  }
  // Asks for step n (the last one again where there is none), says which tokens come.
  __device__ __forceinline__ void issue(int n, int (&first)[2]) {
    if ((n & 31) == 0) locate(n);
    const uint8_t *keys[2], *values[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int tile = __builtin_amdgcn_readlane(tile_of, 2 * (n & 31) + k);
      first[k] = tile < 0 ? -1 : tiles.at(2 * step_of(n) + k) * kCacheTile;
      // (a tile that is not there reads the cache's first rows; there is a page)
      const size_t base = (size_t)max(tile, 0) * kCacheTile * p.c.row_bytes;
      keys[k] = p.c.keys + base, values[k] = p.c.values + base;
    }
    const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds + (n % kAtStages) * R::kStage));
    if constexpr (D == 64) {
      const bool second = lane >= 32;
      dma16((second ? keys[1] : keys[0]) + key_at, to + R::kKeys);
      dma16((second ? values[1] : values[0]) + value_at[0], to + R::kValues);
    } else {
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
          dma16(keys[k] + key_at + c * 64, to + R::kKeys + k * R::kTile + c * 1024);
          dma16(values[k] + value_at[0] + c * 64, to + R::kValues + k * R::kTile + c * 1024);
        }
    }
    const uint8_t *scales = q == 0 ? keys[0] : q == 1 ? keys[1] : q == 2 ? values[0] : values[1];
#pragma unroll
    for (int w = 0; w < R::kWords; w++) dma4(scales + scale_at + w * 4, to + R::kScales + w * 256);
  }
  // A step that has landed, from LDS.
  __device__ __forceinline__ void read(AtKeys<D> &s, const uint8_t *ring, int n, int h) const {
    const uint8_t *at = ring + (n % kAtStages) * R::kStage;
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int c = 0; c < kChunks; c++) {
        const uint8_t *scales = at + R::kScales + c * 256;
        if constexpr (D == 64) {
          const int block = q & 1;                  // (lanes q = 2 and 3 have no columns)
          s.codes[k][c] = *reinterpret_cast<const at_v4i *>(at + R::kKeys + k * R::kTile + l16 * 32 + block * 16);
          s.scale[k][c] = scales[(k * 16 + l16) * 4 + (h & 1) * 2 + block];
        } else {
          s.codes[k][c] = *reinterpret_cast<const at_v4i *>(at + R::kKeys + k * R::kTile + c * 1024 + l16 * 64 +
                                                            ((q ^ mx4_swizzle(l16)) << 4));
          s.scale[k][c] = scales[(k * 16 + l16) * 4 + q];
        }
      }
  }
  __device__ __forceinline__ void read(AtWords<D> &s, const uint8_t *ring, int n, int h) const {
    const uint8_t *at = ring + (n % kAtStages) * R::kStage;
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int c = 0; c < kChunks; c++) {
        const at_v4i words = *reinterpret_cast<const at_v4i *>(at + R::kScales + c * 256 + 128 + (k * 16 + 4 * q) * 4);
        const int shift = D == 64 ? 8 * ((h & 1) * 2 + (l16 >> 3)) : 8 * (l16 >> 2);
        const uint8_t *v = at + R::kValues + k * R::kTile + c * 1024;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if constexpr (COLS == 8) s.codes[c][k * 4 + i] = reinterpret_cast<const uint32_t *>(v)[i * 64 + lane];
          else s.codes[c][k * 4 + i] = reinterpret_cast<const uint16_t *>(v)[i * 64 + lane];
          s.scale[c][k * 4 + i] = (uint32_t)words[i] >> shift & 255;
        }
      }
  }
};

template <class E, int D> struct AtState {
  at_v4f acc[D / 16];
  float most, sum;                     // of this lane's query, and its part of the sum
};

// Keys to weights.
template <class E, int D>
__device__ __forceinline__ void at_keys(AtState<E, D> &a, at_v4i (&packed)[AtKind<E>::kP], const AtQueries<E, D> &queries,
                                        const AtKeys<D> &s, const Attention &p, int low, int high, int position) {
  constexpr int kChunks = (D + 127) / 128;
  const int lane = threadIdx.x & 63, q = lane >> 4;
  float score[8];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    at_v4f r = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      at_v4i codes = s.codes[k][c];
      int byte = s.scale[k][c];
      if (D == 64 && q >= 2) codes = at_v4i{0, 0, 0, 0}, byte = 127;
      r = at_scores<E, D>(codes, byte, queries, c, r);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) score[k * 4 + i] = r[i];
  }
  // whether every row sees all of these tokens
  const bool whole = at_sees_all(p, low, high, s.first[0]) && at_sees_all(p, low, high, s.first[1]);
  unsigned seen = 0xff;
  if (!whole) {
    seen = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int first = s.first[j >> 2];
      const bool yes = first >= 0 && at_sees(p, position, first + 4 * q + (j & 3));
      seen |= yes ? 1u << j : 0;
      score[j] = yes ? score[j] : kAtNone;
    }
  }
  at_weigh<E>(score, a.most, a.sum, a.acc, p.scale, whole, seen);
  at_pack<E>(packed, score);
}

// Weights by values.
template <class E, int D>
__device__ __forceinline__ void at_values(AtState<E, D> &a, const at_v4i (&packed)[AtKind<E>::kP], AtWords<D> &s,
                                          const int (&tile)[2], const Attention &p, int position) {
  constexpr int kChunks = (D + 127) / 128, COLS = D == 64 ? 4 : 8;
  const int q = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int c = 0; c < kChunks; c++) {
    uint32_t high_byte = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) high_byte = max(high_byte, s.scale[c][j]);
    if (__ballot(high_byte >= (uint32_t)AtKind<E>::kNan)) {
      // Blocks that are NaN count as zeros in the product; who sees them becomes NaN.
      bool hit = false;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const bool is_bad = s.scale[c][j] >= (uint32_t)AtKind<E>::kNan;
        const unsigned long long bad = __ballot(is_bad);
        s.codes[c][j] = is_bad ? 0 : s.codes[c][j];
        s.scale[c][j] = is_bad ? 127 : s.scale[c][j];
        const int first = tile[j >> 2];
        if (bad && first >= 0) {
#pragma unroll 1
          for (int team = 0; team < 4; team++) hit = hit || (at_bad_block<D>(bad, team, q) && at_sees(p, position, first + 4 * team + (j & 3)));
        }
      }
#pragma unroll
      for (int m = 0; m < COLS; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) a.acc[c * 8 + m][i] = hit ? __builtin_nanf("") : a.acc[c * 8 + m][i];
    }
    float scale[8];
#pragma unroll
    for (int j = 0; j < 8; j++) scale[j] = at_value_scale<E>(s.scale[c][j]);
    at_transpose<E, COLS>(s.codes[c], scale, [&](int m, at_v4i values) {
#pragma unroll
      for (int t = 0; t < AtKind<E>::kP; t++) a.acc[c * 8 + m] = AtValues<E>::multiply(values, packed[t], a.acc[c * 8 + m]);
    });
  }
}

// Bound by the latency of its loads: 61 slots of up to 8 shares and 8 heads 7 us, 4 of 128 shares 21.
// The shares of sixteen rows joined, and what is done with the whole: wave 4 g + i has component i of every G-th share,
// from the g-th on, and these meet in LDS.
template <class E, class OUT, int D, int G>
__global__ __launch_bounds__(256 * G) void mx4_attention_join_kernel(Attention p) {
  __shared__ float s_x[G > 1 ? 4 * G - 4 : 1][D / 16][64], s_sum[G][16];
  __shared__ uint32_t s_most[4][64];
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = wave & 3, g = wave >> 2;
  const int h = (int)(blockIdx.x % (unsigned)p.kv_heads), slot = (int)(blockIdx.x / (unsigned)p.kv_heads);
  const float *part = p.part + ((size_t)slot * p.splits * p.kv_heads + h) * at_part_floats<D>();
  const size_t next = (size_t)p.kv_heads * at_part_floats<D>();
  // the first share says how many there are; a single one has stored the whole
  const int shares = p.target ? (int)part[16 * D + 32] : p.splits;
  AtRows r;
  if (!at_rows<16>(p, slot, r) || shares <= 1) return;
  const bool there = r.first + l16 < r.last;
  float most = kAtNone, sum = 0, x[D / 16];
#pragma unroll
  for (int m = 0; m < D / 16; m++) x[m] = 0;
  if (there) {
#pragma unroll 4
    for (int k = g; k < shares; k += G) {
      const float *from = part + k * next;
      const float of = from[16 * D + l16], weight = from[16 * D + 16 + l16];
      float y[D / 16];
#pragma unroll
      for (int m = 0; m < D / 16; m++) y[m] = from[(i * (D / 16) + m) * 64 + lane];
      const float top = fmaxf(most, of);
      // (sums of NaN come without a largest score)
      const float before = most == kAtNone ? 1.0f : at_exp2(most - top);
      const float factor = of == kAtNone ? (weight == 0 ? 0.0f : __builtin_nanf("")) : at_exp2(of - top);
      sum = sum * before + weight * factor;
#pragma unroll
      for (int m = 0; m < D / 16; m++) x[m] = x[m] * before + y[m] * factor;
      most = top;
    }
  }
  if (G > 1) {
    __shared__ float s_top[G][16];
    if (i == 0 && lane < 16) s_top[g][l16] = most;
    __syncthreads();
    float top = kAtNone;
#pragma unroll
    for (int k = 0; k < G; k++) top = fmaxf(top, s_top[k][l16]);
    const float factor = most == kAtNone ? 1.0f : at_exp2(most - top);
    sum *= factor;
#pragma unroll
    for (int m = 0; m < D / 16; m++) x[m] *= factor;
  }
  if (G > 1) {
    if (g > 0) {
#pragma unroll
      for (int m = 0; m < D / 16; m++) s_x[wave - 4][m][lane] = x[m];
    }
    if (i == 0 && lane < 16) s_sum[g][l16] = sum;
    __syncthreads();
    // (where blocks of results are formed, all waves meet at the barriers)
    if (g > 0 && OUT::kSize != 0) return;
    sum = 0;
#pragma unroll
    for (int k = 0; k < G; k++) sum += s_sum[k][l16];
    if (g == 0) {
#pragma unroll
      for (int k = 1; k < G; k++)
#pragma unroll
        for (int m = 0; m < D / 16; m++) x[m] += s_x[(k - 1) * 4 + i][m][lane];
    }
  }
#pragma unroll
  for (int m = 0; m < D / 16; m++) x[m] = sum == 0 ? 0.0f : x[m] / at_divisor<E>(sum);
  at_store<E, OUT, D>(p, r, h, i, x, s_most, g == 0);
}

// Bytes of the rings, in which results meet afterwards; queries' last terms lie behind them.
template <int D> constexpr int at_rows_rings() { return kAtWaves<D> * std::max(16 * D * 4, kAtStages * AtRing<D>::kStage); }
template <class E, int D> constexpr int at_rows_lds() { return at_rows_rings<D>() + kAtWaves<D> * AtQueries<E, D>::kLds; }
// Waves that share a SIMD's registers.
template <class E, int D> constexpr int at_rows_waves() { return D == 256 ? 1 : AtKind<E>::kQ == 6 ? 2 : 4; }

template <class E, class OUT, int D>
__global__ __launch_bounds__(kAtWaves<D> * 64, (at_rows_waves<E, D>())) void mx4_attention_rows_kernel(Attention p, unsigned units) {
  constexpr int WAVES = kAtWaves<D>;
  extern __shared__ __attribute__((aligned(16))) uint8_t s_ring[];
  float *const s_acc = reinterpret_cast<float *>(s_ring);           // [waves][4][D / 16][64]
  __shared__ float s_top[WAVES][16], s_sum[WAVES][16];
  __shared__ uint32_t s_most[4][64];
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // heads of the cache whose rows share lines run on one die, one behind the other, and shares on all dies in turn
  const unsigned place = blockIdx.x >> 3, of_all = place / (unsigned)p.kv_heads * 8 + (blockIdx.x & 7);
  if (of_all >= units) return;
  const int h = (int)(place % (unsigned)p.kv_heads), share = (int)(of_all % (unsigned)p.splits), slot = (int)(of_all / (unsigned)p.splits);
  AtRows r;
  if (!at_rows<16>(p, slot, r)) return;

  const int at = min(r.first + l16, r.last - 1), token = at / p.group, head = h * p.group + (at - token * p.group);
  auto position_of = [&](int row) { return max(r.length - r.count + row / p.group, -1); };
  const int position = position_of(at), low = position_of(r.first), high = position_of(r.last - 1);
  AtQueries<E, D> queries;
  queries.load(reinterpret_cast<const typename E::T *>(p.q + (size_t)(r.begin + token) * p.q_row_bytes) + (size_t)head * D,
               p.negative, s_ring + at_rows_rings<D>() + wave * AtQueries<E, D>::kLds);

  const AtTiles tiles = at_tiles(p, low, high);
  const int steps = (int)((tiles.all + 1ll) / 2), chunk = at_share_steps(p, steps, kAtLeast);
  const int begin = (int)min((long long)share * chunk, (long long)steps), end = (int)min((long long)begin + chunk, (long long)steps);
  const bool alone = steps <= chunk;            // (a slot without tokens is the first share's)
  if (share > 0 && begin >= steps) return;
  // (the joining launch asks how many shares there are; every wave of a head's tells it the same)
  if (share == 0 && p.splits > 1 && lane == 0)
    p.part[((size_t)of_all * p.kv_heads + h) * at_part_floats<D>() + 16 * D + 32] = alone ? 1.0f : (float)(((long long)steps + chunk - 1) / chunk);
  AtState<E, D> a;
  a.most = kAtNone, a.sum = 0;
#pragma unroll
  for (int m = 0; m < D / 16; m++) a.acc[m] = at_v4f{0, 0, 0, 0};
  const uint8_t *ring = s_ring + (size_t)wave * kAtStages * AtRing<D>::kStage;
  const int mine = end - begin - wave > 0 ? (end - begin - wave + WAVES - 1) / WAVES : 0;
  if (mine > 0) {
    AtLoader<D> loader(p, tiles, r.sequence, h, begin + wave, WAVES, end, lds_address(ring));
    int first[kAtStages][2];
#pragma unroll
    for (int k = 0; k < kAtStages; k++) loader.issue(k, first[k]);
    for (int n = 0; n < mine; n++) {
      AtKeys<D> keys;
      AtWords<D> words;
      at_v4i packed[AtKind<E>::kP];
      dma_wait<(kAtStages - 1) * AtRing<D>::kLoads>();
      loader.read(keys, ring, n, h);
      keys.first[0] = first[0][0], keys.first[1] = first[0][1];
      first[0][0] = first[1][0], first[0][1] = first[1][1];
      at_keys<E, D>(a, packed, queries, keys, p, low, high, position);
      asm volatile("" ::: "memory");                   // (not read before the keys' registers are free)
      loader.read(words, ring, n, h);
      // the slot is free when it has been read
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      loader.issue(n + kAtStages, first[1]);
      at_values<E, D>(a, packed, words, keys.first, p, position);
    }
    dma_wait<0>();
  }
  __syncthreads();                    // the rings' memory is used again

  const float sum = add_across32(add_across16(a.sum));
  if (lane < 16) s_top[wave][l16] = a.most, s_sum[wave][l16] = sum;
  __syncthreads();
  float most = kAtNone, whole = 0;
#pragma unroll
  for (int k = 0; k < WAVES; k++) most = fmaxf(most, s_top[k][l16]);
  // a wave that saw nothing has no part in it; sums of NaN come without a largest score
  auto factor_of = [&](float top, float of) {
    return top == kAtNone ? (of == 0 ? 0.0f : __builtin_nanf("")) : at_exp2(top - most);
  };
#pragma unroll
  for (int k = 0; k < WAVES; k++) whole += s_sum[k][l16] * factor_of(s_top[k][l16], s_sum[k][l16]);
  const float factor = factor_of(a.most, sum);
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int m = 0; m < D / 16; m++)
      s_acc[((wave * 4 + i) * (D / 16) + m) * 64 + lane] = a.acc[m][i] * factor;     // (NaN stays)
  __syncthreads();
  // (where blocks of results are formed, all waves meet at the barriers)
  if (wave >= 4 && (OUT::kSize != 0 || !alone)) return;
  float x[D / 16];
  const int i = wave & 3;
#pragma unroll
  for (int m = 0; m < D / 16; m++) x[m] = 0;
#pragma unroll
  for (int k = 0; k < WAVES; k++)
#pragma unroll
    for (int m = 0; m < D / 16; m++) x[m] += s_acc[((k * 4 + i) * (D / 16) + m) * 64 + lane];
  if (!alone) {
    float *part = p.part + ((size_t)of_all * p.kv_heads + h) * at_part_floats<D>();
    if (r.first + l16 < r.last) {
#pragma unroll
      for (int m = 0; m < D / 16; m++) part[(i * (D / 16) + m) * 64 + lane] = x[m];
    }
    if (wave == 0 && lane < 16) part[16 * D + l16] = most, part[16 * D + 16 + l16] = whole;
    return;
  }
#pragma unroll
  for (int m = 0; m < D / 16; m++) x[m] = whole == 0 ? 0.0f : x[m] / at_divisor<E>(whole);
  at_store<E, OUT, D>(p, r, h, i, x, s_most, wave < 4);
}

// The same for heads of 128 columns of which two, four or eight neighbours share a workgroup (HG), a wave each; where they
// are fewer than eight, further waves have further steps. What these heads have of a token is one stretch of memory: a load
// of 1 KB has 16 / HG tokens of all of them, lines whole, where a head's own rows come in pieces of 64 bytes and its
// scales in pieces of four (a large copy's rate against 60 % of it, nothing but loads). Waves wait for
// each other's loads at two barriers a step: when rows have landed, and when they are in registers. Bound by memory:
// four sequences of 100 000 to 131 072 tokens, 8 heads, fp16 queries 113 us (513 MB, 4.5 TB/s; 105 with nothing but the loads), and 21 to
// join them. A head a workgroup, before queries had a fourth term: 171 in all for 130.
//
// Piece k of a load, 16 bytes, lies at 16 k in LDS, and lanes choose theirs so that no read meets a bank twice, pieces of a
// head's 64 bytes side by side: with k = 16 xh + 4 xl + c', t a token of the tile, c a piece of its head,
//   keys    xl = (t ^ h) & 3, c' = c ^ t / 4    (a read has sixteen tokens, one c for each team of lanes)
//   values  xl = (t / 4 ^ h') & 3, c' = c       (a read has four tokens 4 q + i and all c; h' = 2 h for HG = 2)
// and xh what these leave open.
template <int HG> struct AtHeads {
  static constexpr int kWaves = 8, kGroups = kWaves / HG;       // groups of waves with steps of their own
  static constexpr int kTile = HG * 1024, kScales = 4 * kTile;  // sixteen tokens' codes; keys, keys, values, values, scales
  static constexpr int kGroup = kScales + HG * 256, kStage = kGroups * kGroup, kLoads = 5;
  static constexpr int kRings = 2 * kStage;
  static constexpr int kTokens = 16 / HG;                       // of a load

  // The token and head of piece group x (k / 4) of load j of a tile.
  static __device__ __forceinline__ void key(int x, int j, int &t, int &h) {
    const int xl = x & 3, xh = x >> 2;
    if constexpr (HG == 8) t = 2 * j + (xh & 1), h = (xh >> 1) * 4 + (xl ^ (t & 3));
    else if constexpr (HG == 4) h = xh, t = 4 * j + (xl ^ h);
    else h = xh & 1, t = 8 * j + 4 * (xh >> 1) + (xl ^ h);
  }
  static __device__ __forceinline__ void value(int x, int j, int &t, int &h) {
    const int xl = x & 3, xh = x >> 2;
    if constexpr (HG == 8) t = 2 * j + (xh & 1), h = (xh >> 1) * 4 + (xl ^ (j >> 1));
    else if constexpr (HG == 4) t = 4 * j + xh, h = xl ^ j;
    else t = 8 * j + 4 * (xl & 1) + xh, h = (xl >> 1) ^ j;
  }
  // Where piece c of a token's head lies in a tile.
  static __device__ __forceinline__ int key_place(int t, int h, int c) {
    const int xl = (t ^ h) & 3, xh = HG == 8 ? (h >> 2) * 2 + (t & 1) : HG == 4 ? h : (t >> 2 & 1) * 2 + h;
    return t / kTokens * 1024 + ((xh * 4 + xl) * 4 + (c ^ (t >> 2))) * 16;
  }
  static __device__ __forceinline__ int value_place(int t, int h, int c) {
    const int xl = ((t >> 2) ^ (HG == 2 ? 2 * h : h)) & 3, xh = HG == 8 ? (h >> 2) * 2 + (t & 1) : t & 3;
    return t / kTokens * 1024 + ((xh * 4 + xl) * 4 + c) * 16;
  }
  // How much further on token 4 q + i lies than token 4 q.
  static __device__ __forceinline__ constexpr int value_next(int i) { return HG == 8 ? (i >> 1) * 1024 + (i & 1) * 256 : i * 256; }
};

template <class E, class OUT, int HG>
__global__ __launch_bounds__(512, AtKind<E>::kQ == 6 ? 2 : 4) void mx4_attention_heads_kernel(Attention p, unsigned units) {
  typedef AtHeads<HG> H;
  constexpr int D = 128, TG = H::kGroups;
  extern __shared__ __attribute__((aligned(16))) uint8_t s_ring[];
  __shared__ float s_top[8][16], s_sum[8][16];
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), own = wave % HG, group = wave / HG;
  const unsigned sets = (unsigned)p.kv_heads / HG;
  const unsigned place = blockIdx.x >> 3, of_all = place / sets * 8 + (blockIdx.x & 7);
  if (of_all >= units) return;
  const int head0 = (int)(place % sets) * HG, h = head0 + own;
  const int share = (int)(of_all % (unsigned)p.splits), slot = (int)(of_all / (unsigned)p.splits);
  AtRows r;
  if (!at_rows<16>(p, slot, r)) return;

  const int at = min(r.first + l16, r.last - 1), token = at / p.group, head = h * p.group + (at - token * p.group);
  auto position_of = [&](int row) { return max(r.length - r.count + row / p.group, -1); };
  const int position = position_of(at), low = position_of(r.first), high = position_of(r.last - 1);
  AtQueries<E, D> queries;
  queries.load(reinterpret_cast<const typename E::T *>(p.q + (size_t)(r.begin + token) * p.q_row_bytes) + (size_t)head * D,
               p.negative, s_ring + H::kRings + wave * AtQueries<E, D>::kLds);
  const AtTiles tiles = at_tiles(p, low, high);
  const int steps = (int)((tiles.all + 1ll) / 2), chunk = at_share_steps(p, steps, kAtLeast);
  const int begin = (int)min((long long)share * chunk, (long long)steps), end = (int)min((long long)begin + chunk, (long long)steps);
  const bool alone = steps <= chunk;            // (a slot without tokens is the first share's)
  if (share > 0 && begin >= steps) return;
  // (the joining launch asks how many shares there are; every wave of a head's tells it the same)
  if (share == 0 && p.splits > 1 && lane == 0)
    p.part[((size_t)of_all * p.kv_heads + h) * at_part_floats<D>() + 16 * D + 32] = alone ? 1.0f : (float)(((long long)steps + chunk - 1) / chunk);
  AtState<E, D> a;
  a.most = kAtNone, a.sum = 0;
#pragma unroll
  for (int m = 0; m < D / 16; m++) a.acc[m] = at_v4f{0, 0, 0, 0};

  // what this lane asks for of each step, and where it finds its own
  const uint32_t row_bytes = (uint32_t)p.c.row_bytes, ring = lds_address(s_ring) + (uint32_t)group * H::kGroup;
  uint32_t key_at, value_at, scale_at;
  // (scales: keys, keys, values or values of the step's two tiles)
  const int array = HG == 2 ? own * 2 + (lane >> 5) : own * 64 / (16 * HG);
  {
    int t, of;
    H::key(lane >> 2, own, t, of);
    key_at = t * row_bytes + (uint32_t)(head0 + of) * 64 + ((lane & 3) ^ (t >> 2)) * 16;
    H::value(lane >> 2, own, t, of);
    value_at = t * row_bytes + (uint32_t)(head0 + of) * 64 + (lane & 3) * 16;
    const int word = own * 64 + lane;            // of [4 arrays][16 tokens][HG heads]
    scale_at = (word / HG % 16) * row_bytes + p.c.scales_at + (uint32_t)(head0 + word % HG) * 4;
  }
  const int key_place = H::key_place(l16, own, q);
  const int value_place = H::value_place(4 * q, own, l16 >> 2) + (l16 & 3) * 4;
  const int count = (end - begin + TG - 1) / TG;       // steps of every wave
  int tile_of = -1;
  auto issue = [&](int n, int (&first)[2]) {
    if ((n & 31) == 0) {                               // the rows of 32 steps' tiles, a lane each
      const long long step = begin + (long long)(n + (lane >> 1)) * TG + group;
      const int u = (int)min(2 * step + (lane & 1), (long long)tiles.all);
      tile_of = step < end && u < tiles.all ? cache_tile(p.c, r.sequence, (unsigned)tiles.at(u)) : -1;
    }
    const uint8_t *keys[2], *values[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int tile = __builtin_amdgcn_readlane(tile_of, 2 * (n & 31) + k);
      first[k] = tile < 0 ? -1 : tiles.at(2 * (begin + n * TG + group) + k) * kCacheTile;
      // (a tile that is not there reads the cache's first rows; there is a page)
      const size_t base = (size_t)max(tile, 0) * kCacheTile * p.c.row_bytes;
      keys[k] = p.c.keys + base, values[k] = p.c.values + base;
    }
    const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(ring + (n & 1) * H::kStage));
    // (added to each step's addresses, not kept as 64-bit sums with the cache's: registers)
    asm volatile("" : "+v"(key_at), "+v"(value_at), "+v"(scale_at));
#pragma unroll
    for (int k = 0; k < 2; k++) {
      dma16(keys[k] + key_at, to + k * H::kTile + own * 1024);
      dma16(values[k] + value_at, to + (2 + k) * H::kTile + own * 1024);
    }
    dma4((array == 0 ? keys[0] : array == 1 ? keys[1] : array == 2 ? values[0] : values[1]) + scale_at,
         to + H::kScales + own * 256);
  };
  if (count > 0) {
    int first[2][2];
    issue(0, first[0]);
    issue(1, first[1]);
    int key_from = key_place, value_from = value_place, key_scale = l16 * HG * 4 + q, value_scale = (32 + 4 * q) * HG * 4 + (l16 >> 2);
    for (int n = 0; n < count; n++) {
      asm volatile("" : "+v"(key_from), "+v"(value_from), "+v"(key_scale), "+v"(value_scale));
      dma_wait<H::kLoads>();
      __syncthreads();
      const uint8_t *from = s_ring + (size_t)group * H::kGroup + (n & 1) * H::kStage;
      const uint8_t *scales = from + H::kScales + own * 4;
      AtKeys<D> keys;
#pragma unroll
      for (int k = 0; k < 2; k++) {
        keys.codes[k][0] = *reinterpret_cast<const at_v4i *>(from + k * H::kTile + key_from);
        keys.scale[k][0] = scales[k * 64 * HG + key_scale];
        keys.first[k] = first[0][k];
        first[0][k] = first[1][k];
      }
      const bool some = keys.first[0] >= 0 || keys.first[1] >= 0;
      at_v4i packed[AtKind<E>::kP];
      if (some) at_keys<E, D>(a, packed, queries, keys, p, low, high, position);
      asm volatile("" ::: "memory");                   // (not read before the keys' registers are free)
      AtWords<D> words;
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          words.codes[0][k * 4 + i] = *reinterpret_cast<const uint32_t *>(from + (2 + k) * H::kTile + H::value_next(i) + value_from);
          words.scale[0][k * 4 + i] = scales[(k * 16 + i) * 4 * HG + value_scale];
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __syncthreads();
      issue(n + 2, first[1]);
      if (some) at_values<E, D>(a, packed, words, keys.first, p, position);
    }
    dma_wait<0>();
  }
  float whole = add_across32(add_across16(a.sum));
  if constexpr (TG > 1) {
    // the first group's waves take what the others have; a wave that saw nothing has no part in it, and sums of NaN
    // come without a largest score
    float *const s_acc = reinterpret_cast<float *>(s_ring);
    __syncthreads();
    if (lane < 16) s_top[wave][l16] = a.most, s_sum[wave][l16] = whole;
    __syncthreads();
    auto factor_of = [&](float top, float of, float most) {
      return top == kAtNone ? (of == 0 ? 0.0f : __builtin_nanf("")) : at_exp2(top - most);
    };
    float most = kAtNone;
#pragma unroll
    for (int k = 0; k < TG; k++) most = fmaxf(most, s_top[k * HG + own][l16]);
    const float factor = factor_of(a.most, whole, most);
#pragma unroll
    for (int m = 0; m < D / 16; m++)
#pragma unroll
      for (int i = 0; i < 4; i++) a.acc[m][i] *= factor;
    if (group > 0) {
#pragma unroll
      for (int m = 0; m < D / 16; m++) *reinterpret_cast<at_v4f *>(s_acc + (((wave - HG) * (D / 16) + m) * 64 + lane) * 4) = a.acc[m];
    }
    __syncthreads();
    if (group > 0) return;
    whole = 0;
#pragma unroll
    for (int k = 0; k < TG; k++) whole += s_sum[k * HG + own][l16] * factor_of(s_top[k * HG + own][l16], s_sum[k * HG + own][l16], most);
#pragma unroll
    for (int k = 1; k < TG; k++)
#pragma unroll
      for (int m = 0; m < D / 16; m++)
        a.acc[m] += *reinterpret_cast<const at_v4f *>(s_acc + ((((k - 1) * HG + own) * (D / 16) + m) * 64 + lane) * 4);
    a.most = most;
  }
  if (alone) {
    at_store_whole<E, OUT, D>(p, r, h, a.acc, whole);
    return;
  }
  float *part = p.part + ((size_t)of_all * p.kv_heads + h) * at_part_floats<D>();
  if (r.first + l16 < r.last) {
#pragma unroll
    for (int m = 0; m < D / 16; m++)
#pragma unroll
      for (int i = 0; i < 4; i++) part[(i * (D / 16) + m) * 64 + lane] = a.acc[m][i];
  }
  if (lane < 16) part[16 * D + l16] = a.most, part[16 * D + 16 + l16] = whole;
}

// How many heads of the cache a workgroup has.
static int at_head_set(const Attention &p, int dim) {
  return dim != 128 ? 1 : p.kv_heads % 8 == 0 ? 8 : p.kv_heads % 4 == 0 ? 4 : p.kv_heads % 2 == 0 ? 2 : 1;
}
template <class E, class OUT, int HG> static int at_heads_launch(const Attention &p, hipStream_t st) {
  constexpr size_t kLds = AtHeads<HG>::kRings + 8 * AtQueries<E, 128>::kLds;
  static_assert(AtHeads<HG>::kRings >= (8 - HG) * 16 * 128 * 4, "results of the other groups");
  static std::atomic<uint64_t> attr_set{0};
  auto kernel = mx4_attention_heads_kernel<E, OUT, HG>;
  if (int rc = set_lds_attr(kernel, kLds, attr_set)) return rc;
  const unsigned units = (unsigned)((long long)p.slots * p.splits);
  kernel<<<(units + 7) / 8 * 8 * (p.kv_heads / HG), 512, kLds, st>>>(p, units);
  return check_launch("mx4_attention");
}

// Shares of a slot's tokens: as many as give each CU two workgroups, of `least` tokens at least.
static int at_splits(long long units, long long tokens, long long least) {
  const long long fill = 512 / units, most = (tokens + least - 1) / least;
  return (int)std::max(1ll, std::min({fill, most, 256ll}));
}
static long long at_slots(size_t rows, size_t group, size_t sequences, int per_slot) {
  return (long long)(rows * group / per_slot + sequences);
}

template <class E, class OUT, int D> static int at_launch(Attention p, int type, bool prompt, int sixteens, hipStream_t st) {
  if (prompt) {
    if (int rc = at_prompt_launch(p, type, OUT::kSize == 0, D, st)) return rc;
  } else if (D == 128 && at_head_set(p, D) > 1) {
    const int set = at_head_set(p, D);
    if (int rc = set == 8   ? at_heads_launch<E, OUT, 8>(p, st)
                 : set == 4 ? at_heads_launch<E, OUT, 4>(p, st)
                            : at_heads_launch<E, OUT, 2>(p, st))
      return rc;
  } else {
    const unsigned units = (unsigned)((long long)p.slots * p.splits);
    constexpr size_t kLds = at_rows_lds<E, D>();
    static std::atomic<uint64_t> attr_set{0};
    auto kernel = mx4_attention_rows_kernel<E, OUT, D>;
    if (int rc = set_lds_attr(kernel, kLds, attr_set)) return rc;
    kernel<<<(units + 7) / 8 * 8 * p.kv_heads, kAtWaves<D> * 64, kLds, st>>>(p, units);
    if (int rc = check_launch("mx4_attention")) return rc;
  }
  if (p.splits == 1) return MI355X_OK;
  p.slots = sixteens;
  const unsigned blocks = (unsigned)((long long)p.slots * p.kv_heads);
  if (p.splits > 16) mx4_attention_join_kernel<E, OUT, D, 4><<<blocks, 1024, 0, st>>>(p);
  else mx4_attention_join_kernel<E, OUT, D, 1><<<blocks, 256, 0, st>>>(p);
  return check_launch("mx4_attention");
}
static size_t at_part_bytes(size_t dim) { return (16 * dim + 48) * sizeof(float); }

// How a call is cut, which does not depend on where its tensors lie.
struct AtPlan {
  bool prompt;
  int sixteens;                   // slots of sixteen rows
  size_t bytes;                   // of workspace
};
static int at_plan(const mi355x_mx4_cache *cache, size_t heads, int type, size_t sequences, size_t rows, size_t max_length,
                   size_t window, size_t sinks, Attention *p, AtPlan *plan) {
  MI355X_REQUIRE(heads > 0 && heads <= 0x7fffffff / cache->head_dim && heads % cache->kv_heads == 0,
                 "mx4_attention: %zu heads over the cache's %u", heads, cache->kv_heads);
  p->kv_heads = (int)cache->kv_heads;
  p->group = (int)(heads / cache->kv_heads);
  p->most = cache->n_pages ? (int)std::min<size_t>(max_length, (size_t)p->c.capacity) : 0;
  p->window = window == 0 || window > 0x7fffffff ? 0x7fffffff : (int)window;
  p->sinks = window == 0 || sinks == 0 ? 0 : (int)std::min<size_t>(sinks, 0x7fffffff);
  *plan = AtPlan{};
  p->splits = 1;
  if (!rows || !sequences) return MI355X_OK;
  if (rows > (size_t)0x7fff0000 / p->group)
    return fail(MI355X_ERR_NOT_SUPPORTED, "mx4_attention: %zu rows of %d heads to one of the cache", rows, p->group);
  const long long sixteens = at_slots(rows, p->group, sequences, 16);
  if (sixteens * p->kv_heads > 1 << 22)
    return fail(MI355X_ERR_NOT_SUPPORTED, "mx4_attention: %zu rows of %zu heads, %zu sequences", rows, heads, sequences);
  // Many rows of a sequence share what is read and converted. us, sixteens of rows / prompts' kernel, 32 heads of 128 over 8, bf16, 16
  // sequences of 4096 tokens: 32 pairs of a row and a head a sequence 41 / 58, 64 58 / 66, 96 83 / 71, 256 161 / 123; of 500 tokens: 96
  // 26 / 27.5, 128 34 / 28. (The average decides for the whole batch: single tokens beside a long prompt go with it.)
  plan->prompt = rows * p->group > 64 * sequences;
  plan->sixteens = (int)sixteens;
  const int per_slot = plan->prompt ? kPromptWaves * 16 * at_prompt_sixteens(type, (int)cache->head_dim) : 16;
  p->slots = (int)at_slots(rows, p->group, sequences, per_slot);
  const long long tokens = std::min<long long>(p->most, (long long)p->window + p->sinks + per_slot + 48);
  // (slots that have rows: not many more than this)
  const long long filled = std::max<long long>(sequences, rows * p->group / per_slot);
  const int set = plan->prompt ? 1 : at_head_set(*p, (int)cache->head_dim);
  p->splits = at_splits(filled * p->kv_heads / set, tokens, plan->prompt ? 512 : 32 * kAtLeast);
  // (no more shares than run at once: a few more would run alone, and a workgroup that finds nothing to do still takes
  // a place for a while: twice the shares, half of them without tokens, 165 us for 134 over 4 x 115 000 tokens)
  if (!plan->prompt && p->splits > 1) p->target = (int)std::max<long long>(filled, 512 / (p->kv_heads / set) - filled);
  if (p->splits > 1) plan->bytes = (size_t)sixteens * p->kv_heads * p->splits * at_part_bytes(cache->head_dim);
  return MI355X_OK;
}

} // namespace mi355x

using namespace mi355x;

extern "C" {

int mi355x_mx4_attention_workspace_bytes(const mi355x_mx4_cache *cache, size_t heads, size_t sequences, size_t rows,
                                         size_t max_length, size_t *bytes) {
  MI355X_REQUIRE(bytes, "mx4_attention_workspace_bytes: NULL");
  Attention p{};
  if (int rc = check_cache("mx4_attention", cache, &p.c)) return rc;
  MI355X_REQUIRE(sequences <= 0x3fffffff && rows <= 0x3fffffff,
                 "mx4_attention: %zu sequences, %zu rows: up to 2^30 - 1 are supported", sequences, rows);
  // (whatever the type; a window takes no more shares)
  *bytes = 0;
  for (int type : {MI355X_F32, MI355X_BF16}) {
    AtPlan plan;
    if (int rc = at_plan(cache, heads, type, sequences, rows, max_length, 0, 0, &p, &plan)) return rc;
    *bytes = std::max(*bytes, plan.bytes);
  }
  return MI355X_OK;
}

int mi355x_mx4_attention(void *out, int out_type, size_t out_row_bytes, const void *q, int type, size_t q_row_bytes,
                         size_t heads, const mi355x_mx4_cache *cache, const int32_t *starts, const int32_t *lengths,
                         size_t sequences, size_t rows, size_t max_length, float scale, size_t window, size_t sinks,
                         void *workspace, size_t workspace_bytes, void *stream) {
  Attention p{};
  if (int rc = check_cache("mx4_attention", cache, &p.c)) return rc;
  if (int rc = check_batch("mx4_attention", starts, lengths, sequences, rows, &p.c)) return rc;
  MI355X_REQUIRE(float_type(type), "mx4_attention: query type %d is none of the float types", type);
  MI355X_REQUIRE(out_type == type || out_type == MI355X_MX4,
                 "mx4_attention: result type %d: the queries' (%d) or microscaled rows are supported", out_type, type);
  MI355X_REQUIRE(scale - scale == 0, "mx4_attention: scale %g", (double)scale);
  AtPlan plan;
  if (int rc = at_plan(cache, heads, type, sequences, rows, max_length, window, sinks, &p, &plan)) return rc;
  const size_t need = plan.bytes;
  const size_t cols = heads * cache->head_dim;
  if (int rc = check_rows("mx4_attention: queries", q, type, q_row_bytes, rows, cols)) return rc;
  if (int rc = check_rows("mx4_attention: result", out, out_type, out_row_bytes, rows, cols)) return rc;
  if (!rows || !sequences) return MI355X_OK;
  const size_t out_span = rows_span(out_type, out_row_bytes, rows, cols), q_span = rows_span(type, q_row_bytes, rows, cols);
  MI355X_REQUIRE((out == q && out_type == type && out_row_bytes == q_row_bytes) || !overlaps(out, out_span, q, q_span),
                 "mx4_attention: the result overlaps the queries without being their place");
  const size_t span = cache_span(cache), table = cache->pages ? sequences * cache->pages_per_sequence * 4 : 0;
  auto meets = [&](const void *a, size_t bytes) {
    return overlaps(a, bytes, cache->keys, span) || overlaps(a, bytes, cache->values, span) ||
           overlaps(a, bytes, cache->pages, table) || overlaps(a, bytes, starts, 4 * (sequences + 1)) ||
           overlaps(a, bytes, lengths, 4 * sequences);
  };
  MI355X_REQUIRE(!meets(out, out_span), "mx4_attention: the result overlaps the cache or the batch's starts or lengths");
  if (need) {
    MI355X_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0,
                   "mx4_attention: a workspace of %zu bytes on a multiple of 16 is needed "
                   "(mi355x_mx4_attention_workspace_bytes)", need);
    MI355X_REQUIRE(!meets(workspace, need) && !overlaps(workspace, need, out, out_span) &&
                       !overlaps(workspace, need, q, q_span),
                   "mx4_attention: the workspace overlaps a tensor");
  }
  p.q = static_cast<const uint8_t *>(q);
  p.out = static_cast<uint8_t *>(out);
  p.part = static_cast<float *>(workspace);
  p.q_row_bytes = q_row_bytes;
  p.out_row_bytes = out_row_bytes;
  p.out_groups = (int)mx4_groups(cols);
  p.scale = __builtin_fabsf(scale) * 1.4426950408889634f;
  p.negative = scale < 0;
  const int dim = (int)cache->head_dim;
  hipStream_t st = as_stream(stream);
  const bool mx4 = out_type == MI355X_MX4;
  auto launch = [&](auto e, auto result) {
    typedef decltype(e) E;
    typedef decltype(result) OUT;
    return dim == 64    ? at_launch<E, OUT, 64>(p, type, plan.prompt, plan.sixteens, st)
           : dim == 128 ? at_launch<E, OUT, 128>(p, type, plan.prompt, plan.sixteens, st)
                        : at_launch<E, OUT, 256>(p, type, plan.prompt, plan.sixteens, st);
  };
  if (type == MI355X_F32) return mx4 ? launch(F32(), MX4()) : launch(F32(), F32());
  if (type == MI355X_F16) return mx4 ? launch(AtWide(), MX4()) : launch(F16(), F16());
  return mx4 ? launch(BF16(), MX4()) : launch(BF16(), BF16());
}

} // extern "C"
