// Attention over a cache of microscaled rows: many rows of queries a sequence.
#include "mx4_attention.h"

#include "gemm_i8.h"

namespace mi355x {

// A workgroup has 128 rows of queries (64 in fp32 or of 256 columns), 32 a wave, and takes the tokens that they see
// 64 at a time: each wave brings one tile of sixteen into LDS, keys as they are, values converted and transposed to
// what the matrix instructions want, once for all waves. Two buffers: a step is prepared while the one in front is
// multiplied, and its successor's rows are on their way from memory into registers.
//
// Two prompts of 4096, 32 heads of 128 over 8, bf16: 411 us, 669 TFLOP/s (a workgroup for sixteen rows, each converting
// values for itself: 1884). A wave's step is 68 matrix instructions of 16 cycles and 365 others. Matrix cores are busy for 26 % of the
// cycles, vector instructions for 48 %: the chain of a step, the largest score above all, is waited for, and no more than two waves
// fit the registers.
constexpr int kPromptTiles = kPromptWaves;

// What is said of a tile.
constexpr int kPromptNan = 1, kPromptAbsent = 2;

template <class E, int D> struct PromptLds {
  static constexpr int kChunks = (D + 127) / 128, COLS = D == 64 ? 4 : 8;
  at_v4i values[2][kChunks * COLS][64];             // [32 tokens][column][lane]
  at_v4i keys[kPromptTiles][kChunks][64];
  uint8_t key_scale[kPromptTiles][kChunks][64];
  unsigned long long bad[kPromptTiles][kChunks][4];     // lanes whose values are NaN, for each of a lane's tokens
  int flags[kPromptTiles];
};

// What a wave has asked for of a tile.
template <int D> struct PromptTile {
  static constexpr int kChunks = (D + 127) / 128;
  at_v4i keys[kChunks];
  int key_scale[kChunks];
  uint32_t values[kChunks][4], value_scale[kChunks][4];
  bool there;
};

template <class E, class OUT, int D, int QT>
__global__ __launch_bounds__(kPromptWaves * 64, 2) void mx4_attention_prompt_kernel(Attention p, unsigned blocks) {
  constexpr int kChunks = (D + 127) / 128, COLS = D == 64 ? 4 : 8, ROWS = kPromptWaves * QT * 16, P = AtKind<E>::kP;
  extern __shared__ __attribute__((aligned(16))) uint8_t s_all[];
  PromptLds<E, D> *const lds = reinterpret_cast<PromptLds<E, D> *>(s_all);
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the last rows, which see most, begin
  const unsigned id = blockIdx.x;
  if (id >= blocks) return;
  const int h = (int)(id % (unsigned)p.kv_heads), share = (int)(id / (unsigned)p.kv_heads % (unsigned)p.splits),
            slot = p.slots - 1 - (int)(id / (unsigned)p.kv_heads / (unsigned)p.splits);
  AtRows r;
  if (!at_rows<ROWS>(p, slot, r)) return;
  auto position_of = [&](int row) { return max(r.length - r.count + row / p.group, -1); };
  const int low = position_of(r.first), high = position_of(r.last - 1);

  // this wave's rows
  AtQueries<E, D> queries[QT];
  int position[QT], my_low[QT], my_high[QT];
#pragma unroll
  for (int t = 0; t < QT; t++) {
    const int first = r.first + (wave * QT + t) * 16, at = min(first + l16, r.last - 1);
    const int token = at / p.group, head = h * p.group + (at - token * p.group);
    position[t] = position_of(at);
    // (none: rows that see nothing)
    my_low[t] = first < r.last ? position_of(first) : -1;
    my_high[t] = first < r.last ? position_of(min(first + 15, r.last - 1)) : -1;
    queries[t].load(reinterpret_cast<const typename E::T *>(p.q + (size_t)(r.begin + token) * p.q_row_bytes) + (size_t)head * D,
                    p.negative, s_all + 2 * sizeof(PromptLds<E, D>) + (wave * QT + t) * AtQueries<E, D>::kLds);
  }
  // Sums of weights are products with a column of ones, whose results are all the same: the vector unit has more to do than
  // the matrix cores (16 additions of 110 instructions for sixteen rows and 64 tokens).
  at_v4f acc[QT][D / 16 + 1];
  float most[QT];
#pragma unroll
  for (int t = 0; t < QT; t++) {
    most[t] = kAtNone;
#pragma unroll
    for (int m = 0; m <= D / 16; m++) acc[t][m] = at_v4f{0, 0, 0, 0};
  }

  const AtTiles tiles = at_tiles(p, low, high);
  const long long steps = (tiles.all + kPromptTiles - 1) / kPromptTiles;
  const int begin = (int)(steps * share / p.splits), end = (int)(steps * (share + 1) / p.splits);

  // ---- a tile from memory to LDS
  const uint32_t row_bytes = (uint32_t)p.c.row_bytes, codes_at = (uint32_t)h * (D / 2), scales_at = p.c.scales_at + (uint32_t)h * (D / 32);
  const int block = D == 64 ? q & 1 : q;
  const uint32_t key_at = l16 * row_bytes + codes_at + block * 16, key_scale_at = l16 * row_bytes + scales_at + block;
  uint32_t value_at[4], value_scale_at[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    value_at[i] = (4 * q + i) * row_bytes + codes_at + l16 * (COLS / 2);
    value_scale_at[i] = (4 * q + i) * row_bytes + scales_at + l16 * COLS / 32;
  }
  // Where this wave's tiles lie, a lane each of 64 steps, which are asked for in order: an entry of the page table asked for
  // at each step would be waited for together with all that was asked for in front of it (4 % over 2 x 4096).
  int tile_of = -1;
  auto locate = [&](int step) {
    const int n = step - begin;
    if ((n & 63) == 0) {
      const long long u = ((long long)step + lane) * kPromptTiles + wave;
      tile_of = u < tiles.all ? cache_tile(p.c, r.sequence, (unsigned)tiles.at((int)u)) : -1;
    }
    return __builtin_amdgcn_readlane(tile_of, n & 63);
  };
  auto load = [&](PromptTile<D> &t, int tile) {
    t.there = tile >= 0;
    // (a tile that is not there reads the cache's first rows; there is a page)
    const size_t base = (size_t)max(tile, 0) * kCacheTile * p.c.row_bytes;
    const uint8_t *keys = p.c.keys + base, *values = p.c.values + base;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      t.keys[c] = *reinterpret_cast<const at_v4i *>(keys + (key_at + c * 64));
      t.key_scale[c] = keys[key_scale_at + c * 4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (COLS == 8) t.values[c][i] = *reinterpret_cast<const uint32_t *>(values + (value_at[i] + c * 64));
        else t.values[c][i] = *reinterpret_cast<const uint16_t *>(values + value_at[i]);
        t.value_scale[c][i] = values[value_scale_at[i] + c * 4];
      }
    }
  };
  auto store = [&](PromptTile<D> &t, PromptLds<E, D> &to) {
    bool any = false;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const bool none = D == 64 && q >= 2;           // (these lanes have no columns)
      to.keys[wave][c][lane] = none ? at_v4i{0, 0, 0, 0} : t.keys[c];
      to.key_scale[wave][c][lane] = none ? 127 : (uint8_t)t.key_scale[c];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) top = max(top, t.value_scale[c][i]);
      if (__ballot(top >= (uint32_t)AtKind<E>::kNan)) {
        // blocks that are NaN count as zeros in the product; who sees them becomes NaN
        any = true;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const bool is_bad = t.value_scale[c][i] >= (uint32_t)AtKind<E>::kNan;
          const unsigned long long mask = __ballot(is_bad);
          if (lane == 0) to.bad[wave][c][i] = mask;
          t.values[c][i] = is_bad ? 0 : t.values[c][i];
          t.value_scale[c][i] = is_bad ? 127 : t.value_scale[c][i];
        }
      } else if (kChunks > 1 && lane == 0) {
#pragma unroll
        for (int i = 0; i < 4; i++) to.bad[wave][c][i] = 0;
      }
      float scale[4];
#pragma unroll
      for (int i = 0; i < 4; i++) scale[i] = at_value_scale<E>(t.value_scale[c][i]);
      typedef int Half __attribute__((ext_vector_type(2)));
      Half columns[COLS];
      at_transpose4<E, COLS>(columns, t.values[c], scale);
#pragma unroll
      for (int m = 0; m < COLS; m++) reinterpret_cast<Half *>(&to.values[wave >> 1][c * COLS + m][lane])[wave & 1] = columns[m];
    }
    if (lane == 0) to.flags[wave] = t.there ? (any ? kPromptNan : 0) : kPromptAbsent;
  };

  PromptTile<D> next;
  if (begin < end) {
    load(next, locate(begin));
    store(next, lds[0]);
    if (begin + 1 < end) load(next, locate(begin + 1));
  }
  __syncthreads();
  for (int step = begin; step < end; step++) {
    const PromptLds<E, D> &now = lds[(step - begin) & 1];
    if (step + 1 < end) {
      store(next, lds[(step - begin + 1) & 1]);
      if (step + 2 < end) load(next, locate(step + 2));
    }
    // (which tokens come is known without LDS; whether they are there, and are numbers, when it is needed)
    int first[kPromptTiles];
    bool nothing = true, whole = true;
#pragma unroll
    for (int k = 0; k < kPromptTiles; k++) {
      const int u = step * kPromptTiles + k;
      first[k] = u < tiles.all ? tiles.at(u) * kCacheTile : -1;
#pragma unroll
      for (int t = 0; t < QT; t++) {
        nothing = nothing && at_sees_none(p, my_low[t], my_high[t], first[k]);
        whole = whole && at_sees_all(p, my_low[t], my_high[t], first[k]);
      }
    }
    if (!nothing) {
      // The sixteens of rows go through each step side by side: alone, each would wait for its own results.
      const at_v4i flag = *reinterpret_cast<const at_v4i *>(now.flags);
      float score[QT][16];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int k = 0; k < kPromptTiles; k++) {
        at_v4f s[QT];
#pragma unroll
        for (int t = 0; t < QT; t++) s[t] = at_v4f{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
          const at_v4i codes = now.keys[k][c][lane];
          const int byte = now.key_scale[k][c][lane];
#pragma unroll
          for (int t = 0; t < QT; t++) s[t] = at_scores<E, D>(codes, byte, queries[t], c, s[t]);
        }
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) score[t][k * 4 + i] = s[t][i];
      }
      __builtin_amdgcn_s_setprio(0);
      const int flags = __builtin_amdgcn_readfirstlane(flag[0] | flag[1] | flag[2] | flag[3]);
      whole = whole && !(flags & kPromptAbsent);
      unsigned seen[QT];
      if (!whole) {
#pragma unroll
        for (int k = 0; k < kPromptTiles; k++)
          if (__builtin_amdgcn_readfirstlane(flag[k]) & kPromptAbsent) first[k] = -1;
#pragma unroll
        for (int t = 0; t < QT; t++) {
          seen[t] = 0;
#pragma unroll
          for (int j = 0; j < 16; j++) {
            const bool yes = first[j >> 2] >= 0 && at_sees(p, position[t], first[j >> 2] + 4 * q + (j & 3));
            seen[t] |= yes ? 1u << j : 0;
            score[t][j] = yes ? score[t][j] : kAtNone;
          }
        }
      }
      float top[QT];
      bool up = false;
#pragma unroll
      for (int t = 0; t < QT; t++) {
        top[t] = at_top(score[t], p.scale);
        up = up || top[t] > most[t] + kAtSlack;
      }
      if (__ballot(up)) {
#pragma unroll
        for (int t = 0; t < QT; t++) {
          const bool mine = top[t] > most[t] + kAtSlack;
          const float factor = mine ? at_exp2(most[t] - top[t]) : 1.0f;
          most[t] = mine ? top[t] : most[t];
#pragma unroll
          for (int m = 0; m <= D / 16; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[t][m][i] *= factor;
        }
      }
#pragma unroll
      for (int t = 0; t < QT; t++) {
        const float off = AtKind<E>::kUp - most[t];
#pragma unroll
        for (int j = 0; j < 16; j++) score[t][j] = at_exp2(fmaf(score[t][j], p.scale, off));
      }
      if (!whole) {
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int j = 0; j < 16; j++) score[t][j] = seen[t] >> j & 1 ? score[t][j] : 0.0f;
      }
      at_v4i packed[QT][2][P];
#pragma unroll
      for (int t = 0; t < QT; t++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          float part[8];
#pragma unroll
          for (int j = 0; j < 8; j++) part[j] = score[t][k * 8 + j];
          at_pack<E>(packed[t][k], part);
        }
      __builtin_amdgcn_s_setprio(1);
      const at_v4i ones = {AtValues<E>::kOnes, AtValues<E>::kOnes, AtValues<E>::kOnes, AtValues<E>::kOnes};
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int s = 0; s < P; s++) acc[t][D / 16] = AtValues<E>::multiply(ones, packed[t][k][s], acc[t][D / 16]);
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int m = 0; m < kChunks * COLS; m++) {
          const at_v4i values = now.values[k][m][lane];
#pragma unroll
          for (int t = 0; t < QT; t++)
#pragma unroll
            for (int s = 0; s < P; s++) acc[t][m] = AtValues<E>::multiply(values, packed[t][k][s], acc[t][m]);
        }
      __builtin_amdgcn_s_setprio(0);
      if (flags & kPromptNan) {
        bool hit[QT][kChunks] = {};
#pragma unroll 1
        for (int k = 0; k < kPromptTiles; k++) {
          const int u = step * kPromptTiles + k, from = u < tiles.all ? tiles.at(u) * kCacheTile : -1;
          if (now.flags[k] != kPromptNan || from < 0) continue;        // (not there: not seen)
#pragma unroll 1
          for (int x = 0; x < 16; x++)
#pragma unroll
            for (int c = 0; c < kChunks; c++) {
              const bool mine = at_bad_block<D>(now.bad[k][c][x & 3], x >> 2, q);
#pragma unroll
              for (int t = 0; t < QT; t++) hit[t][c] = hit[t][c] || (mine && at_sees(p, position[t], from + x));
            }
        }
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int c = 0; c < kChunks; c++)
#pragma unroll
            for (int m = 0; m < COLS; m++)
#pragma unroll
              for (int e = 0; e < 4; e++) acc[t][c * COLS + m][e] = hit[t][c] ? __builtin_nanf("") : acc[t][c * COLS + m][e];
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int t = 0; t < QT; t++) {
    AtRows mine = r;
    mine.first = r.first + (wave * QT + t) * 16;
    mine.last = min(r.last, mine.first + 16);
    if (mine.first >= mine.last) continue;
    const float whole = acc[t][D / 16][0];
    if (p.splits == 1) {
      at_store_whole<E, OUT, D>(p, mine, h, acc[t], whole);
    } else {
      const long long sixteen = at_first_slot<16>(p, r.sequence) + mine.first / 16;
      float *part = p.part + ((size_t)(sixteen * p.splits + share) * p.kv_heads + h) * at_part_floats<D>();
#pragma unroll
      for (int m = 0; m < D / 16; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) part[(i * (D / 16) + m) * 64 + lane] = acc[t][m][i];
      if (lane < 16) part[16 * D + l16] = most[t], part[16 * D + 16 + l16] = whole;
    }
  }
}

template <class E, class OUT, int D, int TYPE> static int prompt_launch(const Attention &p, hipStream_t st) {
  constexpr int QT = at_prompt_sixteens(TYPE, D);
  constexpr size_t kLds = 2 * sizeof(PromptLds<E, D>) + kPromptWaves * QT * AtQueries<E, D>::kLds;
  static std::atomic<uint64_t> attr_set{0};
  auto kernel = mx4_attention_prompt_kernel<E, OUT, D, QT>;
  if (int rc = set_lds_attr(kernel, kLds, attr_set)) return rc;
  const unsigned blocks = (unsigned)((long long)p.slots * p.splits * p.kv_heads);
  kernel<<<blocks, kPromptWaves * 64, kLds, st>>>(p, blocks);
  return check_launch("mx4_attention");
}
template <class E, class OUT, int TYPE> static int prompt_launch_dim(const Attention &p, int dim, hipStream_t st) {
  return dim == 64    ? prompt_launch<E, OUT, 64, TYPE>(p, st)
         : dim == 128 ? prompt_launch<E, OUT, 128, TYPE>(p, st)
                      : prompt_launch<E, OUT, 256, TYPE>(p, st);
}
int at_prompt_launch(const Attention &p, int type, bool mx4, int dim, hipStream_t st) {
  if (type == MI355X_F32)
    return mx4 ? prompt_launch_dim<F32, MX4, MI355X_F32>(p, dim, st) : prompt_launch_dim<F32, F32, MI355X_F32>(p, dim, st);
  if (type == MI355X_F16)
    return mx4 ? prompt_launch_dim<AtWide, MX4, MI355X_F16>(p, dim, st) : prompt_launch_dim<F16, F16, MI355X_F16>(p, dim, st);
  return mx4 ? prompt_launch_dim<BF16, MX4, MI355X_BF16>(p, dim, st) : prompt_launch_dim<BF16, BF16, MI355X_BF16>(p, dim, st);
}

} // namespace mi355x
