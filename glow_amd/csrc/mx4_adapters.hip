// A product of microscaled rows with low-rank adapters of its rows' own beside it.
#include "mx4_adapters.h"

namespace mi355x {

// The launch in front of the product: low[m] for tiles of sixteen rows and up to 64 ranks, K over the eight waves of a
// workgroup, and (behind these workgroups) float rows quantised for the product. Rows of a tile may have up to sixteen
// adapters: workgroups take them in turns, one each while rows are few. Where rows are so few that CUs are idle, K goes to
// several workgroups too. What bounds it with many rows is the rate at which a CU pulls rows from its L2, 17 bytes a cycle, however
// many loads it has asked for: 640 KB a workgroup over 4096 columns and 64 ranks. 4096 rows of six adapters of rank 64 / 32 / 16 /
// none 41 / 27 / 20 / 12 us, fp16; 64 rows of 64 adapters of rank 16, bf16, 5.5 us.
constexpr int kDownThreads = 512, kDownWaves = kDownThreads / 64;

struct MxDown {
  const uint8_t *in;
  size_t in_row_bytes;
  const uint8_t *down;
  const float *scales;
  const int32_t *of_row;
  float *low;
  uint8_t *packed;                 // float rows' microscaled form
  size_t packed_row_bytes;
  int M, K, groups, rank, ranks, count;
  int row_tiles, rank_tiles, turns, parts;  // workgroups: row tiles x rank tiles x turns x parts of K
};

// Eight neighbouring values of a row from k on, as they are in memory; zeros from column `end` on unless WHOLE.
template <class E> struct DownValues {
  typedef typename E::Eight Raw;
  template <bool WHOLE> static __device__ __forceinline__ Raw load(const uint8_t *row, int k, int end, int) {
    const typename E::T *at = reinterpret_cast<const typename E::T *>(row) + k;
    return WHOLE || k + 8 <= end ? load_eight<E>(at) : load_eight_end<E>(at, end - k);
  }
  static __device__ __forceinline__ void floats(float (&x)[8], const Raw &r) {
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = E::get(r, j);
  }
};
template <> struct DownValues<MX4> {
  struct Raw {
    uint32_t codes, byte;
  };
  template <bool WHOLE> static __device__ __forceinline__ Raw load(const uint8_t *row, int k, int end, int groups) {
    // (what is past K is zero up to whole groups; `end` is that of a range of eights, or K)
    if (!WHOLE && k >= end) return Raw{0, 0};
    return Raw{*reinterpret_cast<const uint32_t *>(row + (k >> 1)), row[(size_t)groups * kMxGroupBytes + (k >> 5)]};
  }
  static __device__ __forceinline__ void floats(float (&x)[8], const Raw &r) { mx4_values8(x, r.codes, r.byte); }
};

// 16 ranks by 16 rows over 32 columns: bf16 as it is (microscaled values are bf16 numbers), fp16 by fp16, anything
// else in 32 bits by eight instructions of four columns, column j of each lane's in the j-th.
template <class IN, class A> struct DownProduct {
  static constexpr bool kBf16 = std::is_same<A, BF16>::value && (std::is_same<IN, BF16>::value || std::is_same<IN, MX4>::value);
  static constexpr bool kF16 = std::is_same<A, F16>::value && std::is_same<IN, F16>::value;
  static __device__ __forceinline__ mx_v4f run(const typename DownValues<A>::Raw &a, const typename DownValues<IN>::Raw &x, mx_v4f acc) {
    if constexpr (kBf16) {
      v4i v;
      if constexpr (IN::kSize != 0) v = __builtin_bit_cast(v4i, x);
      else {
        float y[8];
        DownValues<IN>::floats(y, x);
        v = __builtin_bit_cast(v4i, BF16::put(y));             // (exact)
      }
      return ad_multiply(__builtin_bit_cast(v4i, a), v, acc);
    } else if constexpr (kF16) {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, x, acc, 0, 0, 0);
    } else {
      float u[8], v[8];
      DownValues<A>::floats(u, a);
      DownValues<IN>::floats(v, x);
#pragma unroll
      for (int j = 0; j < 8; j++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(u[j], v[j], acc, 0, 0, 0);
      return acc;
    }
  }
};

template <class IN, class A, int RT>
__global__ __launch_bounds__(kDownThreads) void mx4_adapters_down_kernel(MxDown p) {
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned tiles = (unsigned)p.row_tiles * p.rank_tiles * p.turns * p.parts;
  if (blockIdx.x >= tiles) {
    if constexpr (IN::kSize != 0) {
      const unsigned long long unit = (blockIdx.x - tiles) * (unsigned long long)(kDownThreads / 16) + (tid >> 4);
      const unsigned long long row = unit / (unsigned)p.groups;
      const int g = (int)(unit % (unsigned)p.groups), k = g * kMxGroup + (tid & 15) * 8;
      if (row < (unsigned)p.M) {
        const typename IN::T *in = reinterpret_cast<const typename IN::T *>(p.in + row * p.in_row_bytes) + k;
        typename IN::Eight x;
        if (k <= p.K - 8) x = load_eight<IN>(in);
        else x = load_eight_end<IN>(in, p.K - k);
        mx4_store_group<IN>(p.packed + row * p.packed_row_bytes, p.groups, g, tid & 15, x);
      }
    }
    return;
  }
  __shared__ float s_part[kDownWaves][RT * 4][64];
  const int part = (int)(blockIdx.x % (unsigned)p.parts);
  unsigned block = blockIdx.x / (unsigned)p.parts;
  const int turn = (int)(block % (unsigned)p.turns);
  block /= (unsigned)p.turns;
  const int rank0 = (int)(block % (unsigned)p.rank_tiles) * 16 * RT, m0 = (int)(block / (unsigned)p.rank_tiles) * 16;
  const int m = m0 + l16;
  const int id = m < p.M ? p.of_row[m] : -1;
  unsigned left = (unsigned)__ballot(id >= 0 && id < p.count) & 0xffff;
  const int shares = kDownWaves * p.parts, per = ((p.K + 63) / 64 + shares - 1) / shares * 64;
  const int begin = min(p.K, (part * kDownWaves + wave) * per), end = min(p.K, begin + per);
  const uint8_t *x_row = p.in + (size_t)min(m, p.M - 1) * p.in_row_bytes;
  for (int k = 0; left; k++) {
    const int a = __builtin_amdgcn_readlane(id, __ffs(left) - 1);
    left &= ~(unsigned)__ballot(id == a);
    if (k % p.turns != turn) continue;
    mx_v4f acc[RT];
    const uint8_t *a_row[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
      acc[t] = mx_v4f{0, 0, 0, 0};
      // ranks past the last re-read it; what they give is not stored
      a_row[t] = p.down + ((size_t)a * p.rank + min(rank0 + t * 16 + l16, p.rank - 1)) * p.K * A::kSize;
    }
    // Several steps' loads at once, without a condition of each lane's while all columns are there. A lane takes 16 neighbouring
    // columns of 64, eight a step, so that two loads in a row use lines of 128 bytes whole.
    constexpr int AHEAD = A::kSize == 4 || IN::kSize == 4 || RT == 4 ? 2 : 4;
    auto steps = [&](int c, auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      typename DownValues<IN>::Raw x[AHEAD];
      typename DownValues<A>::Raw y[AHEAD][RT];
#pragma unroll
      for (int s = 0; s < AHEAD; s++) {
        const int k = c + s / 2 * 64 + 16 * q + s % 2 * 8;
        x[s] = DownValues<IN>::template load<WHOLE>(x_row, k, end, p.groups);
#pragma unroll
        for (int t = 0; t < RT; t++) y[s][t] = DownValues<A>::template load<WHOLE>(a_row[t], k, end, 0);
      }
#pragma unroll
      for (int s = 0; s < AHEAD; s++)
#pragma unroll
        for (int t = 0; t < RT; t++) acc[t] = DownProduct<IN, A>::run(y[s][t], x[s], acc[t]);
    };
    int c = begin;
    for (; c + 32 * AHEAD <= end; c += 32 * AHEAD) steps(c, std::true_type());
    // (columns from `end` on are the next wave's, or not there: with the range cut at `end` they are zeros)
    for (; c < end; c += 32 * AHEAD) steps(c, std::false_type());
    __syncthreads();                               // (the adapter in front may still be read)
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) s_part[wave][t * 4 + e][lane] = acc[t][e];
    __syncthreads();
    // lane (row l16, ranks 4 q + e)
    for (int t = wave; t < (RT == 1 ? 2 : RT); t += kDownWaves) {      // (ranks up to a multiple of 32: zeros)
      const float scale = p.scales ? p.scales[a] : 1.0f;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float sum = 0;
#pragma unroll
        for (int w = 0; w < kDownWaves; w++) sum += s_part[w][min(t, RT - 1) * 4 + e][lane];
        v[e] = rank0 + t * 16 + 4 * q + e < p.rank ? sum * scale : 0.0f;
      }
      const int r = rank0 + t * 16 + 4 * q;
      if (id == a && r < p.ranks) {
        *reinterpret_cast<float4 *>(p.low + ((size_t)part * p.M + m) * p.ranks + r) = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
  }
}

template <class IN, class A> static void down_launch(const MxDown &p, unsigned blocks, hipStream_t st) {
  if (p.rank <= 16) mx4_adapters_down_kernel<IN, A, 1><<<blocks, kDownThreads, 0, st>>>(p);
  else if (p.ranks <= 32) mx4_adapters_down_kernel<IN, A, 2><<<blocks, kDownThreads, 0, st>>>(p);
  else mx4_adapters_down_kernel<IN, A, 4><<<blocks, kDownThreads, 0, st>>>(p);
}
template <class IN> static void down_launch_type(const MxDown &p, int type, unsigned blocks, hipStream_t st) {
  if (type == MI355X_F32) down_launch<IN, F32>(p, blocks, st);
  else if (type == MI355X_F16) down_launch<IN, F16>(p, blocks, st);
  else down_launch<IN, BF16>(p, blocks, st);
}

template <class OUT> static int adapted_launch(const MxFcAdapted &p, int K, FcTile tile, hipStream_t st) {
  if constexpr (OUT::kSize == 0) {
    if (tile == kFc16) return mx4_fc_small_launch<MX4, OUT, 1, 2>(p, K, st);
  } else {
    if (tile == kFc16) return mx4_fc_small_launch<MX4, OUT, 1, 1>(p, K, st);
    if (tile == kFc32x16) return mx4_fc_small_launch<MX4, OUT, 2, 1>(p, K, st);
  }
  if (tile <= kFc32) return mx4_fc_small_launch<MX4, OUT, 2, 2>(p, K, st);
  if (tile == kFcShort64) return mx4_fc_short_launch<MX4, OUT, 64, 64, 32, 32, 4>(p, K, st);
  if (tile == kFcShort128) return mx4_fc_short_launch<MX4, OUT, 128, 128, 64, 64, 2>(p, K, st);
  return tile == kFc256   ? mx4_fc_tile_launch<OUT, 256, 256, 128, 64, 4, 1>(p, st)
         : tile == kFc128 ? mx4_fc_tile_launch<OUT, 128, 128, 64, 64, 4, 2>(p, st)
                          : mx4_fc_tile_launch<OUT, 64, 64, 32, 32, 4, 4>(p, st);
}

constexpr size_t kMostRank = 1024;
// Columns are counted in 32 bits, by waves that have up to 2048 of them behind the last and look two steps ahead.
constexpr size_t kMostColumns = 0x7fffffff - 4096;

// Two turns for many rows: where requests meet in a tile, its two adapters would take turns in one workgroup.
static int down_turns(size_t M) { return M <= 256 ? (int)std::min<size_t>(16, M) : 2; }
// Parts of K, of two steps a wave at least, for up to 256 rows. us, this launch / the product, 64 rows of 64 adapters of rank 16,
// 4096 x 4096 weights: 1 part 11.0 / 15.8, 4 parts 5.6 / 19.3. More rows have a workgroup for each CU: 4096 of six adapters of
// rank 64, 1 part 41.0 / 71.2, 2 parts 41.4 / 83.7.
static int down_parts(size_t M, size_t K, size_t rank) {
  if (M > 256) return 1;
  const size_t tiles = (M + 15) / 16 * (rank <= 32 ? 1 : (rank + 63) / 64) * down_turns(M);
  return (int)std::max<size_t>(1, std::min<size_t>({(size_t)kMostParts, 512 / tiles, K / 512}));
}
static size_t low_bytes(size_t M, size_t K, size_t rank) {
  return down_parts(M, K, rank) * M * ((rank + 31) / 32 * 32) * sizeof(float);
}

} // namespace mi355x

using namespace mi355x;

extern "C" {

int mi355x_mx4_fc_adapters_workspace_bytes(size_t M, size_t K, size_t N, int in_type, size_t rank, size_t *bytes) {
  MI355X_REQUIRE(bytes, "mx4_fc_adapters_workspace_bytes: NULL");
  MI355X_REQUIRE(in_type == MI355X_MX4 || float_type(in_type), "mx4_fc_adapters_workspace_bytes: unknown element type %d",
                 in_type);
  MI355X_REQUIRE(M <= 0x7fffffff && K <= 0x7fffffff && N <= 0x7fffffff,
                 "mx4_fc_adapters_workspace_bytes: %zu x %zu x %zu, up to 2^31 - 1 each are supported", M, K, N);
  MI355X_REQUIRE(rank <= kMostRank, "mx4_fc_adapters: rank %zu, up to %zu is supported", rank, kMostRank);
  *bytes = !M || !N || !rank ? (in_type == MI355X_MX4 || !M || !N ? 0 : M * mx4_row_bytes_of(K)) : low_bytes(M, K, rank) + (in_type == MI355X_MX4 ? 0 : M * mx4_row_bytes_of(K));
  return MI355X_OK;
}

int mi355x_mx4_fc_adapters(void *out, int out_type, size_t out_row_bytes, const void *in, int in_type, size_t in_row_bytes,
                           const uint8_t *weights, size_t weights_row_bytes, const float *bias,
                           const mi355x_mx4_adapters *adapters, const int32_t *row_adapters, size_t M, size_t K, size_t N,
                           int activation, void *workspace, size_t workspace_bytes, void *stream) {
  MI355X_REQUIRE(adapters, "mx4_fc_adapters: no adapters");
  const size_t rank = adapters->rank, count = adapters->count;
  MI355X_REQUIRE(float_type(adapters->type), "mx4_fc_adapters: adapters' type %d is none of the float types", adapters->type);
  size_t need;
  if (int rc = mi355x_mx4_fc_adapters_workspace_bytes(M, K, N, in_type, rank, &need)) return rc;
  if (int rc = check_rows("mx4_fc_adapters: result", out, out_type, out_row_bytes, M, N)) return rc;
  if (int rc = check_rows("mx4_fc_adapters: input", in, in_type, in_row_bytes, M, K)) return rc;
  if (int rc = check_rows("mx4_fc_adapters: weights", weights, MI355X_MX4, weights_row_bytes, N, K)) return rc;
  MI355X_REQUIRE(activation == MI355X_ACT_NONE || activation == MI355X_ACT_RELU || activation == MI355X_ACT_SILU,
                 "mx4_fc_adapters: activation %d: none, Relu and SiLU are supported", activation);
  MI355X_REQUIRE((uintptr_t)bias % 4 == 0, "mx4_fc_adapters: the bias has to lie on a multiple of 4");
  if (!M || !N) return MI355X_OK;
  if (!rank || !count || !K)                       // nothing beside the product
    return mi355x_mx4_fc(out, out_type, out_row_bytes, in, in_type, in_row_bytes, weights, weights_row_bytes, bias, M, K, N,
                         activation, workspace, workspace_bytes, stream);
  if (K > kMostColumns) return fail(MI355X_ERR_NOT_SUPPORTED, "mx4_fc_adapters: %zu columns, up to %zu are supported", K, kMostColumns);
  const size_t size = float_size(adapters->type);
  MI355X_REQUIRE(count <= 0x7fffffff, "mx4_fc_adapters: %zu adapters", count);
  MI355X_REQUIRE(adapters->down && adapters->up && row_adapters, "mx4_fc_adapters: NULL");
  MI355X_REQUIRE((uintptr_t)adapters->down % size == 0 && (uintptr_t)adapters->up % size == 0,
                 "mx4_fc_adapters: the adapters have to lie on multiples of %zu", size);
  MI355X_REQUIRE((uintptr_t)row_adapters % 4 == 0 && (uintptr_t)adapters->scales % 4 == 0,
                 "mx4_fc_adapters: the rows' adapters and the scales have to lie on multiples of 4");
  const unsigned __int128 down_span = (unsigned __int128)count * rank * K * size,
                          up_span = (unsigned __int128)count * rank * N * size;
  MI355X_REQUIRE(down_span <= PTRDIFF_MAX && up_span <= PTRDIFF_MAX, "mx4_fc_adapters: %zu adapters of rank %zu", count, rank);
  const size_t out_span = rows_span(out_type, out_row_bytes, M, N), in_span = rows_span(in_type, in_row_bytes, M, K);
  const size_t w_span = rows_span(MI355X_MX4, weights_row_bytes, N, K);
  auto meets = [&](const void *a, size_t bytes) {
    return overlaps(a, bytes, in, in_span) || overlaps(a, bytes, weights, w_span) || overlaps(a, bytes, bias, 4 * N) ||
           overlaps(a, bytes, adapters->down, (size_t)down_span) || overlaps(a, bytes, adapters->up, (size_t)up_span) ||
           overlaps(a, bytes, adapters->scales, 4 * count) || overlaps(a, bytes, row_adapters, 4 * M);
  };
  MI355X_REQUIRE(!meets(out, out_span), "mx4_fc_adapters: the result overlaps what it is made from");
  MI355X_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0,
                 "mx4_fc_adapters: a workspace of %zu bytes on a multiple of 16 is needed "
                 "(mi355x_mx4_fc_adapters_workspace_bytes)", need);
  MI355X_REQUIRE(!meets(workspace, need) && !overlaps(workspace, need, out, out_span),
                 "mx4_fc_adapters: the workspace overlaps a tensor");

  hipStream_t st = as_stream(stream);
  MxDown d{};
  d.in = static_cast<const uint8_t *>(in);
  d.in_row_bytes = in_row_bytes;
  d.down = static_cast<const uint8_t *>(adapters->down);
  d.scales = adapters->scales;
  d.of_row = row_adapters;
  d.low = static_cast<float *>(workspace);
  d.packed = static_cast<uint8_t *>(workspace) + low_bytes(M, K, rank);
  d.packed_row_bytes = mx4_row_bytes_of(K);
  d.M = (int)M;
  d.K = (int)K;
  d.groups = (int)mx4_groups(K);
  d.rank = (int)rank;
  d.ranks = (int)((rank + 31) / 32 * 32);
  d.count = (int)count;
  d.row_tiles = (int)((M + 15) / 16);
  d.rank_tiles = d.ranks <= 32 ? 1 : (d.ranks + 63) / 64;
  d.turns = down_turns(M);
  d.parts = down_parts(M, K, rank);
  unsigned long long blocks = (unsigned long long)d.row_tiles * d.rank_tiles * d.turns * d.parts;
  if (in_type != MI355X_MX4) blocks += ((unsigned long long)M * d.groups + kDownThreads / 16 - 1) / (kDownThreads / 16);
  if (blocks > (1u << 22)) return fail(MI355X_ERR_NOT_SUPPORTED, "mx4_fc_adapters: %zu rows of %zu columns", M, K);
  if (in_type == MI355X_F32) down_launch_type<F32>(d, adapters->type, (unsigned)blocks, st);
  else if (in_type == MI355X_F16) down_launch_type<F16>(d, adapters->type, (unsigned)blocks, st);
  else if (in_type == MI355X_BF16) down_launch_type<BF16>(d, adapters->type, (unsigned)blocks, st);
  else down_launch_type<MX4>(d, adapters->type, (unsigned)blocks, st);
  if (int rc = check_launch("mx4_fc_adapters")) return rc;

  MxFcAdapted p{};
  p.in = in_type == MI355X_MX4 ? d.in : d.packed;
  p.in_row_bytes = in_type == MI355X_MX4 ? in_row_bytes : d.packed_row_bytes;
  p.out = static_cast<uint8_t *>(out);
  p.out_row_bytes = out_row_bytes;
  p.weights = weights;
  p.weights_row_bytes = weights_row_bytes;
  p.bias = bias;
  p.M = (int)M;
  p.N = (int)N;
  p.groups = d.groups;
  p.out_groups = (int)mx4_groups(N);
  p.act = activation;
  p.ad.up = static_cast<const uint8_t *>(adapters->up);
  p.ad.low = d.low;
  p.ad.of_row = row_adapters;
  p.ad.type = adapters->type;
  p.ad.rank = d.rank;
  p.ad.ranks = d.ranks;
  p.ad.count = d.count;
  p.ad.parts = d.parts;
  const FcTile tile = fc_tile((long long)M, (long long)K, (long long)N, out_type == MI355X_MX4);
  const int k = (int)K;
  if (out_type == MI355X_F32) return adapted_launch<F32>(p, k, tile, st);
  if (out_type == MI355X_F16) return adapted_launch<F16>(p, k, tile, st);
  if (out_type == MI355X_BF16) return adapted_launch<BF16>(p, k, tile, st);
  return adapted_launch<MX4>(p, k, tile, st);
}

} // extern "C"
