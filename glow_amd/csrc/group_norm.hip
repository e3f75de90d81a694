// Group norm with an activation over channels-last tensors.
//
// Values x[n][p][c]; a group is C / groups neighbouring channels over all pixels of a
// sample: y = act((x - mean) / sqrt(variance + epsilon) * gamma[c] + beta[c]).
//
// A slice is some neighbouring groups of a sample, 128 bytes of a pixel if they give as
// much: whole lines. A thread holds eight channels of every stride-th pixel, a power of two
// of neighbouring lanes the slice's channels, so that a thread's channels never change.
// Two ways:
//   resident  a workgroup reads a slice into its registers (up to 64 a thread: 256 KB a
//             workgroup, half of a CU's), finds mean and variance, and writes it: one launch,
//             every value read once
//   in parts  slices that do not fit, or too few of them to fill the chip: one launch
//             leaves mean and sum of squares of every part of a slice's pixels in the
//             workspace, a second joins them and writes
// All sums are of distances: from the group's first value, the pivot, and with that a thread's mean;
// then the squares of what the thread's values are off its mean, and what that is off the whole's.
// So the error goes by how far a group's values lie from each other, whatever the mean is. That is
// kept as its rounding and the rest of it, and a value loses the first before it is scaled. (Slices of
// over 8192 channels, a third way: sums in 64 bits.)
//
// us: 64 x 3136 x 256 of fp16 55 (206 MB, 3.8 TB/s: 40 at the rate of a large copy; a workgroup fills a
// CU and reads, computes and writes in turn), 32 x 784 x 512 of bf16 with SiLU to microscaled rows 16.6
// (32 MB; 14.4 without SiLU: all CUs read, then compute, then write), 1 x 49 x 512 4.5 (the launch and
// two rounds of sums), 4 x 16384 x 128 in parts 18, 3 x 1225 x 100 of fp32 in parts 9.6 (two launches).
// Distances instead of values cost 0 to 6 % of these; the times beside gn_plan's rules are of
// before, on both sides.
#include "mx4.h"

#include <algorithm>

namespace mi355x {

struct alignas(16) GroupStats {
  float mean, square;     // of a part: sum of the squares of what is left of the mean
  float low;              // what the mean's rounding left out
  float unused;           // (one load of sixteen bytes)
};
struct GroupNorm {
  uint8_t *out;
  const uint8_t *in;
  size_t out_row_bytes, in_row_bytes;
  const float *gamma, *beta;
  GroupStats *stats;      // [N][groups][chunks]
  int pixels, C, groups, per;
  float epsilon;
  int act;
  int samples;            // of this launch
  // a slice is `in_slice` groups, `width` channels; 2^lg_vec lanes hold one pixel of it
  int in_slice, width, slices, lg_vec;
  int chunks, chunk_pixels;
  int by_die;             // neighbouring slices of a sample on one die
  int channel_groups;     // of a microscaled result's row
  size_t mx4_bytes;       // of its row
};

enum { kGnResident, kGnStats, kGnApply };
constexpr int kGnMost = 1024;         // threads of a workgroup
constexpr int kGnMostChunks = 128;    // parts of a slice

// The group of a channel, and of those behind it (a division for each of eight costs more than
// the statistics do).
struct GnGroup {
  int group, in;
  __device__ __forceinline__ GnGroup(int channel, int per)
      : group((int)((unsigned)channel / (unsigned)per)), in(channel - group * per) {}
  __device__ __forceinline__ void next(int per) {
    if (++in == per) in = 0, group++;
  }
};

// Sums over a wave in 64 bits.
template <int N> __device__ __forceinline__ double add_rotated(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b, 0x120 + N, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), 0x120 + N, 0xf, 0xf, true);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double add_across16(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
}
__device__ __forceinline__ double add_across32(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
}
__device__ __forceinline__ double wave_sum(double x) {
  x = add_rotated<1>(add_rotated<2>(add_rotated<4>(add_rotated<8>(x))));
  return add_across32(add_across16(x));
}

// Sums over a slice's pixels and a group's channels: done(g, sum) of each of the slice's groups, in one
// thread. A thread's eight channels are NP parts that each lie in one group: one where groups are
// whole vectors, two (the first channels and the rest) where a vector meets two groups at most,
// else one for each channel. x[i] is the sum over part i, its place in a row of s_part `at` + i;
// parts before `from` are another thread's. Lanes of a wave that hold the same channels are summed
// first, then a wave takes a group, always in 64 bits. X: double where roundings of the lanes' sums
// would be seen, in those that give means of one or two parts (as floats, a mean of 600 values is off
// by 6 * 10^-8 of their spread, else by 10^-8; 1% of the time of small calls).
template <int NP, class X, class Done>
__device__ __forceinline__ void gn_reduce(X (&x)[NP], X *s_part, int at, int from, int groups,
                                          const GroupNorm &p, Done &&done) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = (int)blockDim.x >> 6;
  const int V = 1 << p.lg_vec;
#pragma unroll
  for (int j = 0; j < NP; j++) {
    if (V <= 8) x[j] = add_rotated<8>(x[j]);
    if (V <= 4) x[j] = add_rotated<4>(x[j]);
    if (V <= 2) x[j] = add_rotated<2>(x[j]);
    if (V <= 1) x[j] = add_rotated<1>(x[j]);
    if (V <= 16) x[j] = add_across16(x[j]);
    if (V <= 32) x[j] = add_across32(x[j]);
  }
  const int rows = V < 64 ? waves : (int)blockDim.x >> p.lg_vec;
  if (V >= 64 || lane < V) {
    const int row = V < 64 ? wave : tid >> p.lg_vec;
#pragma unroll
    for (int j = 0; j < NP; j++)
      if (NP < 8 || j >= from) s_part[(row << p.lg_vec) * NP + at + j] = x[j];
  }
  __syncthreads();
  // many small groups: a thread each, instead of wave after wave
  const int most = NP == 8 ? p.per : (p.per + 6) / 8 + 1;
  const bool thread_each = groups > waves && most * rows <= 32;
  for (int g = thread_each ? tid : wave; g < groups; g += thread_each ? (int)blockDim.x : waves) {
    // a group's parts in a row: `len` of them from `begin` on, `apart` places from each other; where
    // it begins within a vector, the first is that vector's second part
    const int channel = g * p.per;
    const int begin = NP == 8 ? channel : (channel >> 3) * NP, apart = NP == 2 ? 2 : 1;
    const int inner = NP == 2 && (channel & 7) ? 1 : 0;
    const int len = NP == 8 ? p.per : ((channel + p.per - 1) >> 3) - (channel >> 3) + 1;
    double t = 0;
    if (thread_each) {
      for (int row = 0; row < rows; row++)
        for (int k = 0; k < len; k++) t += s_part[(row << p.lg_vec) * NP + begin + k * apart + (k == 0 ? inner : 0)];
      done(g, t);
      continue;
    }
    if (len < 64) {
      for (int e = lane; e < len * rows; e += 64) {
        const int row = (int)((unsigned)e / (unsigned)len), k = e - row * len;
        t += s_part[(row << p.lg_vec) * NP + begin + k * apart + (k == 0 ? inner : 0)];
      }
    } else {
      for (int row = 0; row < rows; row++)
        for (int k = lane; k < len; k += 64)
          t += s_part[(row << p.lg_vec) * NP + begin + k * apart + (k == 0 ? inner : 0)];
    }
    t = wave_sum(t);
    if (lane == 0) done(g, t);
  }
  __syncthreads();
}

// 1 / (pixels * per) to 40 bits and more.
__device__ __forceinline__ double gn_over(int pixels, int per) {
  const double n = (double)pixels * per, r = __builtin_amdgcn_rcpf((float)n);
  return fma(fma(-n, r, 1.0), r, r);
}

// base + rest, rounded, and what the rounding left out: exact where the base is no smaller than the
// rest, else off by a rounding of the rest.
struct GnMean {
  float high, low;
  __device__ __forceinline__ GnMean(float base, float rest) : high(base + rest), low(rest - (high - base)) {}
  __device__ __forceinline__ GnMean(float base, double rest)
      : high((float)(base + rest)), low((float)(rest - ((double)high - base))) {}
};

// A thread's sums, of up to 128 values at a time, of what they are from the pivot. 32-bit values lose
// that one by one. 16-bit ones are summed as they are, kGnShare of each, so that no sum is
// past 32 bits: where they are so near to each other that the pivot matters, they are multiples of one
// step whose sum has 11 + 7 bits and few more, and the pivot is taken off it without a rounding (gn_rest).
constexpr float kGnShare = 1.0f / 128;
template <class E> __device__ __forceinline__ float gn_add(float sum, const typename E::Eight &e, int j, float pivot) {
  if constexpr (E::kSize == 4) return sum + (e[j] - pivot);
  else return fmaf(E::get(e, j), kGnShare, sum);
}
// The same of eight values: of 16-bit types two to an instruction, of others in pairs.
template <class E> __device__ __forceinline__ float gn_sum8(float sum, const typename E::Eight &e, float pivot) {
  if constexpr (std::is_same_v<E, F16>) {
    typedef _Float16 Two __attribute__((ext_vector_type(2)));
    const _Float16 share = (_Float16)kGnShare;
#pragma unroll
    for (int i = 0; i < 4; i++)
      sum = __builtin_amdgcn_fdot2(Two{e[2 * i], e[2 * i + 1]}, Two{share, share}, sum, false);
  } else if constexpr (std::is_same_v<E, BF16>) {
    typedef __bf16 Two __attribute__((ext_vector_type(2)));
    const __bf16 share = (__bf16)kGnShare;
#pragma unroll
    for (int i = 0; i < 4; i++)
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(Two, (uint32_t)e[i]), Two{share, share}, sum, false);
  } else {
    const auto two = [&](int j) { return (e[j] - pivot) + (e[j + 1] - pivot); };
    sum += (two(0) + two(2)) + (two(4) + two(6));
  }
  return sum;
}
// What `count` values of such a sum are from the pivot in all.
template <class E> __device__ __forceinline__ float gn_rest(float sum, float count, float pivot) {
  if constexpr (E::kSize == 4) return sum;
  else return fmaf(-count * kGnShare, pivot, sum) * (1.0f / kGnShare);
}
// x - mean of a value; of fp16 one instruction with the widening (`one` hides a factor of 1 that
// would be taken out of it).
template <class E> __device__ __forceinline__ float gn_less(const typename E::Eight &e, int j, float mean, float one) {
  if constexpr (std::is_same_v<E, F16>) return fmaf((float)e[j], one, -mean);
  else return E::get(e, j) - mean;
}

// Writes one pixel's eight channels.
template <class E, class OUT, int ACT, int NM>
__device__ __forceinline__ void gn_write(uint8_t *row, int c, int left, int twice, bool block_inside,
                                         const typename E::Eight &raw, const float (&mean)[NM],
                                         const float (&scale)[8], const float (&shift)[8], float one,
                                         const GroupNorm &p) {
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; j++)
    y[j] = activate<ACT>(fmaf(gn_less<E>(raw, j, mean[NM == 1 ? 0 : j], one), scale[j], shift[j]));
  if constexpr (OUT::kSize == 0) {
    if (__ballot(left < 8)) {        // (a branch, not a selection for every value of every pixel)
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = j < left ? y[j] : 0.0f;
    }
    const uint32_t byte = mx4_scale_byte(quad_max(largest8(y)));
    if (block_inside) {
      *reinterpret_cast<uint32_t *>(row + (c >> 1)) = mx4_codes8(y, byte);
      if ((c & 31) == 0) row[(size_t)p.channel_groups * kMxGroupBytes + (c >> 5)] = (uint8_t)byte;
    }
  } else {
    // (two lanes of a wave that store the same channels store the same bits; lanes of two waves may
    // not, in place: one may not have read yet what the other overwrites)
    typename OUT::T *o = reinterpret_cast<typename OUT::T *>(row) + c;
    if (left >= 8 && (twice == 0 || p.lg_vec <= 6)) store8<OUT>(o, y);
    else
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j >= twice && j < left) o[j] = OUT::from(y[j]);
  }
}

// what the sums that give means are held in, between lanes
template <int NP> using GnWide = std::conditional_t<NP <= 2, double, float>;

template <class E, class OUT, int R, int MODE, int NP>
__global__ __launch_bounds__(kGnMost) void group_norm_kernel(GroupNorm p) {
  typedef GnWide<NP> Wide;
  extern __shared__ __attribute__((aligned(16))) float s_mem[];
  // of each group: its mean's rounding and the rest, 1 / sqrt(variance + epsilon), and a mean on the way
  float *s_group = s_mem, *s_low = s_mem + p.in_slice, *s_second = s_mem + 2 * p.in_slice;
  float *s_rest = s_mem + 3 * p.in_slice, *s_part = s_mem + 4 * ((p.in_slice + 1) & ~1);
  const int tid = threadIdx.x, V = 1 << p.lg_vec;
  const int v = tid & (V - 1), first = tid >> p.lg_vec, stride = (int)blockDim.x >> p.lg_vec;

  unsigned id = blockIdx.x;
  const int chunk = (int)(id % (unsigned)p.chunks);
  id /= (unsigned)p.chunks;
  int sample, slice;
  if (p.by_die) {            // consecutive workgroups are dealt over the eight dies
    const unsigned die = id & 7, at = id >> 3;
    sample = (int)(die + 8 * (at / (unsigned)p.slices));
    slice = (int)(at % (unsigned)p.slices);
    if (sample >= p.samples) return;
  } else {
    sample = (int)(id / (unsigned)p.slices);
    slice = (int)(id % (unsigned)p.slices);
  }
  const int c0 = slice * p.width, c_end = min(p.C, c0 + p.width);
  // The last vector of a slice that is no whole number of them begins earlier and overlaps the one in
  // front (a load of eight instead of eight of one, for the whole wave); `twice` channels are that
  // one's in the statistics. Blocks of microscaled rows begin where they begin.
  int c = c0 + v * 8;
  const int twice = NP > 1 && OUT::kSize && c < c_end && c_end - c0 >= 8 ? max(0, c + 8 - c_end) : 0;
  c -= twice;
  const int left = c_end - c;
  const int px0 = chunk * p.chunk_pixels, px_end = px0 + min(p.chunk_pixels, p.pixels - px0);
  const uint8_t *in = p.in + (size_t)sample * p.pixels * p.in_row_bytes + (ptrdiff_t)c * E::kSize;

  typename E::Eight raw[R];
  auto load = [&](int from) {
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int px = from + first + i * stride;
      if (first + i * stride < px_end - from) {
        const typename E::T *at = reinterpret_cast<const typename E::T *>(in + (size_t)px * p.in_row_bytes);
        if (left >= 8) raw[i] = load_eight<E>(at);
        else raw[i] = load_eight_end<E>(at, left);
      }
    }
  };
  // pixels of this thread among those of a block that begins at `from`
  auto mine = [&](int from) {
    const int rest = px_end - from - first;
    return left > 0 && rest > 0 ? min(R, (rest - 1) / stride + 1) : 0;
  };
  const int block = R * stride;
  const float of_group = (float)p.per;
  const int groups = (c_end - c0) / p.per;

  load(px0);
  float scale[8], shift[8];
  auto load_affine = [&]() {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      scale[j] = p.gamma && j < left ? p.gamma[c + j] : 1.0f;
      shift[j] = p.beta && j < left ? p.beta[c + j] : 0.0f;
    }
  };
  // asked for with the values, ahead of the statistics, where registers are left for it
  constexpr bool kAffineAhead = R < 16 && (R * E::kSize < 32 || NP == 1);
  if constexpr (MODE != kGnStats && kAffineAhead) load_affine();
  float one = 1.0f;
  asm("" : "+s"(one));
  if constexpr (MODE != kGnApply) {
    // The groups of a thread's parts: f(part, its group, the part's place in it). (Their division is made
    // here, while the values are on their way.)
    GnGroup own(NP == 8 ? c - c0 : v * 8, p.per);
    asm volatile("" : "+v"(own.group), "+v"(own.in));
    auto parts = [&](auto &&f) {
      GnGroup of = own;
#pragma unroll
      for (int j = 0; j < NP; j++) {
        f(j, min(of.group, groups - 1), of.in);
        if (NP == 8) of.next(p.per);
        else of.group++, of.in = 0;
      }
    };
    // a group's pivot is its first channel of the sample's first pixel, whichever part of a slice this is
    const typename E::T *pixel = reinterpret_cast<const typename E::T *>(
        p.in + (size_t)sample * p.pixels * p.in_row_bytes) + c0;
    float pivot[NP];
    parts([&](int j, int g, int) { pivot[j] = E::to(pixel[g * p.per]); });
    // a thread's own counts (exact: a part of a slice has 2^24 pixels at most), means and squares.
    // Channel j belongs to part `j >= border` of two, to its own of eight.
    const int border = NP == 2 && left > 0 ? min(8, twice + p.per - own.in) : 8;
    const int channels_lo = border - twice, channels_hi = 8 - border;
    // (sum and mean are of distances from the pivot; eight parts have one count, and no registers for
    // sums as well)
    constexpr int NC = NP == 8 ? 1 : NP;
    float count[NC], sum[NC], mean[NP], square[NP];
#pragma unroll
    for (int j = 0; j < NP; j++) count[j % NC] = sum[j % NC] = mean[j] = square[j] = 0;
    // (the end of the sums finds them in s_low)
    if (first == 0 && left > 0)
      parts([&](int j, int g, int in) {
        if (in == 0 && (NP == 2 ? j == 0 || border < min(8, left) : NP == 1 || (j >= twice && j < left))) s_low[g] = pivot[j];
      });
    for (int from = px0;;) {
      const int n = mine(from);
      if (n > 0) {
        constexpr int NA = NP == 1 ? 1 : 8;       // sums in the loop over pixels
        float m[NA], q[NA], here[NC], all[NP], own[NP], rest[NP];
#pragma unroll
        for (int j = 0; j < NA; j++) m[j] = q[j] = 0;
#pragma unroll
        for (int i = 0; i < R; i++)
          if (i < n) {
            if constexpr (NP == 1) m[0] = gn_sum8<E>(m[0], raw[i], pivot[0]);
            else {
#pragma unroll
              for (int j = 0; j < 8; j++)
                m[j] = gn_add<E>(m[j], raw[i], j, NP == 8 ? pivot[j] : j < border ? pivot[0] : pivot[1]);
            }
          }
        if constexpr (NP == 1) {
          here[0] = (float)n * 8;
          all[0] = gn_rest<E>(m[0], here[0], pivot[0]);
        } else if constexpr (NP == 2) {
          here[0] = (float)(n * channels_lo);
          here[1] = (float)(n * channels_hi);
          float lo = 0, hi = 0;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            lo += j >= twice && j < border ? m[j] : 0.0f;
            hi += j >= border ? m[j] : 0.0f;
          }
          all[0] = gn_rest<E>(lo, here[0], pivot[0]);
          all[1] = gn_rest<E>(hi, here[1], pivot[1]);
        } else {
          here[0] = (float)n;
#pragma unroll
          for (int j = 0; j < 8; j++) all[j] = gn_rest<E>(m[j], here[0], pivot[j]);
        }
#pragma unroll
        for (int j = 0; j < NP; j++) own[j] = j == 1 && NP == 2 && !channels_hi ? 0.0f : all[j] * (1.0f / here[j % NC]);
        // the squares are of the distances from the mean's rounding, and less of what that is off
        float low[NP];
#pragma unroll
        for (int j = 0; j < NP; j++) {
          const GnMean center(pivot[j], own[j]);
          low[j] = center.low;
          if constexpr (NP == 2) {
#pragma unroll
            for (int k = 0; k < 8; k++)
              if (j == 0 || k >= border) m[k] = center.high;
          } else m[j] = center.high;
        }
#pragma unroll
        for (int i = 0; i < R; i++)
          if (i < n)
#pragma unroll
            for (int j = 0; j < 8; j++) {
              const float d = gn_less<E>(raw[i], j, m[NP == 1 ? 0 : j], one);
              q[NP == 1 ? 0 : j] = fmaf(d, d, q[NP == 1 ? 0 : j]);
            }
        if constexpr (NP == 2) {
          rest[0] = rest[1] = 0;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            rest[0] += j >= twice && j < border ? q[j] : 0.0f;
            rest[1] += j >= border ? q[j] : 0.0f;
          }
        } else {
#pragma unroll
          for (int j = 0; j < NP; j++) rest[j] = q[j];
        }
#pragma unroll
        for (int j = 0; j < NP; j++) {
          rest[j] = fmaf(-low[j] * low[j], here[j % NC], rest[j]);
          rest[j] = rest[j] < 0 ? 0.0f : rest[j];    // (NaN stays)
          if (MODE == kGnResident || count[j % NC] == 0) {
            mean[j] = own[j], square[j] = rest[j];
          } else {           // joins two sets: the squares of each, and of what their means are apart
            const float part = here[j % NC] / (count[j % NC] + here[j % NC]), d = own[j] - mean[j];
            mean[j] = fmaf(d, part, mean[j]);
            square[j] += fmaf(d * d, count[j % NC] * part, rest[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < NC; j++) count[j] += here[j], sum[j] += all[j];
      }
      if (MODE == kGnResident || px_end - from <= block) break;
      from += block;
      load(from);
    }
    const int at = NP == 8 ? c - c0 : v * NP;
    Wide wide[NP];
#pragma unroll
    for (int j = 0; j < NP; j++) wide[j] = NP == 8 ? mean[j] * count[0] : sum[j % NC];
    gn_reduce<NP>(wide, reinterpret_cast<Wide *>(s_part), at, twice, groups, p, [&](int g, double all) {
      const double rest = all * gn_over(px_end - px0, p.per);
      const GnMean m(s_low[g], rest);
      s_rest[g] = (float)rest;
      s_group[g] = m.high;
      s_low[g] = m.low;
    });
    float x[NP];
    parts([&](int j, int g, int) {
      const float d = mean[j] - s_rest[g];
      x[j] = count[j % NC] > 0 ? fmaf(d * d, count[j % NC], square[j]) : 0.0f;
    });
    gn_reduce<NP>(x, s_part, at, twice, groups, p, [&](int g, double all) {
      if constexpr (MODE == kGnStats)
        p.stats[((size_t)sample * p.groups + slice * p.in_slice + g) * p.chunks + chunk] =
            GroupStats{s_group[g], (float)all, s_low[g], 0};
      else s_second[g] = 1.0f / sqrtf((float)(all * gn_over(px_end - px0, p.per)) + p.epsilon);
    });
    if (MODE == kGnStats) return;
  } else {
    // joins the parts: what their means are from the first one's, then their squares and what their
    // means are off the whole's
    const int lane = tid & 63, wave = tid >> 6, waves = (int)blockDim.x >> 6;
    const double over = gn_over(p.pixels, p.per);
    for (int g = wave; g < groups; g += waves) {
      const GroupStats *s = p.stats + ((size_t)sample * p.groups + slice * p.in_slice + g) * p.chunks;
      GroupStats own[kGnMostChunks / 64];
#pragma unroll
      for (int i = 0; i < kGnMostChunks / 64; i++) {
        const int k = lane + 64 * i;
        if (k < p.chunks) own[i] = s[k];
      }
      const float pivot = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(own[0].mean)));
      float mean[kGnMostChunks / 64], square[kGnMostChunks / 64];
      double m = 0, q = 0;
      auto values = [&](int k) {     // of part k
        return (float)min(p.chunk_pixels, p.pixels - min(k, p.chunks - 1) * p.chunk_pixels) * of_group;
      };
#pragma unroll
      for (int i = 0; i < kGnMostChunks / 64; i++) {
        const int k = lane + 64 * i;
        mean[i] = (own[i].mean - pivot) + own[i].low;
        square[i] = own[i].square;
        if (k < p.chunks) m = fma((double)mean[i], (double)values(k), m);
      }
      m = wave_sum(m) * over;
#pragma unroll
      for (int i = 0; i < kGnMostChunks / 64; i++) {
        const int k = lane + 64 * i;
        const float d = mean[i] - (float)m;
        if (k < p.chunks) q += fmaf(d * d, values(k), square[i]);
      }
      q = wave_sum(q);
      if (lane == 0) {
        const GnMean all(pivot, m);
        s_group[g] = all.high;
        s_low[g] = all.low;
        s_second[g] = 1.0f / sqrtf((float)(q * over) + p.epsilon);
      }
    }
    __syncthreads();
  }

  if constexpr (!kAffineAhead) load_affine();
  constexpr int NM = NP == 1 ? 1 : 8;
  float mean[NM];
  GnGroup of(c - c0, p.per);
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int g = j < left ? of.group : 0;
    if (NM == 8 || j == 0) mean[NM == 1 ? 0 : j] = s_group[g];
    scale[j] *= s_second[g];
    shift[j] = fmaf(-s_low[g], scale[j], shift[j]);
    if (NM == 8) of.next(p.per);
  }
  uint8_t *out = p.out + (size_t)sample * p.pixels * p.out_row_bytes;
  // microscaled: lanes up to the end of the slice's last block
  const bool inside = OUT::kSize ? left > 0 : c < ((c_end + 31) & ~31);
  auto write = [&](int from, auto act) {
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int px = from + first + i * stride;
      if (first + i * stride < px_end - from && (OUT::kSize == 0 || inside))
        gn_write<E, OUT, decltype(act)::value, NM>(out + (size_t)px * p.out_row_bytes, c, left, twice, inside, raw[i], mean,
                                                   scale, shift, one, p);
    }
  };
  for (int from = px0;;) {
    with_activation(p.act, [&](auto act) { write(from, act); });
    if (MODE == kGnResident || px_end - from <= block) break;
    from += block;
    load(from);
  }
  if constexpr (OUT::kSize == 0) {
    // what lies behind the last block of a row: codes and scales of blocks past C, and the end
    if (c_end == p.C) {
      const int blocks = (p.C + 31) / 32, codes = p.channel_groups * kMxGroupBytes;
      const int tail = codes + blocks, tail_end = (int)p.mx4_bytes;
      for (int at = first; at < px_end - px0; at += stride) {
        uint8_t *row = out + (size_t)(px0 + at) * p.out_row_bytes;
        for (int b = blocks * 16 + v * 4; b < codes; b += V * 4) *reinterpret_cast<uint32_t *>(row + b) = 0;
        for (int b = tail + v; b < tail_end; b += V) row[b] = 0;
      }
    }
  }
}

// Slices too wide for a workgroup's lanes, over 8192 channels (a group of that many, or 32 of an odd
// number each to microscaled rows): a workgroup reads a group once, then sixteen lanes take 128
// channels of a pixel.
//
// A thread's sums run over up to every 256th value of a group, too many for 32 bits: they are held in
// 64, of the values' distances from the group's first one and of the squares of these. That one
// is sqrt(values of the group) deviations from the mean at most, so that the difference of the
// two sums loses log2(values) of their 53 bits at worst. One workgroup a group, one value a load:
// 1 x 784 x 16384 of fp16 in one group 13.4 ms, bound by the time that loads take to arrive.
constexpr int kGnWideThreads = 256;

template <class E>
__global__ __launch_bounds__(kGnWideThreads) void group_norm_wide_stats_kernel(GroupNorm p) {
  __shared__ double s_sum[kGnWideThreads], s_square[kGnWideThreads];
  const int tid = threadIdx.x;
  const int group = (int)(blockIdx.x % (unsigned)p.groups);
  const size_t sample = blockIdx.x / (unsigned)p.groups;
  const uint8_t *base = p.in + sample * p.pixels * p.in_row_bytes + (size_t)group * p.per * E::kSize;
  const double pivot = E::to(*reinterpret_cast<const typename E::T *>(base));
  double sum = 0, square = 0;
  for (int px = 0; px < p.pixels; px++) {
    const typename E::T *row = reinterpret_cast<const typename E::T *>(base + (size_t)px * p.in_row_bytes);
    for (int i = tid; i < p.per; i += kGnWideThreads) {
      const double d = (double)E::to(row[i]) - pivot;
      sum += d;
      square = fma(d, d, square);
    }
  }
  s_sum[tid] = sum;
  s_square[tid] = square;
  for (int half = kGnWideThreads / 2; half > 0; half /= 2) {
    __syncthreads();
    if (tid < half) {
      s_sum[tid] += s_sum[tid + half];
      s_square[tid] += s_square[tid + half];
    }
  }
  if (tid == 0) {
    const double n = (double)p.pixels * p.per, rest = s_sum[0] / n, mean = pivot + rest;
    double variance = s_square[0] / n - rest * rest;
    variance = variance < 0 ? 0 : variance;          // (NaN stays)
    const float high = (float)mean;
    // (what is left of the mean is taken from its parts: their sum is rounded too)
    p.stats[blockIdx.x] = GroupStats{high, (float)(1.0 / sqrt(variance + p.epsilon)), (float)(rest - (high - pivot)), 0};
  }
}

template <class E, class OUT>
__global__ __launch_bounds__(kGnWideThreads) void group_norm_wide_apply_kernel(GroupNorm p, unsigned long long units) {
  const int l = threadIdx.x & 15;
  for (unsigned long long u = blockIdx.x * 16ull + (threadIdx.x >> 4); u < units; u += gridDim.x * 16ull) {
    const size_t row = u / (unsigned)p.channel_groups;
    const int g = (int)(u % (unsigned)p.channel_groups), c = g * kMxGroup + l * 8;
    const typename E::T *in = reinterpret_cast<const typename E::T *>(p.in + row * p.in_row_bytes) + c;
    const int left = p.C - c;
    float x[8];
    if (left >= 8) load8<E>(x, in);
    else load8_end<E>(x, in, left);
    const GroupStats *stats = p.stats + row / (unsigned)p.pixels * p.groups;
    with_activation(p.act, [&](auto act) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (j < left) {
          const GroupStats s = stats[(c + j) / p.per];
          const float scale = s.square * (p.gamma ? p.gamma[c + j] : 1.0f);
          const float shift = fmaf(-s.low, scale, p.beta ? p.beta[c + j] : 0.0f);
          x[j] = activate<decltype(act)::value>(fmaf(x[j] - s.mean, scale, shift));
        }
      }
    });
    uint8_t *out = p.out + row * p.out_row_bytes;
    if constexpr (OUT::kSize == 0) {
      mx4_store_group<F32>(out, p.channel_groups, g, l, F32::put(x));
    } else if (left > 0) {
      typename OUT::T *o = reinterpret_cast<typename OUT::T *>(out) + c;
      if (left >= 8) store8<OUT>(o, x);
      else store8_end<OUT>(o, x, left);
    }
  }
}

// ---- how a call is cut -------------------------------------------------------------

// The most parts that a slice of this call may be cut into, whatever its types: what the workspace has
// room for.
static int gn_most_chunks(size_t N, size_t pixels) {
  const size_t n = N < 1024 ? 1024 / N : 1;
  return (int)std::min<size_t>({n, pixels, (size_t)kGnMostChunks});
}

// Parts of a thread's eight channels that lie in one group each (gn_reduce).
static int gn_parts(int per) { return per % 8 == 0 ? 1 : per >= 7 || per == 4 ? 2 : 8; }
struct GnPlan {
  bool wide, resident;
  int threads, regs;      // pixels a thread holds at a time
};
static GnPlan gn_plan(GroupNorm &p, size_t N, int size, bool mx4) {
  GnPlan plan{};
  // a slice that is written as blocks begins with one
  int unit = 1;
  if (mx4)
    while (unit < 32 && (long long)unit * p.per % 32) unit *= 2;
  unit = std::min(unit, p.groups);
  // slices that share lines run on one die, whose L2 then has the line whole
  const bool by_die = N >= 8;
  int k = unit;
  while (k < p.groups && (long long)k * p.per * size < (by_die ? 64 : 128)) k = std::min(k + unit, p.groups);
  auto set = [&](int groups) {
    p.in_slice = groups;
    p.width = (int)std::min<long long>((long long)groups * p.per, 0x7fffffff);
    p.slices = (p.groups + groups - 1) / groups;
    p.lg_vec = mx4 ? 2 : 0;
    while (p.lg_vec < 11 && (8 << p.lg_vec) < p.width) p.lg_vec++;
  };
  set(k);
  if (p.lg_vec > 10) {
    plan.wide = true;
    return plan;
  }
  // (as many as leave room for the sums: one for a thread, two parts, or eight)
  const int parts = gn_parts(p.per);
  const int most_regs = size == 2 ? (parts == 1 ? 16 : 8) : (parts == 8 ? 4 : 8);
  auto fits = [&] { return p.pixels <= (long long)(kGnMost >> p.lg_vec) * most_regs; };
  // Narrower slices where they are too few for the chip, or too large for a workgroup: as many lines
  // are asked for then, and less is used of each (64 x 3136 x 256 of fp16, slices of 64 / 32 / 16
  // bytes: 53 / 64 / 82 us), but the launch in front that parts need is saved (26 x 2733 x 32 of bf16:
  // 16 bytes on one die 10.7, in parts 18.1; 7 x 870 x 96 of fp16: 24 bytes 10.2, 66 bytes 15.8; 1 x
  // 3136 x 256 of fp16 over all dies: 16 bytes 12.7, in parts 9.1).
  // A vector of eight channels is the least (16 x 3136 x 40 of fp32 in 8 groups: 20 bytes 26, in parts 18).
  const int wide = k, least = by_die ? 8 * size : std::max(24, 8 * size);
  while (k > unit && (long long)(k / 2 / unit * unit) * p.per * size >= least &&
         ((long long)N * p.slices < 256 || !fits())) {
    k = std::max(unit, k / 2 / unit * unit);
    set(k);
  }
  // Few large slices leave most of the chip idle. us, resident / in parts: 1 x 3136 x 256 of fp16 in 16
  // slices of 100 KB 9.8 / 9.1, 4 x 52 x 626 in 4 of 65 KB 17.0 / 10.2, 4 x 268 x 260 in 16 of 35 KB 12.6 /
  // 10.3; 1 x 784 x 512 in 32 of 25 KB 6.7 / 9.6.
  const long long all = (long long)N * p.slices, bytes = (long long)p.pixels * p.width * size;
  plan.resident = fits() && (all >= 128 || bytes <= 16 * 1024 || (all >= 24 && bytes <= 32 * 1024));
  if (plan.resident) {
    // few pixels a thread as long as the workgroup is small, so that several share a CU (32 x 784 x
    // 512, microscaled, 64 bytes: 512 threads of eight pixels 16.3 us, 1024 of four 19.7)
    plan.threads = std::max(64, 1 << p.lg_vec);
    plan.regs = 1;
    auto holds = [&] { return (long long)(plan.threads >> p.lg_vec) * plan.regs; };
    while (holds() < p.pixels) {
      if (plan.regs < 4 || (plan.threads >= 512 && plan.regs < std::min(8, most_regs)) || plan.threads >= kGnMost)
        plan.regs *= 2;
      else plan.threads *= 2;
    }
    p.chunks = 1;
    p.chunk_pixels = p.pixels;
    return plan;
  }
  // In parts: slices of 64 bytes, a workgroup for each CU (4 x 16384 x 128 of fp16: 16 parts of 64
  // bytes 17.7 us, 64 parts of 128 bytes 20.5, 128 parts 26; the second launch reads all parts of
  // its slice), smaller ones where that leaves a workgroup less than four pixels a thread.
  k = unit;
  while (k < wide && (long long)k * p.per * size < 64) k = std::min(k + unit, p.groups);
  set(k);
  plan.regs = 4;
  const int chunks = std::max(1, std::min<int>(gn_most_chunks(N, (size_t)p.pixels),
                                               (int)(256 / std::min<long long>(256, (long long)N * p.slices))));
  plan.threads = std::max(512, 1 << p.lg_vec);
  if ((long long)(plan.threads >> p.lg_vec) * plan.regs * chunks > p.pixels) plan.threads = std::max(256, 1 << p.lg_vec);
  const int stride = plan.threads >> p.lg_vec;
  p.chunk_pixels = (int)std::min<long long>(p.pixels, ((long long)p.pixels + (long long)chunks * stride - 1) /
                                                          ((long long)chunks * stride) * stride);
  p.chunks = (int)(((long long)p.pixels + p.chunk_pixels - 1) / p.chunk_pixels);
  return plan;
}

template <class E, class OUT, int R, int MODE, int NP>
static int gn_launch_one(const GroupNorm &p, const GnPlan &plan, hipStream_t st) {
  const int V = 1 << p.lg_vec;
  const int rows = V < 64 ? plan.threads / 64 : plan.threads >> p.lg_vec;
  const size_t lds = 16 * ((size_t)p.in_slice + 1) +
                     (MODE == kGnApply ? 0 : (size_t)rows * V * NP * sizeof(GnWide<NP>));
  const size_t sets = (size_t)(p.by_die ? (p.samples + 7) / 8 * 8 : p.samples) * p.slices * p.chunks;
  group_norm_kernel<E, OUT, R, MODE, NP><<<(unsigned)sets, plan.threads, lds, st>>>(p);
  return check_launch("group_norm");
}
template <class E, class OUT, int MODE, int NP>
static int gn_launch_regs(const GroupNorm &p, const GnPlan &plan, hipStream_t st) {
  if constexpr (MODE != kGnResident) return gn_launch_one<E, OUT, 4, MODE, NP>(p, plan, st);
  else {
    if (plan.regs == 1) return gn_launch_one<E, OUT, 1, MODE, NP>(p, plan, st);
    if (plan.regs == 2) return gn_launch_one<E, OUT, 2, MODE, NP>(p, plan, st);
    if (plan.regs == 4) return gn_launch_one<E, OUT, 4, MODE, NP>(p, plan, st);
    if constexpr (E::kSize == 2 && NP == 1)
      if (plan.regs == 16) return gn_launch_one<E, OUT, 16, MODE, NP>(p, plan, st);
    if constexpr (E::kSize == 2 || NP < 8) return gn_launch_one<E, OUT, 8, MODE, NP>(p, plan, st);
    return fail(MI355X_ERR_RUNTIME, "group_norm: %d pixels a thread", plan.regs);
  }
}
template <class E, class OUT, int NP>
static int gn_launch_as(const GroupNorm &p, const GnPlan &plan, hipStream_t st) {
  if (plan.resident) return gn_launch_regs<E, OUT, kGnResident, NP>(p, plan, st);
  // (the first launch does not depend on the result's type)
  if (int rc = gn_launch_regs<E, E, kGnStats, NP>(p, plan, st)) return rc;
  return gn_launch_regs<E, OUT, kGnApply, NP>(p, plan, st);
}
template <class E, class OUT>
static int gn_launch(GroupNorm p, size_t N, hipStream_t st) {
  const GnPlan plan = gn_plan(p, N, E::kSize, OUT::kSize == 0);
  // 2^32 threads are a launch's limit: more samples than that go in turns
  const size_t per_sample = plan.wide ? (size_t)p.groups * kGnWideThreads
                                      : (size_t)p.slices * p.chunks * plan.threads;
  if (per_sample > 0xf0000000ull / 8)
    return fail(MI355X_ERR_NOT_SUPPORTED, "group_norm: %d channels in %d groups", p.C, p.groups);
  const size_t most = 0xf0000000ull / per_sample / 8 * 8;
  const uint8_t *in = p.in;
  uint8_t *out = p.out;
  for (size_t done = 0; done < N; done += most) {
    p.samples = (int)std::min(most, N - done);
    p.in = in + done * p.pixels * p.in_row_bytes;
    p.out = out + done * p.pixels * p.out_row_bytes;
    int rc;
    if (plan.wide) {
      group_norm_wide_stats_kernel<E><<<(unsigned)((size_t)p.samples * p.groups), kGnWideThreads, 0, st>>>(p);
      if ((rc = check_launch("group_norm"))) return rc;
      const unsigned long long units = (unsigned long long)p.samples * p.pixels * p.channel_groups;
      const unsigned blocks = (unsigned)std::min<unsigned long long>(units / 16 + 1, 65536);
      group_norm_wide_apply_kernel<E, OUT><<<blocks, kGnWideThreads, 0, st>>>(p, units);
      rc = check_launch("group_norm");
    } else {
      p.by_die = plan.resident && p.slices > 1 && p.samples >= 8;
      const int parts = gn_parts(p.per);
      rc = parts == 1   ? gn_launch_as<E, OUT, 1>(p, plan, st)
           : parts == 2 ? gn_launch_as<E, OUT, 2>(p, plan, st)
                        : gn_launch_as<E, OUT, 8>(p, plan, st);
    }
    if (rc) return rc;
  }
  return MI355X_OK;
}

} // namespace mi355x

using namespace mi355x;

extern "C" {

int mi355x_group_norm_workspace_bytes(size_t N, size_t pixels, size_t C, size_t groups, size_t *bytes) {
  MI355X_REQUIRE(bytes, "group_norm_workspace_bytes: NULL");
  MI355X_REQUIRE(groups > 0 && C % groups == 0, "group_norm: %zu channels in %zu groups", C, groups);
  MI355X_REQUIRE(N <= 0x7fffffff && pixels <= 0x7fffffff && C <= 0x7fffffff,
                 "group_norm: %zu x %zu x %zu, up to 2^31 - 1 each are supported", N, pixels, C);
  if (!N || !pixels || !C) {
    *bytes = 0;
    return MI355X_OK;
  }
  size_t slots;
  MI355X_REQUIRE(!__builtin_mul_overflow(N * groups, gn_most_chunks(N, pixels) * sizeof(GroupStats), &slots) &&
                     slots <= PTRDIFF_MAX,
                 "group_norm: %zu x %zu groups", N, groups);
  *bytes = slots;
  return MI355X_OK;
}

int mi355x_group_norm(void *out, int out_type, size_t out_row_bytes, const void *in, int in_type,
                      size_t in_row_bytes, const float *gamma, const float *beta, size_t N,
                      size_t pixels, size_t C, size_t groups, float epsilon, int activation,
                      void *workspace, size_t workspace_bytes, void *stream) {
  size_t need;
  if (int rc = mi355x_group_norm_workspace_bytes(N, pixels, C, groups, &need)) return rc;
  MI355X_REQUIRE(float_type(in_type), "group_norm: input type %d is none of the float types", in_type);
  MI355X_REQUIRE(out_type == in_type || out_type == MI355X_MX4,
                 "group_norm: result type %d: the input's (%d) or microscaled rows are supported", out_type, in_type);
  if (int rc = check_rows("group_norm: input", in, in_type, in_row_bytes, N * pixels, C)) return rc;
  if (int rc = check_rows("group_norm: result", out, out_type, out_row_bytes, N * pixels, C)) return rc;
  MI355X_REQUIRE(epsilon >= 0, "group_norm: epsilon %g", (double)epsilon);
  MI355X_REQUIRE(activation == MI355X_ACT_NONE || activation == MI355X_ACT_RELU || activation == MI355X_ACT_SILU,
                 "group_norm: activation %d: none, Relu and SiLU are supported", activation);
  MI355X_REQUIRE((uintptr_t)gamma % 4 == 0 && (uintptr_t)beta % 4 == 0,
                 "group_norm: gamma and beta have to lie on multiples of 4");
  if (!N || !pixels || !C) return MI355X_OK;
  const size_t out_span = rows_span(out_type, out_row_bytes, N * pixels, C);
  const size_t in_span = rows_span(in_type, in_row_bytes, N * pixels, C);
  MI355X_REQUIRE((out == in && out_type == in_type && out_row_bytes == in_row_bytes) ||
                     !overlaps(out, out_span, in, in_span),
                 "group_norm: the result overlaps the input without being its place");
  MI355X_REQUIRE(!overlaps(out, out_span, gamma, 4 * C) && !overlaps(out, out_span, beta, 4 * C),
                 "group_norm: the result overlaps gamma or beta");
  MI355X_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0,
                 "group_norm: a workspace of %zu bytes on a multiple of 16 is needed "
                 "(mi355x_group_norm_workspace_bytes)", need);
  MI355X_REQUIRE(!overlaps(workspace, need, out, out_span) && !overlaps(workspace, need, in, in_span) &&
                     !overlaps(workspace, need, gamma, 4 * C) && !overlaps(workspace, need, beta, 4 * C),
                 "group_norm: the workspace overlaps a tensor");
  GroupNorm p{};
  p.out = static_cast<uint8_t *>(out);
  p.in = static_cast<const uint8_t *>(in);
  p.out_row_bytes = out_row_bytes;
  p.in_row_bytes = in_row_bytes;
  p.gamma = gamma;
  p.beta = beta;
  p.stats = static_cast<GroupStats *>(workspace);
  p.pixels = (int)pixels;
  p.C = (int)C;
  p.groups = (int)groups;
  p.per = (int)(C / groups);
  p.epsilon = epsilon;
  p.act = activation;
  p.channel_groups = (int)mx4_groups(C);
  p.mx4_bytes = mx4_row_bytes_of(C);
  hipStream_t st = as_stream(stream);
  const bool mx4 = out_type == MI355X_MX4;
  if (in_type == MI355X_F32) return mx4 ? gn_launch<F32, MX4>(p, N, st) : gn_launch<F32, F32>(p, N, st);
  if (in_type == MI355X_F16) return mx4 ? gn_launch<F16, MX4>(p, N, st) : gn_launch<F16, F16>(p, N, st);
  return mx4 ? gn_launch<BF16, MX4>(p, N, st) : gn_launch<BF16, BF16>(p, N, st);
}

} // extern "C"
