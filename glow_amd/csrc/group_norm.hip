// Group norm with an activation over channels-last tensors.
//
// Values x[n][p][c]; a group is C / groups neighbouring channels over all pixels of a
// sample: y = act((x - mean) / sqrt(variance + epsilon) * gamma[c] + beta[c]). Two launches:
// a workgroup for each group finds its mean and the mean square of what is left of it, in
// two passes; then sixteen lanes take 128 channels of a pixel, eight each, as the writers of
// microscaled rows do.
#include "mx4.h"

namespace mi355x {

struct GroupStats {
  float mean, scale;      // scale: 1 / sqrt(variance + epsilon)
};
struct GroupNorm {
  uint8_t *out;
  const uint8_t *in;
  size_t out_row_bytes, in_row_bytes;
  const float *gamma, *beta;
  GroupStats *stats;      // [N][groups]
  long long rows;         // N * pixels
  int pixels, C, groups, per;
  float epsilon;
  int act;
};

constexpr int kGnThreads = 256;

__device__ __forceinline__ float block_sum(float v, float *s_part) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0;
#pragma unroll
  for (int w = 0; w < kGnThreads / 64; w++) t += s_part[w];
  return t;
}

template <class E>
__global__ __launch_bounds__(kGnThreads) void group_norm_stats_kernel(GroupNorm p) {
  __shared__ float s_part[kGnThreads / 64];
  const int group = (int)(blockIdx.x % (unsigned)p.groups);
  const size_t sample = blockIdx.x / (unsigned)p.groups;
  const uint8_t *base = p.in + sample * p.pixels * p.in_row_bytes + (size_t)group * p.per * E::kSize;
  const long long n = (long long)p.pixels * p.per;
  auto value = [&](long long i) {
    return E::to(reinterpret_cast<const typename E::T *>(base + (size_t)(i / p.per) * p.in_row_bytes)[i % p.per]);
  };
  float sum = 0;
  for (long long i = threadIdx.x; i < n; i += kGnThreads) sum += value(i);
  const float mean = block_sum(sum, s_part) / (float)n;
  float square = 0;
  for (long long i = threadIdx.x; i < n; i += kGnThreads) {
    const float d = value(i) - mean;
    square = fmaf(d, d, square);
  }
  const float var = block_sum(square, s_part) / (float)n;
  if (threadIdx.x == 0) p.stats[blockIdx.x] = GroupStats{mean, 1.0f / sqrtf(var + p.epsilon)};
}

__device__ __forceinline__ float gn_act(float v, int act) {
  if (act == MI355X_ACT_RELU) return v < 0 ? 0.0f : v;     // (NaN stays)
  if (act == MI355X_ACT_SILU) return v / (1.0f + expf(-v));
  return v;
}

template <class E, class OUT>
__global__ __launch_bounds__(kGnThreads) void group_norm_apply_kernel(GroupNorm p, int channel_groups,
                                                                      unsigned long long units) {
  const int l = threadIdx.x & 15;
  for (unsigned long long u = blockIdx.x * 16ull + (threadIdx.x >> 4); u < units; u += gridDim.x * 16ull) {
    const size_t row = u / (unsigned)channel_groups;
    const int g = (int)(u % (unsigned)channel_groups), c = g * kMxGroup + l * 8;
    const typename E::T *in = reinterpret_cast<const typename E::T *>(p.in + row * p.in_row_bytes) + c;
    const int left = p.C - c;
    float x[8];
    if (left >= 8) load8<E>(x, in);
    else load8_end<E>(x, in, left);
    const GroupStats *stats = p.stats + row / (unsigned)p.pixels * p.groups;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (j < left) {
        const GroupStats s = stats[(c + j) / p.per];
        float y = (x[j] - s.mean) * s.scale;
        y = fmaf(y, p.gamma ? p.gamma[c + j] : 1.0f, p.beta ? p.beta[c + j] : 0.0f);
        x[j] = gn_act(y, p.act);
      }
    }
    uint8_t *out = p.out + row * p.out_row_bytes;
    if constexpr (OUT::kSize == 0) {
      mx4_store_group(out, channel_groups, g, l, x);
    } else if (left > 0) {
      typename OUT::T *o = reinterpret_cast<typename OUT::T *>(out) + c;
      if (left >= 8) store8<OUT>(o, x);
      else store8_end<OUT>(o, x, left);
    }
  }
}

template <class E>
static int group_norm_launch(const GroupNorm &p, size_t N, bool mx4, hipStream_t st) {
  group_norm_stats_kernel<E><<<(unsigned)(N * p.groups), kGnThreads, 0, st>>>(p);
  if (int rc = check_launch("group_norm")) return rc;
  const int channel_groups = (int)mx4_groups((size_t)p.C);
  const unsigned long long units = (unsigned long long)p.rows * channel_groups;
  const unsigned blocks = (unsigned)(units / 16 + 1 < 65536 ? units / 16 + 1 : 65536);
  if (mx4) group_norm_apply_kernel<E, MX4><<<blocks, kGnThreads, 0, st>>>(p, channel_groups, units);
  else group_norm_apply_kernel<E, E><<<blocks, kGnThreads, 0, st>>>(p, channel_groups, units);
  return check_launch("group_norm");
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
  if (N * groups > (1u << 23))
    return fail(MI355X_ERR_NOT_SUPPORTED, "group_norm: %zu samples of %zu groups, up to 2^23 in all are supported", N,
                groups);
  *bytes = N * groups * sizeof(GroupStats);
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
  GroupNorm p;
  p.out = static_cast<uint8_t *>(out);
  p.in = static_cast<const uint8_t *>(in);
  p.out_row_bytes = out_row_bytes;
  p.in_row_bytes = in_row_bytes;
  p.gamma = gamma;
  p.beta = beta;
  p.stats = static_cast<GroupStats *>(workspace);
  p.rows = (long long)(N * pixels);
  p.pixels = (int)pixels;
  p.C = (int)C;
  p.groups = (int)groups;
  p.per = (int)(C / groups);
  p.epsilon = epsilon;
  p.act = activation;
  hipStream_t st = as_stream(stream);
  const bool mx4 = out_type == MI355X_MX4;
  if (in_type == MI355X_F32) return group_norm_launch<F32>(p, N, mx4, st);
  if (in_type == MI355X_F16) return group_norm_launch<F16>(p, N, mx4, st);
  return group_norm_launch<BF16>(p, N, mx4, st);
}

} // extern "C"
