// The product of microscaled 4-bit rows: out[m][n] = act(bias[n] + sum_k in[m][k] w[n][k]).
//
// The matrix cores' scaled instruction takes 64 columns of 32 rows of both operands: a lane
// feeds one block (16 bytes of codes of row lane % 32, block lane / 32) and its scale byte,
// and products are summed in 32 bits. The weights are the first operand, so that a lane's
// results belong to one row of the output and lie in fours of neighbouring columns: what a
// microscaled result's blocks and wide stores want.
#include "mx4.h"

namespace mi355x {

typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef int mx_v4i __attribute__((ext_vector_type(4)));
typedef float mx_v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ mx_v8i fp4_operand(mx_v4i v) {
  return mx_v8i{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
}

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

// One wave, one 32x32 tile, fragments straight from memory.
template <class OUT>
__global__ __launch_bounds__(64) void mx4_fc_kernel(MxFc p, int tiles_n) {
  const int lane = threadIdx.x, row = lane & 31, half = lane >> 5;
  const int n0 = (int)(blockIdx.x % (unsigned)tiles_n) * 32, m0 = (int)(blockIdx.x / (unsigned)tiles_n) * 32;
  const int m = m0 + row;
  // rows past the end re-read the last one; what they give is not stored
  const uint8_t *a = p.weights + (size_t)min(n0 + row, p.N - 1) * p.weights_row_bytes;
  const uint8_t *b = p.in + (size_t)min(m, p.M - 1) * p.in_row_bytes;
  const uint32_t *as = reinterpret_cast<const uint32_t *>(a + (size_t)p.groups * kMxGroupBytes);
  const uint32_t *bs = reinterpret_cast<const uint32_t *>(b + (size_t)p.groups * kMxGroupBytes);
  mx_v16f acc;
#pragma unroll
  for (int i = 0; i < 16; i++) acc[i] = 0.0f;
  for (int g = 0; g < p.groups; g++) {
    const mx_v4i *ag = reinterpret_cast<const mx_v4i *>(a + (size_t)g * kMxGroupBytes) + half;
    const mx_v4i *bg = reinterpret_cast<const mx_v4i *>(b + (size_t)g * kMxGroupBytes) + half;
    const uint32_t ae = as[g] >> (8 * half), be = bs[g] >> (8 * half);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(ag[0]), fp4_operand(bg[0]), acc, 4, 4, 0,
                                                          (int)ae, 0, (int)be);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(ag[2]), fp4_operand(bg[2]), acc, 4, 4, 2,
                                                          (int)ae, 2, (int)be);
  }
  // register 4 q + j of a lane: column 8 q + 4 half + j
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int n = n0 + 8 * (i >> 2) + 4 * half + (i & 3);
    acc[i] = n < p.N ? activate(acc[i] + (p.bias ? p.bias[n] : 0.0f), p.act) : 0.0f;
  }
  uint8_t *out = p.out + (size_t)m * p.out_row_bytes;
  if constexpr (OUT::kSize == 0) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) most = max(most, magnitude_bits(acc[i]));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32));
    const uint32_t byte = mx4_scale_byte(most);
    if (m < p.M) {
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const float x[8] = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3], 0, 0, 0, 0};
        *reinterpret_cast<uint16_t *>(out + n0 / 2 + 4 * q + 2 * half) = (uint16_t)mx4_codes8(x, byte);
      }
      if (half == 0) {
        uint8_t *scales = out + (size_t)p.out_groups * kMxGroupBytes;
        scales[n0 / 32] = (uint8_t)byte;
        // the zeros behind the last group's scales
        if (n0 / 32 == 4 * p.out_groups - 1)
          for (int w = 0; w < ((-p.out_groups) & 3); w++)
            reinterpret_cast<uint32_t *>(scales)[p.out_groups + w] = 0;
      }
    }
  } else if (m < p.M) {
    typename OUT::T *o = reinterpret_cast<typename OUT::T *>(out);
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int n = n0 + 8 * (i >> 2) + 4 * half + (i & 3);
      if (n < p.N) o[n] = OUT::from(acc[i]);
    }
  }
}

template <class OUT>
static int fc_launch(const MxFc &p, hipStream_t st) {
  // a microscaled result has whole groups of columns, the ones past N zeros
  const long long tiles_n = OUT::kSize ? (p.N + 31) / 32 : 4LL * p.out_groups;
  const long long tiles = tiles_n * ((p.M + 31) / 32);
  if (tiles > (1 << 26) - 1)
    return fail(MI355X_ERR_NOT_SUPPORTED, "mx4_fc: %d x %d results", p.M, p.N);
  mx4_fc_kernel<OUT><<<(unsigned)tiles, 64, 0, st>>>(p, (int)tiles_n);
  return check_launch("mx4_fc");
}

} // namespace mi355x

using namespace mi355x;

extern "C" {

int mi355x_mx4_fc_workspace_bytes(size_t M, size_t K, size_t N, int in_type, size_t *bytes) {
  MI355X_REQUIRE(bytes, "mx4_fc_workspace_bytes: NULL");
  MI355X_REQUIRE(in_type == MI355X_MX4 || float_type(in_type), "mx4_fc_workspace_bytes: unknown element type %d",
                 in_type);
  MI355X_REQUIRE(M <= 0x7fffffff && K <= 0x7fffffff && N <= 0x7fffffff,
                 "mx4_fc_workspace_bytes: %zu x %zu x %zu, up to 2^31 - 1 each are supported", M, K, N);
  *bytes = in_type == MI355X_MX4 ? 0 : M * mx4_row_bytes_of(K);
  return MI355X_OK;
}

int mi355x_mx4_fc(void *out, int out_type, size_t out_row_bytes, const void *in, int in_type,
                  size_t in_row_bytes, const uint8_t *weights, size_t weights_row_bytes,
                  const float *bias, size_t M, size_t K, size_t N, int activation, void *workspace,
                  size_t workspace_bytes, void *stream) {
  if (int rc = check_rows("mx4_fc: result", out, out_type, out_row_bytes, M, N)) return rc;
  if (int rc = check_rows("mx4_fc: input", in, in_type, in_row_bytes, M, K)) return rc;
  if (int rc = check_rows("mx4_fc: weights", weights, MI355X_MX4, weights_row_bytes, N, K)) return rc;
  MI355X_REQUIRE(activation == MI355X_ACT_NONE || activation == MI355X_ACT_RELU || activation == MI355X_ACT_SILU,
                 "mx4_fc: activation %d: none, Relu and SiLU are supported", activation);
  MI355X_REQUIRE((uintptr_t)bias % 4 == 0, "mx4_fc: the bias has to lie on a multiple of 4");
  if (!M || !N) return MI355X_OK;
  const size_t out_span = rows_span(out_type, out_row_bytes, M, N), in_span = rows_span(in_type, in_row_bytes, M, K);
  const size_t w_span = rows_span(MI355X_MX4, weights_row_bytes, N, K);
  MI355X_REQUIRE(!overlaps(out, out_span, in, in_span) && !overlaps(out, out_span, weights, w_span) &&
                     !overlaps(out, out_span, bias, 4 * N),
                 "mx4_fc: the result overlaps what it is made from");
  size_t need;
  if (int rc = mi355x_mx4_fc_workspace_bytes(M, K, N, in_type, &need)) return rc;
  hipStream_t st = as_stream(stream);
  MxFc p;
  p.in = static_cast<const uint8_t *>(in);
  p.in_row_bytes = in_row_bytes;
  if (need) {
    MI355X_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0,
                   "mx4_fc: a workspace of %zu bytes on a multiple of 16 is needed (mi355x_mx4_fc_workspace_bytes)",
                   need);
    MI355X_REQUIRE(!overlaps(workspace, need, out, out_span) && !overlaps(workspace, need, in, in_span) &&
                       !overlaps(workspace, need, weights, w_span) && !overlaps(workspace, need, bias, 4 * N),
                   "mx4_fc: the workspace overlaps a tensor");
    p.in = static_cast<const uint8_t *>(workspace);
    p.in_row_bytes = mx4_row_bytes_of(K);
    if (int rc = mx4_quantize_launch(static_cast<uint8_t *>(workspace), p.in_row_bytes, in, in_type, in_row_bytes, M,
                                     K, st))
      return rc;
  }
  p.out = static_cast<uint8_t *>(out);
  p.out_row_bytes = out_row_bytes;
  p.weights = weights;
  p.weights_row_bytes = weights_row_bytes;
  p.bias = bias;
  p.M = (int)M;
  p.N = (int)N;
  p.groups = (int)mx4_groups(K);
  p.out_groups = (int)mx4_groups(N);
  p.act = activation;
  if (out_type == MI355X_F32) return fc_launch<F32>(p, st);
  if (out_type == MI355X_F16) return fc_launch<F16>(p, st);
  if (out_type == MI355X_BF16) return fc_launch<BF16>(p, st);
  return fc_launch<MX4>(p, st);
}

} // extern "C"
