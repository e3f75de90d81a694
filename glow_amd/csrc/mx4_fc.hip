// The product of microscaled 4-bit rows: out[m][n] = act(bias[n] + sum_k in[m][k] w[n][k]).
//
// The matrix cores' scaled instruction takes 64 columns of 32 rows of both operands: a lane
// feeds one block (16 bytes of codes of row lane % 32, block lane / 32) and its scale byte,
// and products are summed in 32 bits. The weights are the first operand, so that a lane's
// results belong to one row of the output and lie in fours of neighbouring columns: what a
// microscaled result's blocks and wide stores want.
#include "mx4_tiles.h"

namespace mi355x {

template <class OUT>
static int fc_launch(const MxFc &p, hipStream_t st) {
  const long long n = p.N, m = p.M;
  if (((n + 255) / 256) * ((m + 255) / 256) >= 192)
    return mx4_fc_tile_launch<OUT, 256, 256, 128, 64, 4, 1>(p, st);
  if (((n + 127) / 128) * ((m + 127) / 128) >= 192)
    return mx4_fc_tile_launch<OUT, 128, 128, 64, 64, 4, 2>(p, st);
  return mx4_fc_tile_launch<OUT, 64, 64, 32, 32, 4, 4>(p, st);
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
