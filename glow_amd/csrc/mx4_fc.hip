// The product of microscaled 4-bit rows: out[m][n] = act(bias[n] + sum_k in[m][k] w[n][k]).
//
// The matrix cores' scaled instruction takes 128 columns of 16 rows of both operands: a lane
// feeds one block (16 bytes of codes of row lane % 16, block lane / 16) and its scale byte,
// and products are summed in 32 bits. The weights are the first operand, so that a lane's
// results belong to one row of the output and lie in fours of neighbouring columns: what a
// microscaled result's blocks and wide stores want.
#include "mx4_fc.h"

namespace mi355x {

// Whether a float input is quantised by the kernel itself: every workgroup does so for its rows,
// which a launch in front saves where they are many bytes, or shared by many workgroups. us, in the
// kernel / in front: 128 x 1024 x 1024 of fp16 4.9 / 5.6 (64 KB of rows), 16 x 4096 x 4096 8.6 / 8.3
// (128 KB), 64 x 4096 x 4096 15.3 / 12.3 (256 KB), 61 x 415 x 509 of fp32 3.5 / 5.0; 64x64 tiles
// without a ring: 4096 x 13 x 512 of fp32 4.7 / 5.8 (3 KB, 8 tiles to a row), 25088 x 512 x 128 of
// fp16 11.1 / 13.8 (64 KB, 2), 2000 x 400 x 500 of fp32 8.2 / 6.9 (100 KB, 8), 8192 x 256 x 1024 of
// fp16 10.8 / 10.0 (32 KB, 16). Rows that do not all start on a word (`words`) take three times as
// long to load: 186 x 895 x 792 of fp16 9.2 / 6.4 (57 KB; 186 x 894 x 792 5.6 / 6.4), 40 x 895 x 400 5.5 /
// 5.8 (29 KB); up to four rows, which are loaded once, 1 x 4095 x 4096 4.9 / 6.7.
static bool fc_quantizes(FcTile tile, long long M, long long K, long long N, size_t size, bool words) {
  if (tile == kFcShort64) return 64 * K * (long long)size <= 64 * 1024 && N <= 8 * 64;
  const long long most = words || M <= kSharedRows ? 96 * 1024 : 32 * 1024;
  return tile <= kFc32 && std::min(M, tile == kFc16 ? 16LL : 32LL) * K * (long long)size <= most;
}

template <class IN, class OUT> static int fc_small(const MxFc &p, int K, FcTile tile, hipStream_t st) {
  if constexpr (OUT::kSize == 0) {
    return tile == kFc16 ? mx4_fc_small_launch<IN, OUT, 1, 2>(p, K, st) : mx4_fc_small_launch<IN, OUT, 2, 2>(p, K, st);
  } else {
    return tile == kFc16      ? mx4_fc_small_launch<IN, OUT, 1, 1>(p, K, st)
           : tile == kFc32x16 ? mx4_fc_small_launch<IN, OUT, 2, 1>(p, K, st)
                              : mx4_fc_small_launch<IN, OUT, 2, 2>(p, K, st);
  }
}
template <class OUT> static int fc_launch(const MxFc &p, int K, int in_type, FcTile tile, hipStream_t st) {
  if (tile <= kFc32)
    return in_type == MI355X_F32   ? fc_small<F32, OUT>(p, K, tile, st)
           : in_type == MI355X_F16 ? fc_small<F16, OUT>(p, K, tile, st)
           : in_type == MI355X_BF16 ? fc_small<BF16, OUT>(p, K, tile, st)
                                    : fc_small<MX4, OUT>(p, K, tile, st);
  if (tile == kFcShort64)
    return in_type == MI355X_F32    ? mx4_fc_short_launch<F32, OUT, 64, 64, 32, 32, 4>(p, K, st)
           : in_type == MI355X_F16  ? mx4_fc_short_launch<F16, OUT, 64, 64, 32, 32, 4>(p, K, st)
           : in_type == MI355X_BF16 ? mx4_fc_short_launch<BF16, OUT, 64, 64, 32, 32, 4>(p, K, st)
                                    : mx4_fc_short_launch<MX4, OUT, 64, 64, 32, 32, 4>(p, K, st);
  if (tile == kFcShort128) return mx4_fc_short_launch<MX4, OUT, 128, 128, 64, 64, 2>(p, K, st);
  return tile == kFc256   ? mx4_fc_tile_launch<OUT, 256, 256, 128, 64, 4, 1>(p, st)
         : tile == kFc128 ? mx4_fc_tile_launch<OUT, 128, 128, 64, 64, 4, 2>(p, st)
                          : mx4_fc_tile_launch<OUT, 64, 64, 32, 32, 4, 4>(p, st);
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
  *bytes = 0;
  if (in_type == MI355X_MX4 || !M || !N) return MI355X_OK;
  // (whatever the result's type, and wherever the rows lie)
  for (bool mx4_out : {false, true})
    if (!fc_quantizes(fc_tile((long long)M, (long long)K, (long long)N, mx4_out), (long long)M, (long long)K, (long long)N,
                      float_size(in_type), in_type == MI355X_F32))
      *bytes = M * mx4_row_bytes_of(K);
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
  }
  const FcTile tile = fc_tile((long long)M, (long long)K, (long long)N, out_type == MI355X_MX4);
  const bool words = ((uintptr_t)in | in_row_bytes) % 4 == 0;
  if (in_type != MI355X_MX4 &&
      !fc_quantizes(tile, (long long)M, (long long)K, (long long)N, float_size(in_type), words)) {
    p.in = static_cast<const uint8_t *>(workspace);
    p.in_row_bytes = mx4_row_bytes_of(K);
    if (K)
      if (int rc = mx4_quantize_launch(static_cast<uint8_t *>(workspace), p.in_row_bytes, in, in_type, in_row_bytes, M,
                                       K, st))
        return rc;
    in_type = MI355X_MX4;
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
  const int k = (int)K;
  if (out_type == MI355X_F32) return fc_launch<F32>(p, k, in_type, tile, st);
  if (out_type == MI355X_F16) return fc_launch<F16>(p, k, in_type, tile, st);
  if (out_type == MI355X_BF16) return fc_launch<BF16>(p, k, in_type, tile, st);
  return fc_launch<MX4>(p, k, in_type, tile, st);
}

} // extern "C"
