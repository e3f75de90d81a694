// Quantisation to microscaled 4-bit rows and back.
#include "mx4.h"

namespace mi355x {

// A lane holds eight neighbouring columns, sixteen lanes a group, and a workgroup of 256
// threads sixteen groups: up to sixteen of one row, or one each of sixteen rows. A block is
// four lanes: its largest magnitude takes two exchanges of neighbouring lanes, and 16-bit values
// are neither widened for that nor for the conversion, one instruction for two values.
//
// Bound by what they move: 8192 x 4096 of bf16 21 us to microscaled rows and 14 us back (85 MB
// each: 4.0 and 6.0 TB/s, where copying 1 GiB reaches 5.2 and 100 MiB in the last-level cache
// 8.3). Four shares a thread with their loads ahead of the first conversion take longer (25 and 15).
constexpr int kMxThreads = 256;

struct MxRows {
  long long rows;
  int cols, groups;
  int shift;            // a workgroup takes 2^shift groups of 16 >> shift rows
  unsigned chunks;      // workgroups' shares along a row
  unsigned tiles;       // shares in all
};
struct MxPlace {
  long long row;
  int group, l;
  bool inside;
};
__device__ __forceinline__ MxPlace mx_place(const MxRows &r, unsigned tile) {
  const int unit = threadIdx.x >> 4;
  MxPlace p;
  p.l = threadIdx.x & 15;
  p.row = (long long)(tile / r.chunks) * (16 >> r.shift) + (unit >> r.shift);
  p.group = (int)(tile % r.chunks << r.shift) + (unit & ((1 << r.shift) - 1));
  p.inside = p.row < r.rows && p.group < r.groups;
  return p;
}
// A launch has 2^23 workgroups at most, 2^31 threads (under 2^32 are the limit); they take turns then.
constexpr unsigned kMxMostBlocks = 1u << 23;
static int mx_rows(const char *what, size_t rows, size_t cols, MxRows *r, unsigned *blocks) {
  r->rows = (long long)rows;
  r->cols = (int)cols;
  r->groups = (int)mx4_groups(cols);
  r->shift = 0;
  while (r->shift < 4 && (1 << r->shift) < r->groups) r->shift++;
  r->chunks = (unsigned)((r->groups + (1 << r->shift) - 1) >> r->shift);
  const long long down = (r->rows + (16 >> r->shift) - 1) / (16 >> r->shift);
  const unsigned long long tiles = (unsigned long long)down * r->chunks;
  if (tiles > 0xffffffffull - kMxMostBlocks)
    return fail(MI355X_ERR_NOT_SUPPORTED, "%s: %zu x %zu values", what, rows, cols);
  r->tiles = (unsigned)tiles;
  *blocks = r->tiles < kMxMostBlocks ? r->tiles : kMxMostBlocks;
  return MI355X_OK;
}

template <class E>
__global__ __launch_bounds__(kMxThreads) void mx4_quantize_kernel(uint8_t *dst, size_t dst_row_bytes,
                                                                  const uint8_t *src,
                                                                  size_t src_row_bytes, MxRows r) {
  for (unsigned tile = blockIdx.x; tile < r.tiles; tile += gridDim.x) {
    const MxPlace p = mx_place(r, tile);
    if (!p.inside) continue;                       // whole groups: their sixteen lanes stay together
    const typename E::T *row = reinterpret_cast<const typename E::T *>(src + (size_t)p.row * src_row_bytes);
    const int c = p.group * kMxGroup + p.l * 8;
    typename E::Eight x;
    if (c <= r.cols - 8) x = load_eight<E>(row + c);
    else x = load_eight_end<E>(row + c, r.cols - c);
    mx4_store_group<E>(dst + (size_t)p.row * dst_row_bytes, r.groups, p.group, p.l, x);
  }
}

template <class E>
__global__ __launch_bounds__(kMxThreads) void mx4_dequantize_kernel(uint8_t *dst, size_t dst_row_bytes,
                                                                    const uint8_t *src,
                                                                    size_t src_row_bytes, MxRows r) {
  for (unsigned tile = blockIdx.x; tile < r.tiles; tile += gridDim.x) {
    const MxPlace p = mx_place(r, tile);
    const int c = p.group * kMxGroup + p.l * 8;
    if (!p.inside || c >= r.cols) continue;
    const uint8_t *row = src + (size_t)p.row * src_row_bytes;
    const uint32_t codes = *reinterpret_cast<const uint32_t *>(row + (c >> 1));
    const uint32_t byte = row[(size_t)r.groups * kMxGroupBytes + (c >> 5)];
    float x[8];
    mx4_values8(x, codes, byte);
    typename E::T *out = reinterpret_cast<typename E::T *>(dst + (size_t)p.row * dst_row_bytes) + c;
    if (c <= r.cols - 8) store8<E>(out, x);
    else store8_end<E>(out, x, r.cols - c);
  }
}

int mx4_quantize_launch(uint8_t *dst, size_t dst_row_bytes, const void *src, int src_type,
                        size_t src_row_bytes, size_t rows, size_t cols, hipStream_t st) {
  unsigned blocks;
  MxRows r;
  if (int rc = mx_rows("mx4_quantize", rows, cols, &r, &blocks)) return rc;
  const uint8_t *in = static_cast<const uint8_t *>(src);
  if (src_type == MI355X_F32)
    mx4_quantize_kernel<F32><<<blocks, kMxThreads, 0, st>>>(dst, dst_row_bytes, in, src_row_bytes, r);
  else if (src_type == MI355X_F16)
    mx4_quantize_kernel<F16><<<blocks, kMxThreads, 0, st>>>(dst, dst_row_bytes, in, src_row_bytes, r);
  else
    mx4_quantize_kernel<BF16><<<blocks, kMxThreads, 0, st>>>(dst, dst_row_bytes, in, src_row_bytes, r);
  return check_launch("mx4_quantize");
}

} // namespace mi355x

using namespace mi355x;

extern "C" {

size_t mi355x_mx4_row_bytes(size_t cols) { return mx4_row_bytes_of(cols); }

int mi355x_mx4_quantize(uint8_t *dst, size_t dst_row_bytes, const void *src, int src_type,
                        size_t src_row_bytes, size_t rows, size_t cols, void *stream) {
  MI355X_REQUIRE(float_type(src_type), "mx4_quantize: source type %d is none of the float types", src_type);
  if (int rc = check_rows("mx4_quantize: source", src, src_type, src_row_bytes, rows, cols)) return rc;
  if (int rc = check_rows("mx4_quantize: destination", dst, MI355X_MX4, dst_row_bytes, rows, cols)) return rc;
  if (!rows || !cols) return MI355X_OK;
  MI355X_REQUIRE(!overlaps(dst, rows_span(MI355X_MX4, dst_row_bytes, rows, cols), src,
                           rows_span(src_type, src_row_bytes, rows, cols)),
                 "mx4_quantize: the destination overlaps the source");
  return mx4_quantize_launch(dst, dst_row_bytes, src, src_type, src_row_bytes, rows, cols, as_stream(stream));
}

int mi355x_mx4_dequantize(void *dst, int dst_type, size_t dst_row_bytes, const uint8_t *src,
                          size_t src_row_bytes, size_t rows, size_t cols, void *stream) {
  MI355X_REQUIRE(float_type(dst_type), "mx4_dequantize: destination type %d is none of the float types", dst_type);
  if (int rc = check_rows("mx4_dequantize: source", src, MI355X_MX4, src_row_bytes, rows, cols)) return rc;
  if (int rc = check_rows("mx4_dequantize: destination", dst, dst_type, dst_row_bytes, rows, cols)) return rc;
  if (!rows || !cols) return MI355X_OK;
  MI355X_REQUIRE(!overlaps(dst, rows_span(dst_type, dst_row_bytes, rows, cols), src,
                           rows_span(MI355X_MX4, src_row_bytes, rows, cols)),
                 "mx4_dequantize: the destination overlaps the source");
  unsigned blocks;
  MxRows r;
  if (int rc = mx_rows("mx4_dequantize", rows, cols, &r, &blocks)) return rc;
  uint8_t *out = static_cast<uint8_t *>(dst);
  hipStream_t st = as_stream(stream);
  if (dst_type == MI355X_F32)
    mx4_dequantize_kernel<F32><<<blocks, kMxThreads, 0, st>>>(out, dst_row_bytes, src, src_row_bytes, r);
  else if (dst_type == MI355X_F16)
    mx4_dequantize_kernel<F16><<<blocks, kMxThreads, 0, st>>>(out, dst_row_bytes, src, src_row_bytes, r);
  else
    mx4_dequantize_kernel<BF16><<<blocks, kMxThreads, 0, st>>>(out, dst_row_bytes, src, src_row_bytes, r);
  return check_launch("mx4_dequantize");
}

} // extern "C"
