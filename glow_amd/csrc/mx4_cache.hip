// New tokens' keys and values into a cache of microscaled rows.
#include "mx4_cache.h"

namespace mi355x {

// As the quantisation of rows: sixteen lanes a group of 128 columns, eight columns a lane. A team of
// sixteen finds the sequence of its row first, sixteen places a round, and then the row's page. Bound by these loads, one behind
// the other: 64 tokens of 1024 columns 3.9 us, 12 000 tokens of fp16 22 us (63 MB, 2.9 TB/s).
constexpr int kCacheThreads = 256;

template <class E>
__global__ __launch_bounds__(kCacheThreads) void mx4_cache_write_kernel(MxCache c, const uint8_t *keys, const uint8_t *values,
                                                                        size_t keys_row_bytes, size_t values_row_bytes,
                                                                        int cols, int groups, unsigned long long units) {
  const int l = threadIdx.x & 15;
  for (unsigned long long u = blockIdx.x * 16ull + (threadIdx.x >> 4); u < units; u += gridDim.x * 16ull) {
    const int g = (int)(u % (unsigned)groups);
    const unsigned long long rest = u / (unsigned)groups;
    const bool is_value = rest & 1;
    const int r = (int)(rest >> 1);
    const int s = find_sequence<16>(c.sequences, r, [&](int i) { return batch_start(c, i); });
    const int begin = batch_start(c, s), end = batch_start(c, s + 1);
    if (r < begin || r >= end) continue;          // (whole teams)
    const int length = min(max(c.lengths[s], 0), c.capacity);
    const int t = length - (end - begin) + (r - begin);
    if (t < 0 || t >= length) continue;
    const int tile = cache_tile(c, s, (unsigned)t / kCacheTile);
    if (tile < 0) continue;
    uint8_t *dst = (is_value ? c.values : c.keys) + ((size_t)tile * kCacheTile + t % kCacheTile) * c.row_bytes;
    const uint8_t *src = is_value ? values + (size_t)r * values_row_bytes : keys + (size_t)r * keys_row_bytes;
    if constexpr (E::kSize == 0) {
      reinterpret_cast<uint32_t *>(dst + (size_t)g * kMxGroupBytes)[l] =
          reinterpret_cast<const uint32_t *>(src + (size_t)g * kMxGroupBytes)[l];
      uint32_t *scales = reinterpret_cast<uint32_t *>(dst + (size_t)groups * kMxGroupBytes);
      if (l == 0) scales[g] = reinterpret_cast<const uint32_t *>(src + (size_t)groups * kMxGroupBytes)[g];
      else if (g == groups - 1 && l < 4 && l <= ((-groups) & 3)) scales[g + l] = 0;
    } else {
      const typename E::T *in = reinterpret_cast<const typename E::T *>(src);
      const int at = g * kMxGroup + l * 8;
      typename E::Eight x;
      if (at <= cols - 8) x = load_eight<E>(in + at);
      else x = load_eight_end<E>(in + at, cols - at);
      mx4_store_group<E>(dst, groups, g, l, x);
    }
  }
}

} // namespace mi355x

using namespace mi355x;

extern "C" {

int mi355x_mx4_cache_write(const mi355x_mx4_cache *cache, const void *keys, const void *values, int type,
                           size_t keys_row_bytes, size_t values_row_bytes, const int32_t *starts, const int32_t *lengths,
                           size_t sequences, size_t rows, void *stream) {
  MxCache c;
  if (int rc = check_cache("mx4_cache_write", cache, &c)) return rc;
  if (int rc = check_batch("mx4_cache_write", starts, lengths, sequences, rows, &c)) return rc;
  const size_t cols = (size_t)cache->kv_heads * cache->head_dim;
  if (int rc = check_rows("mx4_cache_write: keys", keys, type, keys_row_bytes, rows, cols)) return rc;
  if (int rc = check_rows("mx4_cache_write: values", values, type, values_row_bytes, rows, cols)) return rc;
  if (!sequences || !rows || !c.n_pages || !c.per_sequence) return MI355X_OK;
  const size_t span = cache_span(cache);
  const size_t table = cache->pages ? sequences * cache->pages_per_sequence * 4 : 0;
  MI355X_REQUIRE(!overlaps(c.keys, span, c.values, span), "mx4_cache_write: the cache's keys overlap its values");
  for (const uint8_t *to : {c.keys, c.values})
    MI355X_REQUIRE(!overlaps(to, span, keys, rows_span(type, keys_row_bytes, rows, cols)) &&
                       !overlaps(to, span, values, rows_span(type, values_row_bytes, rows, cols)) &&
                       !overlaps(to, span, starts, 4 * (sequences + 1)) && !overlaps(to, span, lengths, 4 * sequences) &&
                       !overlaps(to, span, cache->pages, table),
                   "mx4_cache_write: the cache overlaps what is written into it");
  const int groups = (int)mx4_groups(cols);
  const unsigned long long units = 2ull * rows * groups;
  const unsigned blocks = (unsigned)std::min<unsigned long long>((units + 15) / 16, 1u << 20);
  const uint8_t *k = static_cast<const uint8_t *>(keys), *v = static_cast<const uint8_t *>(values);
  hipStream_t st = as_stream(stream);
  auto launch = [&](auto kernel) {
    kernel<<<blocks, kCacheThreads, 0, st>>>(c, k, v, keys_row_bytes, values_row_bytes, (int)cols, groups, units);
  };
  if (type == MI355X_F32) launch(mx4_cache_write_kernel<F32>);
  else if (type == MI355X_F16) launch(mx4_cache_write_kernel<F16>);
  else if (type == MI355X_BF16) launch(mx4_cache_write_kernel<BF16>);
  else launch(mx4_cache_write_kernel<MX4>);
  return check_launch("mx4_cache_write");
}

} // extern "C"
