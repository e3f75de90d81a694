// A cache of keys and values in microscaled rows, and the batch of rows that belong to its
// sequences: what its writer and the attention over it share.
#ifndef GLOW_MI355X_MX4_CACHE_H
#define GLOW_MI355X_MX4_CACHE_H

#include "mx4.h"

#include <algorithm>

namespace mi355x {

constexpr int kCacheTile = 16;        // tokens that lie on one page in any case

// A cache as kernels take it. Tokens are counted in 32 bits, rows of the cache in 64.
struct MxCache {
  uint8_t *keys, *values;
  size_t row_bytes;
  const int32_t *pages;
  unsigned n_pages, page_tiles, page_magic, per_sequence;
  int scales_at;                      // bytes from a row's codes to its scales
  int capacity;                       // tokens of a sequence
  const int32_t *starts, *lengths;
  int sequences, rows;
};

// a / d for a < 2^31, with magic = the lower of 2^32 / d and 2^32 - 1: the product falls short by one
// at most.
__device__ __forceinline__ unsigned divide(unsigned a, unsigned d, unsigned magic) {
  const unsigned e = __umulhi(a, magic);
  return e + (a - e * d >= d);
}
// Which sixteen rows of the cache a tile of sixteen tokens of a sequence has; -1: on no page.
__device__ __forceinline__ int cache_tile(const MxCache &c, int sequence, unsigned tile) {
  const unsigned k = divide(tile, c.page_tiles, c.page_magic);
  if (k >= c.per_sequence) return -1;
  const size_t slot = (size_t)sequence * c.per_sequence + k;
  const size_t page = c.pages ? (size_t)(unsigned)c.pages[slot] : slot;   // (negative ones: past the last)
  if (page >= c.n_pages) return -1;
  return (int)((unsigned)page * c.page_tiles + (tile - k * c.page_tiles));
}

__device__ __forceinline__ int batch_start(const MxCache &c, int s) { return min(max(c.starts[s], 0), c.rows); }

// The last sequence s whose `first` (which does not decrease with s) is at most `at`; TEAM
// neighbouring lanes of a wave search together, TEAM places a round.
template <int TEAM, class F> __device__ __forceinline__ int find_sequence(int sequences, long long at, F &&first) {
  const int lane = threadIdx.x & (TEAM - 1), shift = (threadIdx.x & 63) & ~(TEAM - 1);
  int low = 0, n = sequences;                   // the answer is in [low, low + n)
  while (n > 1) {
    const int step = (n + TEAM - 1) / TEAM, s = lane * step;
    const bool fits = s < n && first(low + s) <= at;
    unsigned long long votes = __ballot(fits) >> shift;
    if (TEAM < 64) votes &= (1ull << (TEAM & 63)) - 1;
    const int last = votes ? 63 - __clzll((long long)votes) : 0;
    low += last * step;
    n = min(step, n - last * step);
  }
  return low;
}

// Checks a cache and a batch, and fills `c` in.
inline int check_cache(const char *what, const mi355x_mx4_cache *cache, MxCache *c) {
  MI355X_REQUIRE(cache, "%s: no cache", what);
  MI355X_REQUIRE(cache->page_tokens > 0 && cache->page_tokens % kCacheTile == 0,
                 "%s: pages of %u tokens, a multiple of %d is needed", what, cache->page_tokens, kCacheTile);
  MI355X_REQUIRE(cache->head_dim == 64 || cache->head_dim == 128 || cache->head_dim == 256,
                 "%s: heads of %u columns: 64, 128 and 256 are supported", what, cache->head_dim);
  MI355X_REQUIRE(cache->kv_heads > 0 && cache->kv_heads <= 0x7fffffff / cache->head_dim, "%s: %u heads of keys", what,
                 cache->kv_heads);
  MI355X_REQUIRE((uint64_t)cache->pages_per_sequence * cache->page_tokens <= 0x7fffffff,
                 "%s: %u pages of %u tokens, up to 2^31 - 1 tokens of a sequence are supported", what,
                 cache->pages_per_sequence, cache->page_tokens);
  MI355X_REQUIRE(cache->row_bytes <= (1u << 26), "%s: rows %llu bytes apart, up to 2^26 are supported", what,
                 (unsigned long long)cache->row_bytes);
  const size_t cols = (size_t)cache->kv_heads * cache->head_dim, least = mx4_row_bytes_of(cols);
  MI355X_REQUIRE(cache->row_bytes >= least, "%s: rows %llu bytes apart, %zu columns take %zu", what,
                 (unsigned long long)cache->row_bytes, cols, least);
  MI355X_REQUIRE(cache->row_bytes % 16 == 0 && (uintptr_t)cache->keys % 16 == 0 && (uintptr_t)cache->values % 16 == 0,
                 "%s: the cache's addresses and the distance between rows have to be multiples of 16", what);
  MI355X_REQUIRE((uintptr_t)cache->pages % 4 == 0, "%s: the pages have to lie on a multiple of 4", what);
  MI355X_REQUIRE(cache->n_pages == 0 || (cache->keys && cache->values), "%s: NULL", what);
  if ((uint64_t)cache->n_pages * (cache->page_tokens / kCacheTile) > 0x7fffffff)
    return fail(MI355X_ERR_NOT_SUPPORTED, "%s: %u pages of %u tokens, up to 2^35 - 16 rows are supported", what,
                cache->n_pages, cache->page_tokens);
  c->keys = cache->keys;
  c->values = cache->values;
  c->row_bytes = cache->row_bytes;
  c->pages = cache->pages;
  c->n_pages = cache->n_pages;
  c->page_tiles = cache->page_tokens / kCacheTile;
  c->page_magic = c->page_tiles == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / c->page_tiles);
  c->per_sequence = cache->pages_per_sequence;
  c->scales_at = (int)(mx4_groups(cols) * kMxGroupBytes);
  c->capacity = (int)(cache->pages_per_sequence * cache->page_tokens);
  return MI355X_OK;
}
// Bytes of the keys, or of the values.
inline size_t cache_span(const mi355x_mx4_cache *cache) {
  return (size_t)cache->n_pages * cache->page_tokens * cache->row_bytes;
}
inline int check_batch(const char *what, const int32_t *starts, const int32_t *lengths, size_t sequences, size_t rows,
                       MxCache *c) {
  MI355X_REQUIRE(sequences <= 0x3fffffff && rows <= 0x3fffffff, "%s: %zu sequences, %zu rows: up to 2^30 - 1 are supported",
                 what, sequences, rows);
  MI355X_REQUIRE((uintptr_t)starts % 4 == 0 && (uintptr_t)lengths % 4 == 0,
                 "%s: starts and lengths have to lie on multiples of 4", what);
  MI355X_REQUIRE(!sequences || !rows || (starts && lengths), "%s: starts or lengths are NULL", what);
  c->starts = starts;
  c->lengths = lengths;
  c->sequences = (int)sequences;
  c->rows = (int)rows;
  return MI355X_OK;
}

} // namespace mi355x

#endif
