// Which kernel a product of microscaled rows runs.
#ifndef GLOW_MI355X_MX4_FC_H
#define GLOW_MI355X_MX4_FC_H

#include "mx4_short.h"
#include "mx4_small.h"
#include "mx4_tiles.h"

namespace mi355x {

// Which kernel a product runs: small tiles of 16 or 32 rows and columns with K over the waves
// (mx4_small.h) while they give each CU one workgroup or less, the smallest that do; else tiles
// of 64 to 256 through LDS. us, 16x16 / 32x16 / 32x32 / 64x64 tiles, fp16 results: 1 x 4096 x
// 4096 4.4 / - / - / 11.4, 500 x 512 x 512 3.8 / 3.3 / 3.4 / 4.2, 256 x 2048 x 1024 7.9 / 6.6 /
// 5.6 / 7.4, 64 x 4096 x 8192 34 / 24 / 18 / 11.5 (rows x K x columns). Up to four rows 16x16
// holds its own over any number of columns (1 x 4096 x 16384 10.9 / 11.9): the input is next
// to nothing then.
// Up to 512 columns the larger tiles need no ring (mx4_short.h): 4096 x 512 x 256 4.7 / 3.8, 25088 x
// 512 x 128 7.6 / 5.4, 8192 x 512 x 4096 29.5 (256x256 tiles) / 24.7 (128x128 without a ring; 64x64
// 27.0).
enum FcTile { kFc16, kFc32x16, kFc32, kFcShort64, kFcShort128, kFc64, kFc128, kFc256 };
static FcTile fc_tile(long long M, long long K, long long N, bool mx4_out) {
  const long long most = 288;
  const long long m16 = (M + 15) / 16, m32 = (M + 31) / 32, n16 = (N + 15) / 16, n32 = (N + 31) / 32;
  if (mx4_out) {                   // a microscaled result's columns go by blocks of 32
    if (m16 * n32 <= most || M <= 4) return kFc16;
  } else {
    if (m16 * n16 <= most || M <= 4) return kFc16;
    if (m32 * n16 <= most) return kFc32x16;
  }
  if (m32 * n32 <= most) return kFc32;
  if (K <= kShortGroups * kMxGroup)
    return N > 64 && ((N + 127) / 128) * ((M + 127) / 128) >= 512 ? kFcShort128 : kFcShort64;
  // Tiles through the ring: what a CU takes for its share of them, us behind a launch's own three, a
  // tile's ends and its steps of K. Estimated / measured: 2048 x 2048 x 2048 in tiles of 64 / 128 / 256
  // 15.5 / 8.9 / 23.2, 14 / 9 / 19; 1024 x 4096 x 4096 27 / 15.3 / 38, 24 / 14.7 / 27; 4096 x 8192 x
  // 4096 - / 112 / 69, 169 / 98 / 65.
  const double steps = (double)((K + kMxGroup - 1) / kMxGroup);
  auto share = [&](long long tile) {
    return (double)((((N + tile - 1) / tile) * ((M + tile - 1) / tile) + 255) / 256);
  };
  const double us64 = share(64) * (1.0 + 0.18 * steps), us128 = share(128) * (2.5 + 0.40 * steps),
               us256 = share(256) * (8.0 + 0.95 * steps);
  return us256 <= us128 && us256 <= us64 ? kFc256 : us128 <= us64 ? kFc128 : kFc64;
}
} // namespace mi355x

#endif
