// Which workgroup of latent attention (latent.h) takes which piece of the keys for which block of rows, plain C++ for
// the device and for the host.
#pragma once
#include "index.h"

namespace fa {

constexpr int kXcds = 8;  // workgroup x runs on XCD x % 8

// The rt row blocks of a piece read the same keys. `near`: they run in workgroups kXcds apart, at one time on one XCD, and
// all but the first find the keys in its L2; pieces go round the XCDs.  Else blocks are neighbours, and so each piece's are on
// all XCDs.  Near is for few blocks of many pieces; with many blocks there are few pieces (a workgroup per compute unit in all), and
// near each other they fill some XCDs and leave others idle.  In us near / not (heads x queries, 64 rows a block): 24 rows of 128 heads
// 62 / 65, of 64 x 8 to 3000 keys 127 / 132, 16 of 32 x 3 39.7 / 41.4; 24 of 64 x 12 207 / 196, 12 of 64 x 36 294 / 194, one of
// 64 x 12 to 8192 keys 68 / 45, of 128 x 100 2160 / 309, of 128 x 300 to 4096 3213 / 495, to 300 644 / 99.
constexpr int kNearBlocks = 8;
FA_HD bool latent_near(long long pieces, int rt) { return rt > 1 && rt <= kNearBlocks && pieces >= kXcds; }
struct LatentPlace {
  int piece, block;
};
FA_HD LatentPlace latent_place(int wg, int rt, bool near) {
  if (!near) return LatentPlace{wg / rt, wg % rt};
  const int slot = wg / kXcds;
  return LatentPlace{slot / rt * kXcds + wg % kXcds, slot % rt};
}
FA_HD long long latent_grid(long long pieces, int rt, bool near) {
  return near ? (pieces + kXcds - 1) / kXcds * kXcds * rt : pieces * rt;
}

}  // namespace fa
