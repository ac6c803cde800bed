// The first key that a query with a window sees (csrc/decode_index.h), at positions and
// windows near the ends of 32 bits, against 64-bit arithmetic; built with
// UndefinedBehaviorSanitizer, so that a sum past 32 bits ends the run.  Prints "ok <cases>".
#include <climits>
#include <cstdio>
#include <cstdlib>

#include "decode_index.h"

int main() {
  const int most = INT_MAX - 2 * fa::kTileKeys, rows = (1 << 27) - 1;  // keys, and queries of a row, at most
  const int pos[] = {-rows, -rows + 1, -1, 0, 1, 31, 32, rows, most - 1, most};
  const int left[] = {0, 1, 31, 32, rows, most / 2, most - 1, most};
  int n = 0;
  for (int p : pos)
    for (int l : left) {
      const long long want = (long long)p - l;
      if (fa::window_first(p, l) != (want > 0 ? want : 0)) {
        std::fprintf(stderr, "position %d, left %d: %d\n", p, l, fa::window_first(p, l));
        return 1;
      }
      // (decode_span's first tile is that key's)
      if (p >= 0 && p < most) {
        const fa::DecodeSpan s = fa::decode_span(p + 1, 1, l);
        if (s.lo != fa::window_first(p, l) / fa::kTileKeys || s.n < 1) {
          std::fprintf(stderr, "span of position %d, left %d: %d, %d\n", p, l, s.lo, s.n);
          return 1;
        }
      }
      ++n;
    }
  std::printf("ok %d\n", n);
  return 0;
}
