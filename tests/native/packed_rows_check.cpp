// Packed rows of any starts, falling ones too (csrc/prefill_plan.h): every token in one span, the tiles of all spans no more than the
// launch has, and rising starts as they are. Prints "ok" or where it differs.
#include <cstdio>
#include <vector>

#include "prefill_plan.h"

using namespace fa;

static unsigned seed = 7;
static int draw(int lo, int hi) {
  seed = seed * 1664525u + 1013904223u;
  return lo + (int)((seed >> 8) % (unsigned)(hi - lo + 1));
}

int main() {
  for (int n = 0; n < 40000; ++n) {
    const int B = draw(1, 150), g = draw(1, 9), total = draw(0, 900);
    std::vector<int> starts(B + 1);
    for (int& s : starts) s = n % 3 == 0 ? draw(-2000, 2000) : n % 3 == 1 ? draw(0, total) : 0;
    if (n % 3 == 2)
      for (int b = 1; b <= B; ++b) starts[b] = draw(0, 4) ? starts[b - 1] + draw(0, 2 * total / B) : starts[b - 1];
    std::vector<int> seen(total, 0);
    long long tiles = 0;
    int high = 0;
    for (int b = 0; b < B + 2; ++b) {
      TokenSpan t = packed_span(starts.data(), b, B, total);
      if (b <= B) {
        const TokenSpan was = t;
        high = t.s > high ? t.s : high;
        t = span_behind(t, high);
        if (n % 3 == 2 && (t.s != was.s || t.e != was.e)) return std::printf("rising starts: row %d\n", b), 1;
      }
      if (t.s < 0 || t.e < t.s || t.e > total) return std::printf("span [%d, %d) of %d tokens\n", t.s, t.e, total), 1;
      for (int i = t.s; i < t.e; ++i) ++seen[i];
      tiles += row_tiles(t.e - t.s, g);
    }
    for (int i = 0; i < total; ++i)
      if (seen[i] != 1) return std::printf("token %d in %d spans\n", i, seen[i]), 1;
    if (tiles > prefill_tiles(true, B, total, g)) return std::printf("%lld tiles\n", tiles), 1;
  }
  std::printf("ok\n");
}
