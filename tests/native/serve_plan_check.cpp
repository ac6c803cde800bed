// The partition of attention of chunks (csrc/prefill_plan.h) and the rows of a page plan (csrc/page_plan.h) against
// plain restatements in 64 bits, at the ends of their 32-bit sizes too.  Prints "ok" or where they differ.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "page_plan.h"
#include "prefill_plan.h"

using namespace fa;
typedef long long i64;

static unsigned seed = 1;
static i64 draw(i64 lo, i64 hi) {
  seed = seed * 1664525u + 1013904223u;
  const i64 x = ((i64)(seed >> 8) << 20) ^ (seed >> 3);
  return lo + x % (hi - lo + 1);
}
static int fail(const char* what, i64 a, i64 b) {
  std::printf("%s: %lld, not %lld\n", what, a, b);
  return 1;
}

static int spans() {
  const int big = 0x7fffffff;
  for (int n = 0; n < 200000; ++n) {
    const bool large = n % 4 == 0;
    const int have = (int)draw(0, large ? big - 200 : 300), ql = (int)draw(0, large ? big - 200 : 200);
    const int left = draw(0, 2) ? (int)draw(0, large ? big : 90) : -1, right = draw(0, 2) ? (int)draw(0, large ? big : 9) : -1;
    if (!ql) continue;
    const int i0 = (int)draw(0, ql - 1), i1 = (int)draw(i0, i0 + 40 < ql ? i0 + 40 : ql - 1);
    i64 lo = 1ll << 40, hi = -1;
    for (int i = i0; i <= i1; ++i) {
      const i64 pos = (i64)have - ql + i;
      const i64 a = left < 0 ? 0 : pos - left > 0 ? pos - left : 0, b = right < 0 ? have - 1 : pos + right < have - 1 ? pos + right : have - 1;
      const KeySpan k = key_span((int)pos, have, left, right);
      const bool none = b < a, knone = k.hi < k.lo;
      if (none != knone || (!none && (k.lo != a || k.hi != b))) return fail("key_span", k.lo, a);
      if (!none) {
        if (a < lo) lo = a;
        if (b > hi) hi = b;
      }
    }
    const TileSpan t = tile_span(have, ql, i0, i1, left, right);
    if (t.t0 < 0 || t.t1 < t.t0 || (i64)t.t1 * kPrefillKeys > (i64)have + kPrefillKeys) return fail("tile_span's end", t.t1, have);
    if (hi >= 0 && (t.t0 > lo / kPrefillKeys || t.t1 < hi / kPrefillKeys + 1)) return fail("tile_span", t.t0, lo);
    // every range of keys of a split call, side by side
    const int splits = (int)draw(1, kPrefillSplits);
    int at = 0;
    for (int s = 0; s < splits; ++s) {
      const SplitRange r = split_range(t.t1 - t.t0, s, splits, 0);
      if (r.it0 != at || r.it1 < r.it0) return fail("split_range", r.it0, at);
      at = r.it1;
    }
    if (at != t.t1 - t.t0) return fail("split_range's end", at, t.t1 - t.t0);
  }
  return 0;
}

// Packed rows: every token in one span, the tiles of all spans no more than the launch has.
static int packed() {
  for (int n = 0; n < 20000; ++n) {
    const int B = (int)draw(1, 70), g = (int)draw(1, 9), total = (int)draw(0, 900);
    std::vector<int> starts(B + 1, 0);
    for (int b = 1; b <= B; ++b) starts[b] = (int)draw(starts[b - 1], b == B || draw(0, 3) ? (starts[b - 1] + total) / 2 : starts[b - 1]);
    if (n % 5 == 0) starts[0] = starts[1];
    if (n % 7 == 0) for (int b = 0; b <= B; ++b) starts[b] = (int)draw(-2000, 2000);  // (nothing may leave the tokens)
    std::vector<int> seen(total, 0);
    i64 tiles = 0;
    for (int b = 0; b < B + 2; ++b) {
      const TokenSpan t = packed_span(starts.data(), b, B, total);
      if (t.s < 0 || t.e < t.s || t.e > total) return fail("packed_span", t.e, total);
      for (int i = t.s; i < t.e; ++i) ++seen[i];
      tiles += row_tiles(t.e - t.s, g);
    }
    if (n % 7 == 0) continue;
    for (int i = 0; i < total; ++i)
      if (seen[i] != 1) return fail("token in spans", seen[i], 1);
    if (tiles > prefill_tiles(true, B, total, g)) return fail("tiles", tiles, prefill_tiles(true, B, total, g));
  }
  return 0;
}

static int rows() {
  const int big = 0x7fffffff;
  for (int n = 0; n < 100000; ++n) {
    const bool large = n % 3 == 0;
    PagePlan a{};
    int len = (int)draw(large ? -big : -9, large ? big : 400), room = (int)draw(large ? -big : -9, large ? big : 400), parent = (int)draw(-1, 1);
    if (n % 11 == 0) len = room = big;
    a.kv_lens = &len;
    a.parents = &parent;
    a.room = &room;
    a.B = a.N = 1;
    a.max_pages = (int)draw(1, large ? big : 9);
    a.page_size = (int)draw(1, large ? big : 70);
    const ForkRow r = fork_row(a, 0);
    const __int128 cap = (__int128)a.max_pages * a.page_size;
    __int128 k = parent == 0 && len > 0 ? len : 0;
    if (k > cap) k = cap;
    __int128 to = k + (room > 0 ? room : 0);
    if (to > cap) to = cap;
    const i64 whole = (i64)(k / a.page_size), have = (i64)((k + a.page_size - 1) / a.page_size), want = (i64)((to + a.page_size - 1) / a.page_size);
    if (r.len != (i64)k || r.whole != whole || r.have != have || r.want != want) return fail("fork_row", r.want, want);
    if (r.want > a.max_pages || r.parent != 0) return fail("fork_row's end", r.want, a.max_pages);
  }
  return 0;
}

// Every range of every item in one workgroup; as many workgroups as are wanted where that can be.
static int cuts() {
  for (int n = 0; n < 4000; ++n) {
    PrefillArgs a{};
    a.tiles = (int)draw(1, 90);
    a.Hkv = (int)draw(1, 9);
    const int items = a.tiles * a.Hkv, tiles = (int)draw(1, 200), want = (int)draw(1, 800);
    const int counted = (int)draw(1, items);  // (of packed rows not all tiles are)
    const PrefillCut c = prefill_cut(counted, tiles, want, n % 3);
    a.n_splits = c.n;
    a.few = c.few;
    if (c.n < 1 || c.n > kPrefillSplits || c.few < 0 || c.few > counted || (c.few && c.n < 2)) return fail("prefill_cut", c.n, c.few);
    if (c.n > 1 && c.n > tiles) return fail("ranges of a walk", c.n, tiles);
    if (n % 3 && counted == items && c.few && prefill_grid(a) != want) return fail("workgroups", prefill_grid(a), want);
    std::vector<int> got((size_t)items * c.n, 0);
    for (int x = 0; x < prefill_grid(a); ++x) {
      const PrefillRange r = prefill_range(a, x);
      if (r.item < 0 || r.item >= items || r.split < 0 || r.split >= r.ranges || r.ranges > c.n) return fail("prefill_range", x, r.item);
      if (r.ranges != c.n - (r.item < c.few ? 1 : 0)) return fail("ranges", r.ranges, c.n);
      ++got[(size_t)r.item * c.n + r.split];
    }
    for (int i = 0; i < items; ++i)
      for (int k = 0; k < c.n; ++k)
        if (got[(size_t)i * c.n + k] != (k < c.n - (i < c.few ? 1 : 0))) return fail("a range's workgroups", i, k);
  }
  return 0;
}

int main() {
  if (spans() || packed() || rows() || cuts()) return 1;
  std::printf("ok\n");
  return 0;
}
