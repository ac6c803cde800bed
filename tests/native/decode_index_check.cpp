// The work partition of decode over a paged cache (csrc/decode_index.h) on the
// CPU: for many batches of lengths, windows, query blocks and chunk sizes, the
// pieces of every item cover its tiles exactly once, none is longer than the
// chunk, the units fit the grid and the pieces of divided items the slots that
// the host reserves.  Prints "ok <cases> <tiles>".
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "decode_index.h"

using namespace fa;

[[noreturn]] static void fail(const char* what, long long a = 0, long long b = 0) {
  std::fprintf(stderr, "%s (%lld, %lld)\n", what, a, b);
  std::abort();
}

int main() {
  std::mt19937 rng(5);
  auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
  long long cases = 0, tiles = 0;
  for (int it = 0; it < 4000; ++it) {
    const int B = pick(1, it % 7 == 0 ? 300 : 9), Hkv = pick(1, 5), rt = pick(1, 3), Sq = pick(1, 6);
    const int cap = it % 5 == 0 ? pick(1, 40) : pick(1, 5000), left = pick(0, 2) ? -1 : pick(0, 700);
    const int pieces = pick(1, 512), least = pick(1, 20);
    std::vector<DecodeSpan> span;
    long long total = 0;
    int most = 1;
    for (int b = 0; b < B; ++b) {
      const int have = clamp_len(pick(-3, cap + 3), cap), ql = clamp_len(pick(-1, Sq + 1), Sq);
      const DecodeSpan s = decode_span(have, ql, left);
      if (s.n < 1 || s.lo < 0) fail("span", s.lo, s.n);
      // every key that a query sees lies in the span, and the span in the row's tiles
      for (int i = 0; i < ql; ++i) {
        const int at = have - ql + i, lo = left < 0 ? 0 : imax(0, at - left);
        if (lo < have && (lo / kTileKeys < s.lo || (have - 1) / kTileKeys >= s.lo + s.n)) fail("key outside", lo, have);
      }
      if (ql > 0 && have > 0 && s.lo + s.n > (have + kTileKeys - 1) / kTileKeys) fail("span past the keys", s.lo, s.n);
      span.push_back(s);
      total += (long long)s.n * Hkv * rt;
      most = imax(most, s.n);
    }
    // the longest walk that the host can know of
    int bound = (cap + kTileKeys - 1) / kTileKeys;
    if (left >= 0) bound = imin(bound, (left + Sq + kTileKeys - 2) / kTileKeys + 1);
    if (most > bound) fail("walk longer than the host's bound", most, bound);
    int chunk = decode_chunk((int)total, pieces, least);
    if ((long long)chunk * pieces < total || chunk < least) fail("chunk", chunk, total);
    for (int i = 0;; ++i) {  // as the device does
      long long all = 0;
      for (int b = 0; b < B; ++b) all += (long long)decode_pieces(span[b].n, chunk) * Hkv * rt;
      if (all <= pieces || B * Hkv * rt >= pieces || i == kChunkTries) break;
      const int next = decode_next_chunk(chunk, (int)all, pieces);
      if (next <= chunk) fail("chunk does not grow", next, chunk);
      chunk = next;
    }
    long long units = 0, slots = 0;
    for (int b = 0; b < B; ++b) {
      const int n = span[b].n, p = decode_pieces(n, chunk);
      int at = 0;
      for (int i = 0; i < p; ++i) {
        const int lo = decode_piece(n, p, i), hi = decode_piece(n, p, i + 1);
        if (lo != at || hi <= lo || hi - lo > chunk) fail("piece", lo, hi);
        at = hi;
        tiles += hi - lo;
      }
      if (at != n) fail("tiles left out", at, n);
      units += (long long)p * Hkv * rt;
      if (p > 1) slots += (long long)p * Hkv * rt;
    }
    const long long grid = decode_grid((long long)B * Hkv * rt, bound, pieces, least);
    if (units > grid) fail("more units than workgroups", units, grid);
    if (slots > decode_slots(grid, pieces)) fail("more pieces than slots", slots, pieces);
    ++cases;
  }
  std::printf("ok %lld %lld\n", cases, tiles);
  return 0;
}
