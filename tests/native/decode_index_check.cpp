// The work partition of decode over a paged cache (csrc/decode_index.h) on the
// CPU: for many batches of lengths, windows, query blocks and workgroup counts,
// every tile of every item is taken by exactly one workgroup, no two pieces of
// different items share a slot, and the pieces that the merge looks for
// are the ones that the workgroups wrote.  Prints "ok <cases> <tiles>".
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <utility>
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
    const int wgs = pick(1, 512), least = pick(1, 20);
    std::vector<DecodeSpan> span;
    std::vector<int> first{0};
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
      first.push_back(first.back() + s.n * Hkv * rt);
    }
    const int total = first.back(), chunk = decode_chunk(total, wgs, least);
    if ((long long)chunk * wgs < total || chunk < least) fail("chunk", chunk, total);
    std::map<int, int> slot_item;                       // slot -> item start
    std::map<int, std::set<std::pair<int, int>>> got;   // item start -> pieces (slot, tiles)
    std::vector<char> seen(total, 0);
    for (int w = 0; w < wgs; ++w) {
      int pos = w * chunk;
      const int end = imin(pos + chunk, total);
      if (pos >= end) continue;
      int b = 0;
      while (first[b + 1] <= pos) ++b;
      while (pos < end) {
        const DecodeSpan s = span[b];
        const int item = (pos - first[b]) / s.n, istart = first[b] + item * s.n;
        const int nt = imin(istart + s.n, end) - pos;
        if (item >= Hkv * rt || nt < 1) fail("item", item, nt);
        for (int t = pos; t < pos + nt; ++t)
          if (seen[t]++) fail("tile twice", t, w);
        tiles += nt;
        if (nt != s.n) {
          const int slot = decode_slot(w, istart, chunk);
          if (slot < 0 || slot >= 2 * wgs) fail("slot", slot, wgs);
          if (!slot_item.emplace(slot, istart).second) fail("slot twice", slot, w);
          got[istart].insert({slot, nt});
        }
        pos += nt;
        if (pos < end && pos >= first[b + 1]) ++b;
      }
    }
    for (int t = 0; t < total; ++t)
      if (!seen[t]) fail("tile left out", t, total);
    for (int b = 0; b < B; ++b)  // as the merge looks for them
      for (int i = 0; i < Hkv * rt; ++i) {
        const int s = first[b] + i * span[b].n, e = s + span[b].n, w0 = s / chunk, w1 = (e - 1) / chunk;
        std::set<int> want;
        if (w0 != w1)
          for (int w = w0; w <= w1; ++w) want.insert(w == w0 ? decode_slot(w0, s, chunk) : 2 * w);
        std::set<int> have;
        for (const auto& p : got[s]) have.insert(p.first);
        if (have != want) fail("merge", b, i);
      }
    ++cases;
  }
  std::printf("ok %lld %lld\n", cases, tiles);
  return 0;
}
