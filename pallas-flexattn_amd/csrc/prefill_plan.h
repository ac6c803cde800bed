// Work partition of attention of chunks of new tokens over a paged cache (prefill.h), plain C++ for the
// device and for the host.
//
// The g query heads of a kv head share its keys: a batch row's q queries are g q rows (row r: query r / g, head
// r % g of the group), kPrefillRows of them a work item, so an item's rows are neighbours in
// time and see nearly the same keys, and a short chunk still fills an item.
#pragma once
#include "decode_index.h"

namespace fa {

struct PrefillArgs {
  const void* q;            // bf16; element strides of (row, head, token)
  long long qsb, qsh, qst;
  void* o;
  long long osb, osh, ost;
  float* lse;               // (B, Hq, Sq), packed (Hq, Sq)
  const char *k, *v;        // (num_pages, Hkv, page_size, D)
  const float *ks, *vs;     // e4m3: (num_pages, Hkv, page_size / 32)
  const int *page_table, *kv_lens, *q_lens;
  const int* starts;        // packed: (B + 1), Sq tokens in all
  int B, Hq, Hkv, Sq, g;
  int page_runs, max_pages, num_pages, cap;
  int win_left, win_right;
  float scale, scale_log2, softcap;
  const float* alibi;
  int tiles;                // row tiles (of each kv head)
  int n_splits;             // most ranges that an item's keys are cut into;
  int few;                  // the first so many items have one less
  float* part;              // n_splits > 1: (n_splits, rows, D), then (m, l) (n_splits, rows, 2); rows as lse's
};

constexpr int kPrefillRows = 128;  // rows of a work item
constexpr int kPrefillKeys = 64;   // keys of a tile

// Tokens [s, e) of packed rows: b in [0, B) a batch row; B and B + 1 the tokens behind the last and before the first, which
// belong to none.
struct TokenSpan {
  int s, e;
};
FA_HD TokenSpan packed_span(const int* starts, int b, int B, int total) {
  TokenSpan t;
  const int first = starts[b < B ? b : B], next = starts[b < B ? b + 1 : 0];  // (both at once, in no branch)
  t.s = b <= B ? clamp_len(first, total) : 0;
  t.e = b == B ? total : clamp_len(next, total);
  if (t.e < t.s) t.e = t.s;
  return t;
}
// A start below an earlier one counts as the highest before it (of row b: `before`), so that every token is in one span and
// the call writes all results, whatever the starts are.
FA_HD TokenSpan span_behind(TokenSpan t, int before) {
  if (t.s < before) t.s = before;
  if (t.e < t.s) t.e = t.s;
  return t;
}
FA_HD int row_tiles(int queries, int g) {  // (queries * g < 2^31: the host's check)
  const int rows = queries * g;
  return rows / kPrefillRows + (rows % kPrefillRows != 0);
}
// Row tiles of a call at most: packed rows end in a partly filled tile each.
FA_HD long long prefill_tiles(bool packed, int B, int tokens, int g) {
  const long long rows = (long long)tokens * g;
  if (packed) return rows / kPrefillRows + B + 2;
  return B * ((rows + kPrefillRows - 1) / kPrefillRows);
}

// Keys that the query at position pos sees of a row with `have` keys: [lo, hi] (hi < lo: none).
struct KeySpan {
  int lo, hi;
};
FA_HD KeySpan key_span(int pos, int have, int left, int right) {
  KeySpan k;
  k.lo = left < 0 ? 0 : window_first(pos, left);
  const long long end = right < 0 ? have - 1 : (long long)pos + right;
  k.hi = end < have - 1 ? (int)(end < -1 ? -1 : end) : have - 1;
  return k;
}
// Tiles [t0, t1) of kPrefillKeys that queries i0 .. i1 (of ql, standing at have - ql + i) see.
struct TileSpan {
  int t0, t1;
};
FA_HD TileSpan tile_span(int have, int ql, int i0, int i1, int left, int right) {
  const KeySpan a = key_span(have - ql + i0, have, left, right), b = key_span(have - ql + i1, have, left, right);
  if (b.hi < a.lo || i1 < i0) return TileSpan{0, 0};
  return TileSpan{a.lo / kPrefillKeys, b.hi / kPrefillKeys + 1};
}

// Joins of at most this many threads (chunks and latent rows alike) take four waves for each one's elements: the join of a 4001-key
// row in 63 pieces takes 3 us less, of 608 rows of 9 splits 0.7 us; of 1536 latent rows in 6 pieces 2.9 us more.
constexpr long long kMergeWide = 1 << 17;

// Ranges of keys that an item is cut into where there are fewer items than `want`, the workgroups that run at a time: each at least
// a tile of the longest row, at most kPrefillSplits.  If the items are `even`, the last of them get one range more, so
// that `want` workgroups come out: 375 of 512 in one range each leave half the compute units with one workgroup and
// half with two (8192 keys, D = 128: 237 us, 257 whole, 245 all in two).
constexpr int kPrefillSplits = 32;
struct PrefillCut {
  int n, few;  // ranges; the first `few` items have one less
};
FA_HD PrefillCut prefill_cut(long long items, int most_tiles, int want, bool even) {
  if (items >= want) return PrefillCut{1, 0};
  const int most = most_tiles < kPrefillSplits ? most_tiles : kPrefillSplits;
  const long long n = want / items;
  if (n >= most) return PrefillCut{most < 1 ? 1 : most, 0};
  if (!even || items * n == want) return PrefillCut{(int)n, 0};
  return PrefillCut{(int)n + 1, (int)(items * (n + 1) - want)};
}
// Workgroups of the call, and what workgroup x does: range `split` of the item's `ranges`.
FA_HD long long prefill_grid(const PrefillArgs& a) { return (long long)a.tiles * a.Hkv * a.n_splits - a.few; }
struct PrefillRange {
  int item, split, ranges;
};
FA_HD PrefillRange prefill_range(const PrefillArgs& a, int x) {
  if (a.n_splits == 1) return PrefillRange{x, 0, 1};
  const int items = a.tiles * a.Hkv, split = x / items;
  int item = x - split * items;
  if (a.few && split == a.n_splits - 1) item += a.few;
  return PrefillRange{item, split, a.n_splits - (item < a.few ? 1 : 0)};
}

}  // namespace fa
