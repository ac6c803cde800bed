// Work partition of attention over a paged cache (decode_fp8.h), plain C++ for
// the device and for the host: which tiles of which item a workgroup takes,
// and where the pieces of an item that several workgroups share lie.
//
// An item is (batch row b, kv head, block of query rows); it walks n_b tiles of
// kRunTokens keys, from the first one that a query sees.  All items' tiles,
// one after another (b slowest, then kv head, then query block), are cut into
// equal chunks, one per workgroup: rows of any lengths give every workgroup
// the same number of tiles.
#pragma once
#include "index.h"

namespace fa {

constexpr int kTileKeys = 32;  // keys of a tile: one scale run

struct DecodeSpan {
  int lo;  // first tile
  int n;   // tiles (at least one: a row without keys still writes its outputs)
};
// `have` keys, the newest `ql` of them the queries, the window's left reach
// (< 0: none).
FA_HD DecodeSpan decode_span(int have, int ql, int left) {
  const long long first = left < 0 ? 0 : (long long)have - ql - left;  // (have - ql: the first query's position)
  const int lo = first > 0 && ql > 0 ? (int)(first / kTileKeys) : 0;
  const int end = ql > 0 ? have / kTileKeys + (have % kTileKeys ? 1 : 0) : 0;
  return DecodeSpan{lo < end ? lo : 0, lo < end ? end - lo : 1};
}
FA_HD int clamp_len(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }

// Tiles per chunk: `total` tiles over `wgs` workgroups, at least `least`.
FA_HD int decode_chunk(int total, int wgs, int least) {
  const int c = (total + wgs - 1) / wgs;
  return c > least ? c : least;
}

// Partial results: workgroup w keeps two slots, 2 w for the item that its
// chunk starts in, 2 w + 1 for another one that it ends in.
FA_HD int decode_slot(int w, int item_start, int chunk) { return 2 * w + (item_start > w * chunk ? 1 : 0); }

}  // namespace fa
