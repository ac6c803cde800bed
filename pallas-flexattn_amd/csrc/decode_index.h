// Work partition of attention over a paged cache (decode_fp8.h), plain C++ for
// the device and for the host: which tiles of which item a workgroup takes,
// and where the pieces of an item that several workgroups share lie.
//
// An item is (batch row b, kv head, block of query rows); it walks n_b tiles of
// kTileKeys keys, from the first one that a query sees. A workgroup takes one
// item, or where an item's walk is longer than the call's chunk one of its
// ceil(n_b / chunk) equal pieces: rows of any lengths give pieces of about the
// same size, and no workgroup more than a chunk.
#pragma once
#include "index.h"

namespace fa {

constexpr int kTileKeys = 32;  // keys of a tile: one scale run
// Batch rows whose tiles a lane of a wave keeps, in calls to 256 rows and in larger ones (those
// to 1024 are cut in pieces).
constexpr int kLaneRows = 4, kMostLaneRows = 16;

struct DecodeSpan {
  int lo;  // first tile
  int n;   // tiles (at least one: a row without keys still writes its outputs)
};
// First key that a query at pos (before the first key: negative) with a window of
// left >= 0 sees, if any; no sum here passes 32 bits.
FA_HD int window_first(int pos, int left) { return pos > left ? pos - left : 0; }
// `have` keys, the newest `ql` of them the queries, the window's left reach
// (< 0: none).
FA_HD DecodeSpan decode_span(int have, int ql, int left) {
  const int lo = left >= 0 && ql > 0 ? window_first(have - ql, left) / kTileKeys : 0;  // (have - ql: the first query's position)
  const int end = ql > 0 ? have / kTileKeys + (have % kTileKeys ? 1 : 0) : 0;
  return DecodeSpan{lo < end ? lo : 0, lo < end ? end - lo : 1};
}
FA_HD int clamp_len(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }

// 16-row blocks of an item (`rows` query rows per kv head, `heads` kv heads in all, walks of
// up to `tiles`): one, or two where the group has more than 16 rows and the call is long (from
// 24000 tiles of such items on). 32 rows read the cache half as often but leave half as many
// waves: in us with 16 / 32, D = 128, B1 8 heads of 32 rows 4000 keys 13.1 / 14.9, B32 to 1500 keys
// 29.6 / 31.9, to 6000 105 / 75; 4 heads of 56 102 / 67, of 136 B8 to 4000 28.7 / 33.2, B32 to
// 6000 190 / 128. 64 rows need twice the registers and were slower than 32 everywhere (78, 51.6
// and 164 in the last three).
FA_HD int decode_blocks(long long rows, long long heads, long long tiles) {
  return rows > 16 && heads * ((rows + 31) / 32) * tiles >= 24000 ? 2 : 1;
}

// Tiles per chunk, at first: `total` tiles (of all items) over `pieces` workgroups, at least `least`.
FA_HD int decode_chunk(int total, int pieces, int least) {
  const int c = total / pieces + (total % pieces ? 1 : 0);
  return c > least ? c : least;
}
// The next chunk to try where cutting at `chunk` makes `units` workgroups, more
// than `pieces`: a few workgroups over a round number leave some compute units with one
// more than the others (8 rows of 3277 to 32768 keys: 84.5 us without, 72.4 with it).
constexpr int kChunkTries = 6;
// (over hundreds of rows the rounding evens out, and a try costs a division per row)
constexpr int decode_tries(int lane_rows) { return lane_rows > kLaneRows ? 0 : kChunkTries; }
FA_HD int decode_next_chunk(int chunk, int units, int pieces) {
  const int more = (int)((long long)chunk * (units - pieces) / (2ll * pieces));
  return chunk + (more > 1 ? more : 1);
}
FA_HD int decode_pieces(int n, int chunk) { return n / chunk + (n % chunk ? 1 : 0); }
// Tiles [first, first + count) of piece p of an n-tile walk in `pieces`.
// (n p / pieces in 32 bits: the remainder's product stays under pieces^2, and an
// item has at most about as many pieces as the call asks for in all, a few thousand)
FA_HD int decode_piece(int n, int pieces, int p) {
  const int q = n / pieces, r = n - q * pieces;
  return q * p + r * p / pieces;
}

// Which row a unit lies in.  A lane of a wave holds kRows consecutive rows, the first of them
// number b0: their tiles n (0: no row) and pieces p per item, `each` items per row; its first
// row's units begin at `unit`, its partial results at `slot`.
struct DecodeRow {
  int b, n, p;     // the row, its tiles, its pieces
  int unit, slot;  // where the row's units and slots begin
};
FA_HD void decode_next_row(int p, int each, int* unit, int* slot) {
  *unit += p * each;
  *slot += p > 1 ? p * each : 0;
}
// (the lane whose units `wg` is one of; the others' results mean nothing)
template <int kRows>
FA_HD DecodeRow decode_find_row(int b0, const int (&n)[kRows], const int (&p)[kRows], int each, int wg, int unit, int slot) {
  DecodeRow r{b0, n[0], p[0], unit, slot};
#pragma unroll
  for (int j = 1; j < kRows; ++j) {
    const bool later = r.b == b0 + j - 1 && wg >= r.unit + r.p * each && n[j] != 0;
    int u = r.unit, s = r.slot;
    decode_next_row(r.p, each, &u, &s);
    r = later ? DecodeRow{b0 + j, n[j], p[j], u, s} : r;
  }
  return r;
}

// Workgroups that a call needs at most: items, plus a piece more for every
// chunk's worth of tiles (n / chunk each, and the chunks are `pieces` in all).
FA_HD long long decode_grid(long long items, int most_tiles, int pieces, int least) {
  const long long each = items * decode_pieces(most_tiles, least), sum = items + pieces;
  return each < sum ? each : sum;
}
// Slots for partial results: the pieces of items that have several.  Each of them is
// longer than half a chunk, so there are fewer than 2 total / chunk.
FA_HD long long decode_slots(long long grid, int pieces) { return grid < 2ll * pieces ? grid : 2ll * pieces; }

}  // namespace fa
