// How the workgroups of a decode call find their work (csrc/decode_index.h), as a wave does
// it: 64 lanes, each with its consecutive rows, the chunk with as many tries as the device makes
// for that many rows, prefix sums over the lanes, then the lane and the row of every
// workgroup.  Every tile of every item is taken exactly once, workgroups past the work find
// none, each piece of a divided item has a slot of its own where the merge looks for it, and all fits the
// grid and the slots that the host reserves.  Prints "ok <cases> <units>".
#include <cstdio>
#include <cstdlib>
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

template <int kRows>
static long long check(const std::vector<int>& tiles, int Hkv, int rt, int pieces, int least, int most) {
  const int B = (int)tiles.size(), each = Hkv * rt, per = (B + 63) / 64;
  if (per > kRows) fail("rows per lane", per, kRows);
  int n[64][kRows], p[64][kRows];
  long long total = 0;
  for (int l = 0; l < 64; ++l)
    for (int j = 0; j < kRows; ++j) {
      const int b = l * per + j;
      n[l][j] = j < per && b < B ? tiles[b] : 0;
      total += n[l][j];
    }
  int chunk = decode_chunk((int)(total * each), pieces, least);
  int units[64], slots[64], upto[64], slot_upto[64];  // a lane's, and with all lanes before it
  int all = 0;
  for (int i = 0;; ++i) {
    all = 0;
    for (int l = 0; l < 64; ++l) {
      units[l] = slots[l] = 0;
      for (int j = 0; j < kRows; ++j) {
        p[l][j] = decode_pieces(n[l][j], chunk);
        decode_next_row(p[l][j], each, &units[l], &slots[l]);
      }
      all += units[l];
      upto[l] = all;
    }
    if (all <= pieces || B * each >= pieces || i == decode_tries(kRows)) break;
    chunk = decode_next_chunk(chunk, all, pieces);
  }
  int all_slots = 0;
  for (int l = 0; l < 64; ++l) slot_upto[l] = all_slots += slots[l];
  const long long grid = decode_grid((long long)B * each, most, pieces, least), room = decode_slots(grid, pieces);
  if (all > grid) fail("more units than workgroups", all, grid);
  if (all_slots > room) fail("more pieces than slots", all_slots, room);
  // what the first workgroup leaves for the merge
  std::vector<int> head(2 * B + 2, -1);
  for (int l = 0; l < 64; ++l) {
    int f = upto[l] - units[l], g = slot_upto[l] - slots[l];
    for (int j = 0; j < kRows; ++j) {
      if (n[l][j]) {
        head[2 * (l * per + j)] = f;
        head[2 * (l * per + j) + 1] = g;
      }
      decode_next_row(p[l][j], each, &f, &g);
    }
  }
  head[2 * B] = all;
  std::vector<std::vector<int>> taken(B, std::vector<int>(each, 0));  // tiles of each item
  std::set<int> used;
  for (int wg = 0; wg < grid; ++wg) {
    int lanes = 0, src = -1;
    for (int l = 63; l >= 0; --l)
      if (wg >= upto[l] - units[l] && wg < upto[l]) ++lanes, src = l;
    if (lanes != (wg < all)) fail("lanes that hold a workgroup's unit", wg, lanes);
    if (src < 0) continue;
    const DecodeRow r = decode_find_row<kRows>(src * per, n[src], p[src], each, wg, upto[src] - units[src], slot_upto[src] - slots[src]);
    if (r.b < 0 || r.b >= B || r.n != tiles[r.b] || r.p != decode_pieces(r.n, chunk)) fail("row", r.b, r.n);
    const int local = wg - r.unit, item = local / r.p, piece = local - item * r.p;
    if (local < 0 || item >= each) fail("item", local, item);
    const int lo = decode_piece(r.n, r.p, piece), hi = decode_piece(r.n, r.p, piece + 1);
    if (lo != taken[r.b][item] || hi <= lo) fail("tiles out of order or taken twice", lo, hi);
    taken[r.b][item] = hi;
    // the merge's view: pieces of the row's items, and this one's slot
    if ((head[2 * r.b + 2] - head[2 * r.b]) / each != r.p || head[2 * r.b] != r.unit) fail("pieces", head[2 * r.b], r.unit);
    if (r.p > 1) {
      const int slot = r.slot + local;
      if (slot != head[2 * r.b + 1] + item * r.p + piece || slot < 0 || slot >= room) fail("slot", slot, room);
      if (!used.insert(slot).second) fail("slot used twice", slot);
    }
  }
  for (int b = 0; b < B; ++b)
    for (int t : taken[b])
      if (t != tiles[b]) fail("tiles left out", t, tiles[b]);
  return all;
}

int main() {
  std::mt19937 rng(11);
  auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
  long long cases = 0, units = 0;
  for (int it = 0; it < 1500; ++it) {
    const int edges[] = {1, 63, 64, 65, 255, 256, 257, 1023, 1024};
    const int B = it % 6 == 0 ? edges[pick(0, 8)] : it % 6 == 1 ? pick(257, 1024) : pick(1, 256);
    const int Hkv = pick(1, B > 256 ? 2 : 5), rt = pick(1, 2), pieces = pick(1, 1024), least = pick(1, 16);
    std::vector<int> tiles(B);
    const int shape = pick(0, 3), longest = pick(1, B > 256 ? 200 : 900);
    int most = 1;
    for (int& t : tiles) {
      t = shape == 0 ? longest : shape == 1 ? pick(1, longest) : pick(0, 20) ? 1 : pick(1, longest);
      most = imax(most, t);
    }
    most += pick(0, 3) ? pick(0, 5000) : 0;  // the table may be wider than the rows
    units += B <= 64 * kLaneRows ? check<kLaneRows>(tiles, Hkv, rt, pieces, least, most)
                                 : check<kMostLaneRows>(tiles, Hkv, rt, pieces, least, most);
    ++cases;
  }
  std::printf("ok %lld %lld\n", cases, units);
  return 0;
}
