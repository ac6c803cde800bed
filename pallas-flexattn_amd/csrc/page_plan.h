// What copies of pages, forks and compactions of paged rows compute from (kv_pages.h), plain C++ for the
// device and for the host.
#pragma once
#include "index.h"

namespace fa {

constexpr int kCopyTensors = 64;        // tensors of a launch (1.3 KB of kernel arguments)
constexpr int kCopyPiece = 16 * 1024;   // bytes of a work item
constexpr int kPlanThreads = 1024;

struct CopyArgs {
  void* data[kCopyTensors];
  long long page_bytes[kCopyTensors];
  int first[kCopyTensors + 1];  // pieces of a page before tensor i; [count]: all
  int count, num_pages, pairs;
  const int *src, *dst;  // pairs of page ids
  const int* live;       // null: all pairs are; else the first *live of them
};

// Marks of a page: the smallest claim on it wins.  A fork's rows claim their partly filled
// last page with their own number, so what stays is the first such row, unless a row has the whole page
// or others keep it.
constexpr int kPageHeld = -1, kPageUsed = 0, kPageFree = 0x7fffffff;

// What one workgroup does in one launch: marks and rows in LDS, and no more table entries than it reads in
// the time of the other form's launches.
constexpr int kPlanPages = 24 * 1024, kPlanRows = 1024, kPlanEntries = 1 << 15;

struct PagePlan {
  const int *table, *kv_lens;  // (B, max_pages), (B)
  const int* parents;          // (N) or null: row b goes on from row b
  const int* room;             // (N) or null: room_all
  const uint8_t* keep;         // (num_pages) or null
  int room_all, B, N, max_pages, page_size, num_pages;
  int *out_table, *out_lens;   // (N, max_pages), (N)
  int* out_count;
  // workspace: marks (num_pages; unused with marks in LDS), first page of each row's
  // fresh ones (N), the free pages, pairs to copy, how many of them (compaction)
  int *marks, *first, *list, *pair_src, *pair_dst, *moved;
};

// Row b of the result: its parent's tokens, the pages that they fill, have at all, and that the row wants with its room.
struct ForkRow {
  int parent, len, whole, have, want;
};
FA_HD ForkRow fork_row(const PagePlan& a, int b) {
  ForkRow r;
  const int p = a.parents ? a.parents[b] : b;
  const bool ok = p >= 0 && p < a.B;
  r.parent = ok ? p : 0;
  // (tokens of a row and its room are below 2^31 each: their sum, and a table's pages times their size, in unsigned 32 and 64 bits)
  const unsigned long long cap = (unsigned long long)a.max_pages * (unsigned)a.page_size;
  const int held = ok ? a.kv_lens[p] : 0, more = a.room ? a.room[b] : a.room_all;
  unsigned n = held > 0 ? (unsigned)held : 0u;
  if (n > cap) n = (unsigned)cap;
  unsigned to = n + (more > 0 ? (unsigned)more : 0u);
  if (to > cap) to = (unsigned)cap;
  const unsigned page = (unsigned)a.page_size;
  r.len = (int)n;
  r.whole = (int)(n / page);
  r.have = r.whole + (n % page != 0u);
  r.want = (int)(to / page + (to % page != 0u));
  return r;
}

}  // namespace fa
