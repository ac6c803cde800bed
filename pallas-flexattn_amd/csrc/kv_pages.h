// The pages of a paged KV cache for gfx950: copies of whole pages in every
// tensor of every layer, and the plans of a fork and of a compaction (which pages the
// rows of a batch go on with, which are copied where), all on whole numbers.
//
// Copies are bound by HBM (2 bytes moved a byte): one launch for all tensors of up to
// kCopyTensors, in pieces of kCopyPiece bytes, four 16-byte loads a thread before its stores.
//
// Plans are bound by latency: a chain of a few dependent reads (parent, length, page
// id), a mark per page, and ranks of the free pages.  Where marks and rows fit in LDS one
// workgroup does all of it in one launch; else the marks lie in the workspace and three
// launches (a compaction: four) follow each other.  A mark is the smallest claim on its page, so no result
// depends on the order of the atomics.  In the larger plans, too, one workgroup ranks all pages, which is most of their time:
// a fork / a compaction of 8 rows of 100 pages among 24000 16 / 34 us (one launch), among 50000 36 / 76, among 500000 229 / 559;
// 64 rows of 4096 among 300000 192 / 682 (pages of 128 bytes, so that the copies take little).
#pragma once
#include "common.h"
#include "page_plan.h"

namespace fa {

// Bytes [0, n) from s to d (T-aligned both, n a multiple of sizeof(T)).
template <typename T>
__device__ __forceinline__ void copy_piece(const char* s, char* d, int n) {
  const int tid = threadIdx.x;
  const int m = n / (int)sizeof(T);
  T x[4];
  for (int i0 = 0; i0 < m; i0 += 1024) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + 256 * j + tid < m) x[j] = reinterpret_cast<const T*>(s)[i0 + 256 * j + tid];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + 256 * j + tid < m) reinterpret_cast<T*>(d)[i0 + 256 * j + tid] = x[j];
  }
}

__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a) {
  const int per = a.first[a.count];
  const int pairs = a.live ? min(scalar_load(a.live, 0), a.pairs) : a.pairs;
  const long long items = (long long)pairs * per;
  for (long long it = blockIdx.x; it < items; it += gridDim.x) {
    const int pair = (int)(it / per), piece = (int)(it - (long long)pair * per);
    const int src = scalar_load(a.src, pair), dst = scalar_load(a.dst, pair);
    if (src < 0 || src >= a.num_pages || dst < 0 || dst >= a.num_pages || src == dst) continue;
    int t = 0;  // the tensor of this piece
    for (int step = kCopyTensors / 2; step; step >>= 1)
      if (t + step < a.count && piece >= a.first[t + step]) t += step;
    const long long bytes = a.page_bytes[t], off = (long long)(piece - a.first[t]) * kCopyPiece;
    const int n = (int)min((long long)kCopyPiece, bytes - off);
    char* base = static_cast<char*>(a.data[t]) + off;
    const char* s = base + src * bytes;
    char* d = base + dst * bytes;
    if (((bytes | (long long)reinterpret_cast<uintptr_t>(a.data[t])) & 15) == 0) copy_piece<u32x4>(s, d, n);
    else copy_piece<uint32_t>(s, d, n);
  }
}

// ------------------------------------------------------------------ plans ----
// Exclusive sum over the workgroup's threads, *all: the total.  Every thread calls it;
// `part` holds a number per wave and is free again behind the call.
__device__ __forceinline__ int block_scan(int x, int* part, int* all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(s, d, 64);
    if (lane >= d) s += y;
  }
  if (lane == 63) part[w] = s;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    const int p = part[i];
    before += i < w ? p : 0;
    sum += p;
  }
  __syncthreads();
  *all = sum;
  return before + s - x;
}

// The marks of the pages in the workspace (atomics and reads past the caches: other workgroups write them too).
struct Marks {
  int* p;
  __device__ __forceinline__ void set(int i, int x) const { p[i] = x; }
  __device__ __forceinline__ void claim(int i, int x) const { atomicMin(&p[i], x); }
  __device__ __forceinline__ int get(int i) const { return __hip_atomic_load(&p[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
};

__device__ __forceinline__ void marks_init(const PagePlan& a, const Marks& m, int tid, int stride) {
  for (int i = tid; i < a.num_pages; i += stride) m.set(i, a.keep && a.keep[i] ? kPageHeld : kPageFree);
}

// Rows wave, wave + waves, ..: the entries that a row keeps go into the new table, whole pages and last ones are claimed.
__device__ __forceinline__ void fork_mark(const PagePlan& a, const Marks& m, int wave, int waves) {
  const int lane = threadIdx.x & 63;
  for (int b = wave; b < a.N; b += waves) {
    const ForkRow r = fork_row(a, b);
    const int* from = a.table + (size_t)r.parent * a.max_pages;
    int* to = a.out_table + (size_t)b * a.max_pages;
    for (int e = lane; e < a.max_pages; e += 64) {
      const int id = e < r.have ? from[e] : -1;
      to[e] = id;
      if (e < r.have && id >= 0 && id < a.num_pages) m.claim(id, e < r.whole ? kPageHeld : b);
    }
    if (lane == 0) a.out_lens[b] = r.len;
  }
}

// One workgroup: which rows need fresh pages, the free ones in ascending order, and who gets which.
__device__ __forceinline__ void fork_assign(const PagePlan& a, const Marks& m, int* part) {
  const int tid = threadIdx.x;
  int need = 0;  // of all rows so far
  for (int b0 = 0; b0 < a.N; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int mine = 0, copy = 0;
    if (b < a.N) {
      const ForkRow r = fork_row(a, b);
      if (r.have > r.whole) {
        const int id = a.table[(size_t)r.parent * a.max_pages + r.whole];
        copy = id >= 0 && id < a.num_pages && m.get(id) != b;
      }
      mine = copy + r.want - r.have;
    }
    int all;
    const int first = block_scan(mine, part, &all);
    if (b < a.N) {
      a.first[b] = need + first;
      a.pair_src[b] = copy;  // (the page's id later)
    }
    need += all;
  }
  int free = 0;
  for (int p0 = 0; p0 < a.num_pages; p0 += 4 * kPlanThreads) {
    const int p = p0 + 4 * tid;
    bool is[4];
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      is[j] = p + j < a.num_pages && m.get(p + j) == kPageFree;
      n += is[j];
    }
    int all;
    int rank = free + block_scan(n, part, &all);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (is[j]) {
        if (rank < need) a.list[rank] = p + j;
        ++rank;
      }
    free += all;
  }
  if (tid == 0) *a.out_count = free - need;
  __syncthreads();  // (the lists are read below by other waves than wrote them)
  const int lane = tid & 63;
  for (int b = tid >> 6; b < a.N; b += kPlanThreads / 64) {
    const ForkRow r = fork_row(a, b);
    const int first = a.first[b], copy = a.pair_src[b];
    int* to = a.out_table + (size_t)b * a.max_pages;
    for (int i = lane; i < r.want - r.have; i += 64) {
      const int at = first + copy + i;
      to[r.have + i] = at < free ? a.list[at] : -1;
    }
    if (lane == 0) {
      int src = -1, dst = -1;
      if (copy) {
        src = a.table[(size_t)r.parent * a.max_pages + r.whole];
        dst = first < free ? a.list[first] : -1;
        to[r.whole] = dst;
      }
      a.pair_src[b] = src;
      a.pair_dst[b] = dst;
    }
  }
}

// Every page id that a row names is claimed as used (kPageUsed; what others hold keeps its mark).
__device__ __forceinline__ void compact_mark(const PagePlan& a, const Marks& m, int wave, int waves) {
  const int lane = threadIdx.x & 63;
  for (int b = wave; b < a.N; b += waves) {
    const ForkRow r = fork_row(a, b);
    const int* from = a.table + (size_t)b * a.max_pages;
    for (int e = lane; e < r.want; e += 64) {
      const int id = from[e];
      if (id >= 0 && id < a.num_pages) m.claim(id, kPageUsed);
    }
  }
}

// One workgroup: pages past the number in use move to the free ones before it; a mark becomes its page's new id.
__device__ __forceinline__ void compact_assign(const PagePlan& a, const Marks& m, int* part) {
  const int tid = threadIdx.x;
  int n = 0;
  for (int i = tid; i < a.num_pages; i += kPlanThreads) n += m.get(i) != kPageFree;
  int used;
  block_scan(n, part, &used);
  int slots = 0;
  for (int p0 = 0; p0 < used; p0 += kPlanThreads) {
    const int p = p0 + tid;
    const bool is = p < used && m.get(p) == kPageFree;
    int all;
    const int rank = slots + block_scan(is, part, &all);
    if (is) a.list[rank] = p;
    slots += all;
  }
  __syncthreads();
  int moved = 0;
  for (int p0 = 0; p0 < a.num_pages; p0 += kPlanThreads) {
    const int p = p0 + tid;
    const bool is = p >= used && p < a.num_pages && m.get(p) == kPageUsed;
    int all;
    const int rank = moved + block_scan(is, part, &all);
    if (is) {  // (pages in use past the number in use: no more than free ones before it)
      a.pair_src[rank] = p;
      a.pair_dst[rank] = a.list[rank];
    }
    if (p < a.num_pages) m.set(p, is ? a.list[rank] : p);
    moved += all;
  }
  if (tid == 0) {
    *a.out_count = used;
    *a.moved = moved;
  }
}

__device__ __forceinline__ void compact_write(const PagePlan& a, const Marks& m, int wave, int waves) {
  const int lane = threadIdx.x & 63;
  for (int b = wave; b < a.N; b += waves) {
    const ForkRow r = fork_row(a, b);
    for (int e = lane; e < a.max_pages; e += 64) {
      const size_t at = (size_t)b * a.max_pages + e;
      int id = -1;
      if (e < r.want) {
        id = a.table[at];
        if (id >= 0 && id < a.num_pages) id = m.get(id);
      }
      a.out_table[at] = id;
    }
  }
}

// f(i, x[i]) of i < n over the workgroup's threads, eight loads x(i) under way at a time.
template <class X, class F>
__device__ __forceinline__ void plan_each(int n, int tid, X x, F f) {
  for (int i0 = tid; i0 < n; i0 += 8 * kPlanThreads) {
    int y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = i0 + j * kPlanThreads < n ? x(i0 + j * kPlanThreads) : 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * kPlanThreads < n) f(i0 + j * kPlanThreads, y[j]);
  }
}
__device__ __forceinline__ void plan_marks(const PagePlan& a, int* marks, int tid) {
  plan_each(a.num_pages, tid, [&](int i) { return a.keep ? (int)a.keep[i] : 0; },
            [&](int i, int held) { marks[i] = held ? kPageHeld : kPageFree; });
}

// A small fork in one launch.  Rows are a thread's each at first (a row after the other in a wave took 2 us a row: three
// reads that wait for each other), entries all threads' together; a free page's thread finds by its rank
// the row that gets it and writes it there.  64 rows of 57 pages among 6000: 11.2 us with rows by waves and the free pages
// in a list, 9.8 so (8 rows of one prompt 6).
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(PagePlan a) {
  __shared__ int marks[kPlanPages];
  __shared__ int parent[kPlanRows], len[kPlanRows], want[kPlanRows], first[kPlanRows], last[kPlanRows];  // last: a page to copy, or -1
  __shared__ int part[kPlanThreads / 64];
  const int tid = threadIdx.x;
  plan_marks(a, marks, tid);
  ForkRow mine{0, 0, 0, 0, 0};
  int id = -1;
  if (tid < a.N) {
    mine = fork_row(a, tid);
    parent[tid] = mine.parent;
    len[tid] = mine.len;
    want[tid] = mine.want;
    a.out_lens[tid] = mine.len;
    if (mine.have > mine.whole) id = a.table[(size_t)mine.parent * a.max_pages + mine.whole];
    if (id >= a.num_pages) id = -1;
  }
  __syncthreads();
  const int entries = a.N * a.max_pages;
  plan_each(entries, tid,
            [&](int i) {
              const int b = i / a.max_pages, e = i - b * a.max_pages;
              return (long long)e * a.page_size < len[b] ? a.table[(size_t)parent[b] * a.max_pages + e] : -1;
            },
            [&](int i, int x) {
              const int b = i / a.max_pages, e = i - b * a.max_pages;
              a.out_table[i] = x;
              // (every claim on such a page says so or more)
              if ((e + 1ll) * a.page_size <= len[b] && x >= 0 && x < a.num_pages) marks[x] = kPageHeld;
            });
  __syncthreads();
  if (id >= 0) atomicMin(&marks[id], tid);
  __syncthreads();
  const bool copy = id >= 0 && marks[id] != tid;
  int need;
  const int at = block_scan(tid < a.N ? copy + mine.want - mine.have : 0, part, &need);
  if (tid < a.N) {
    first[tid] = at;
    last[tid] = copy ? id : -1;
  }
  __syncthreads();
  int free = 0;
  for (int p0 = 0; p0 < a.num_pages; p0 += 4 * kPlanThreads) {
    const int p = p0 + 4 * tid;
    bool is[4];
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      is[j] = p + j < a.num_pages && marks[imin(p + j, kPlanPages - 1)] == kPageFree;
      n += is[j];
    }
    int all;
    int rank = free + block_scan(n, part, &all);
    free += all;
    if (rank >= need) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!is[j]) continue;
      if (rank < need) {  // of the rows that begin there the last one: those before it need none
        int lo = 0, hi = a.N;
        while (hi - lo > 1) {
          const int mid = (lo + hi) / 2;
          if (first[mid] <= rank) lo = mid;
          else hi = mid;
        }
        const int k = rank - first[lo], c = last[lo] >= 0;
        const int whole = (unsigned)len[lo] / (unsigned)a.page_size, have = whole + ((unsigned)len[lo] % (unsigned)a.page_size != 0u);
        a.out_table[(size_t)lo * a.max_pages + (c && k == 0 ? whole : have + k - c)] = p + j;
        if (c && k == 0) a.pair_dst[lo] = p + j;
      }
      ++rank;
    }
  }
  if (tid == 0) *a.out_count = free - need;
  if (tid < a.N) {
    a.pair_src[tid] = copy && at < free ? id : -1;
    if (copy && at >= free) a.out_table[(size_t)tid * a.max_pages + mine.whole] = -1;  // none left
  }
}

// A small compaction in one launch.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(PagePlan a) {
  __shared__ int marks[kPlanPages];
  __shared__ uint16_t list[kPlanPages / 2 + 1];
  __shared__ int want[kPlanRows];
  __shared__ int part[kPlanThreads / 64];
  const int tid = threadIdx.x;
  plan_marks(a, marks, tid);
  if (tid < a.N) want[tid] = fork_row(a, tid).want;
  __syncthreads();
  const int entries = a.N * a.max_pages;
  auto entry = [&](int i) {
    const int b = i / a.max_pages;
    return i - b * a.max_pages < want[b] ? a.table[i] : -1;
  };
  plan_each(entries, tid, entry, [&](int, int x) {
    if (x >= 0 && x < a.num_pages) atomicMin(&marks[x], kPageUsed);
  });
  __syncthreads();
  int n = 0;
  for (int i = tid; i < a.num_pages; i += kPlanThreads) n += marks[i] != kPageFree;
  int used;
  block_scan(n, part, &used);
  int slots = 0;
  for (int p0 = 0; p0 < used; p0 += kPlanThreads) {
    const int p = p0 + tid;
    const bool is = p < used && marks[p] == kPageFree;
    int all;
    const int rank = slots + block_scan(is, part, &all);
    if (is) list[rank] = (uint16_t)p;
    slots += all;
  }
  __syncthreads();
  int moved = 0;
  for (int p0 = used / kPlanThreads * kPlanThreads; p0 < a.num_pages; p0 += kPlanThreads) {
    const int p = p0 + tid;
    const bool is = p >= used && p < a.num_pages && marks[p] == kPageUsed;
    int all;
    const int rank = moved + block_scan(is, part, &all);
    if (is) {  // (pages in use past the number in use: no more than free ones before it)
      const int to = list[rank];
      a.pair_src[rank] = p;
      a.pair_dst[rank] = to;
      marks[p] = to;
    }
    moved += all;
  }
  if (tid == 0) {
    *a.out_count = used;
    *a.moved = moved;
  }
  __syncthreads();
  plan_each(entries, tid, entry, [&](int i, int x) {
    if (x >= used && x < a.num_pages && marks[x] >= 0) x = marks[x];  // (what others hold stays)
    a.out_table[i] = x;
  });
}

// Larger ones in launches of their own, the marks in the workspace.
__global__ __launch_bounds__(256) void page_init_kernel(PagePlan a) {
  marks_init(a, Marks{a.marks}, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}
template <bool kFork>
__global__ __launch_bounds__(256) void page_mark_kernel(PagePlan a) {
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if constexpr (kFork) fork_mark(a, Marks{a.marks}, blockIdx.x * 4 + wave, gridDim.x * 4);
  else compact_mark(a, Marks{a.marks}, blockIdx.x * 4 + wave, gridDim.x * 4);
}
template <bool kFork>
__global__ __launch_bounds__(kPlanThreads) void page_assign_kernel(PagePlan a) {
  __shared__ int part[kPlanThreads / 64];
  if constexpr (kFork) fork_assign(a, Marks{a.marks}, part);
  else compact_assign(a, Marks{a.marks}, part);
}
__global__ __launch_bounds__(256) void page_write_kernel(PagePlan a) {
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  compact_write(a, Marks{a.marks}, blockIdx.x * 4 + wave, gridDim.x * 4);
}

}  // namespace fa
