// Latent attention over a paged cache, absorbed form, for gfx950: all heads read one vector c of L
// elements a token, key and value at once, and a rotary part r of R elements that is key only.
//
//   s = scale (q . c + q_r . r),   o = softmax(mask(s)) c      (per head; o has L elements)
//
// (a key W_k c and a value W_v c of a head, with W_k taken into the query and W_v into what follows.)
// A key costs 2 (L + R) bytes and 2 H (2 L + R) operations a query: 16 heads are bound by the
// reads, 128 heads by both. So every key is read from memory once for up to 64 rows (heads x
// queries), and the 64 keys of a tile serve both products from LDS:
//   * S^T = K Q^T (v_mfma_f32_16x16x32_bf16): a wave takes 16 of the tile's keys and all rows, whose Q
//     stays in registers (4 of them per 32 of L + R and 16 rows);
//   * the waves' P meet in LDS (bf16, half a step 2^-8 as for c; sums take the unrounded values), against maxima that
//     they settle together when one of them has grown;
//   * O^T += C^T P^T: a wave takes L / waves of the elements of all rows, so that each value of the
//     tile is read from LDS once for all rows, by transposing reads; O stays in registers.
// Tiles come by LDS DMA, one ahead, two in LDS (147 KB of 160 for L + R = 576: one workgroup per compute unit).
// Chunk c (16 bytes) of key row r sits at chunk c ^ f(r), with f such that 16 rows of one chunk, and
// the 8 rows by 2 chunks of half a transposing read, lie in different banks.
// Measured at L + R = 576: 16 rows of 16 or 64 heads 5.2 TB/s of keys in the walk (a copy: 4.9); 24 ragged rows of 128 heads, 4500 keys
// on average, 54 us and 9 for the join, of the 54 about 5 launch and search, 5 Q and the first tile, 5 the partial O
// (33 MB), 38 the walk: 2.8 us a tile for both blocks of rows, 2.4 with a quarter of the products and 2.1 without the
// copies.  By the counters no unit is busy for a third of the walk (matrix cores 12 us, VALU 10, LDS 8, reads 2.7 TB/s): a SIMD
// has one wave, whose S, exponentials, two barriers and O follow one another with nothing beside them.  S a tile ahead of O,
// in tiles of 32 keys, four of them in LDS: the same within 2 %.
#pragma once
#include "dma.h"
#include "latent_args.h"
#include "prefill_plan.h"

namespace fa {

template <int CH>
FA_HD int latent_swz(int r) {  // CH 16-byte chunks per row, 8 or 4 more than a multiple of 16
  static_assert(CH % 16 == 8 || CH % 16 == 4, "chunks per row");
  if constexpr (CH % 16 == 8) return ((r >> 3) & 1) << 2 | ((r >> 1) & 1) << 1 | ((r >> 2) & 1);
  else return (r >> 2) & 3;
}

// NB: 16-row blocks of an item
template <int L, int R, int NB>
struct LatentShape {
  static constexpr int NW = 4;
  static constexpr int W = L + R, RB = 2 * W, CH = W / 8, KS = W / 32;
  static constexpr int TILE = kLatentKeys * RB, ROWS = 16 * NB;
  static constexpr int HI = CH / 2;                // copies of 1 KB per run
  static constexpr int J = (HI + NW - 1) / NW;     // of them a wave's
  static constexpr int DTW = L / 16 / NW;          // 16-element blocks of O a wave has
  static constexpr int LDS = 2 * TILE + ROWS * 128 + 16 * ROWS + 64;
  static_assert(L % (16 * NW) == 0 && W % 32 == 0 && LDS <= 160 * 1024, "shape");
};

// c += A B with B, a fragment of Q, in AGPRs ('a'; or VGPRs): the compiler would copy it to VGPRs first, 12 moves for
// every 4 products.  In asm the wait states are explicit (common.h, mfma_acc): A comes from LDS, C is read behind
// mma_q_drain.
template <char kReg>
__device__ __forceinline__ void mma_q(f32x4& c, u32x4 a, u32x4 b) {
  if constexpr (kReg == 'a') asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "a"(b));
  else asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mma_q_drain(f32x4& c, f32x4& d) { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(c), "+v"(d)); }
__device__ __forceinline__ void mma_q_drain(f32x4& c, f32x4& d, f32x4& e) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(c), "+v"(d), "+v"(e));
}
__device__ __forceinline__ void mma_q_drain(f32x4& c, f32x4& d, f32x4& e, f32x4& f) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(c), "+v"(d), "+v"(e), "+v"(f));
}

// bits 0 and 16: whether w's two bf16 are infinities or NaN
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) { return (((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15; }

// A workgroup's piece of work.  The partition (decode_index.h) is one of the batch rows' keys: the rt row blocks of a
// batch row take the same pieces (latent_plan.h).
__device__ __forceinline__ DecodeUnit latent_unit(const LatentArgs& a, int wg, bool first_wave) {
  const DecodeArgs& d = a.d;  // (rt = 1)
  const LatentPlace at = latent_place(wg, a.rt, a.near);
  const int piece = at.piece, block = at.block;
  DecodeUnit u;
  if (d.by_item && piece >= d.B) {
    u.b = -1;
    return u;
  }
  // (a row per lane where 64 suffice: a quarter of the divisions of decode_unit, half a microsecond)
  u = !d.by_item && d.B <= 64 ? decode_piece_unit<1>(d, piece, first_wave) : decode_unit(d, piece, first_wave);
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  u = DecodeUnit{uniform(u.b), uniform(u.have), uniform(u.ql), block, uniform(u.t0), uniform(u.nt), uniform(u.slot)};
  if (u.slot >= 0) u.slot = u.slot * a.rt + block;
  return u;
}

template <int L, int R, int NB>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(
    occupancy_for(LatentShape<L, R, NB>::LDS, LatentShape<L, R, NB>::NW, 2))))
void latent_decode_kernel(LatentArgs a) {
  using X = LatentShape<L, R, NB>;
  constexpr int NW = X::NW, RB = X::RB, CH = X::CH, KS = X::KS, TILE = X::TILE, ROWS = X::ROWS, HI = X::HI, J = X::J;
  constexpr int DTW = X::DTW, BN = kLatentKeys;
  constexpr int AHEAD = NB >= 3 ? 2 : NB == 2 ? 5 : 8;  // LDS reads ahead of their products
  constexpr int JS = NB >= 3 ? J : 2 * J;  // copies that go between the products of S, the others between those of O
  constexpr float kLazy = 8.0f;  // a maximum may be this stale (log2): P stays under 2^8
  __shared__ __attribute__((aligned(1024))) char lds[2 * TILE];
  __shared__ __attribute__((aligned(16))) char pbuf[ROWS * 128];
  __shared__ __attribute__((aligned(16))) float red[ROWS][4];
  constexpr int kHigher = 1, kWild = 2;
  __shared__ __attribute__((aligned(16))) int over[4];  // what each wave found in the tile: a higher maximum, values that are not finite
  __shared__ uint32_t wild[NW][2];  // keys of the tile with values that are not finite, as each wave found them

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const DecodeArgs& p = a.d;
  const DecodeUnit u = latent_unit(a, blockIdx.x, w == 0);
  if (u.b < 0) return;
  const int have = u.have, ql = u.ql, RT = p.g * p.Sq;
  const int row0 = u.item * ROWS;
  const int kfirst = u.t0 * kTileKeys;
  const int kend = imin(have, (u.t0 + u.nt) * kTileKeys);  // this piece's keys: [kfirst, kend)
  const int steps = (u.nt + 1) / 2;

  // Rows as lse has them: a head's queries one after another.  (Computed where it is needed: kept, or taken out of
  // the loop by the compiler, it would push Q out of the registers.)
  auto row_span = [&](int n, bool* live) {
    int row = row0 + 16 * n + r;
    asm volatile("" : "+v"(row));
    const int i = imin(row, RT - 1) % p.Sq;
    *live = row < RT && i < ql;
    KeySpan k = key_span(have - ql + i, have, p.win_left, p.win_right);
    return *live ? k : KeySpan{0, 0x7fffffff};  // (the results of others are not written)
  };

  // copies: lane offsets in a run, the same for both runs of a tile, two to a register
  uint32_t dma[(J + 1) / 2] = {};
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = imin((w + NW * j) * 64 + lane, kTileKeys * CH - 1), row = c / CH;
    dma[j / 2] |= (uint32_t)(row * RB + (((c - row * CH) ^ latent_swz<CH>(row)) * 16)) << (16 * (j & 1));
  }
  // lane i holds the run of tile (of 32 keys) tab + i: -1 for none or a bad page
  int tab = u.t0 - 64, run_l = -1;
  auto table = [&](int t0) {
    tab = t0;
    run_l = -1;
    const int t = t0 + lane;
    if (t < u.t0 + u.nt && t * kTileKeys < have) {
      const int pg = t / p.page_runs;
      const int page = pg >= p.max_pages ? -1 : p.page_table ? p.page_table[(size_t)u.b * p.max_pages + pg] : u.b;
      if (page >= 0 && page < p.num_pages) run_l = page * p.page_runs + (t - pg * p.page_runs);
    }
  };
  // The copies of step i's tile: its runs' resources, then 2 J of them one at a time (between the products of S: issued
  // at once, they held up the wave for 1000 cycles).
  struct Copy {
    i32x4 rs[2];
    char* to;
  };
  auto copy_plan = [&](int i, int buf) {
    const int t = u.t0 + 2 * i;
    if (t - tab >= 64) table(t);
    Copy c;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int run = __builtin_amdgcn_readlane(run_l, t + x - tab);  // (t and tab differ by an even number under 64)
      const uint32_t bytes = run < 0 ? 0u : (uint32_t)imax(imin(kTileKeys, kend - (t + x) * kTileKeys), 0) * RB;
      c.rs[x] = make_rsrc(a.cache + (size_t)imax(run, 0) * (kTileKeys * X::W), bytes);
    }
    c.to = lds + buf * TILE + w * 1024;
    return c;
  };
  auto copy_one = [&](const Copy& c, int i) {
    const int x = i / J, j = i % J;
    uint32_t off = dma[j / 2];
    if constexpr (NB >= 3) asm volatile("" : "+v"(off));  // (not unpacked ahead of the loop)
    off = j & 1 ? off >> 16 : off & 0xffffu;
    if ((j + 1) * NW <= HI || w + NW * j < HI) dma16(c.rs[x], (int)off, c.to + x * (kTileKeys * RB) + NW * j * 1024, j == 0);
  };
  // A tile some of whose keys not all rows see: values that are not finite must be kept from
  // those rows (P = 0 times them is NaN).
  const KeySpan s0 = key_span(have - ql, have, p.win_left, p.win_right);
  const KeySpan s1 = key_span(have - 1, have, p.win_left, p.win_right);
  auto cut = [&](int k0) { return s1.lo > k0 || s0.hi < imin(k0 + BN, kend) - 1; };
  // (A wave's part of the tile holds pieces of all waves' keys: it may be changed only when every wave has read its own
  // keys for S, so the values are noted by key first, and taken out behind the barrier that all waves meet at then.)
  auto piece = [&](int buf, int x, int j) { return reinterpret_cast<u32x4*>(lds + buf * TILE + x * (kTileKeys * RB) + j * 1024 + lane * 16); };
  auto note = [&](int k0, int buf) {  // -> whether this wave's part of a tile that is cut has such values
    if (!cut(k0)) return 0;
    if (lane < 2) wild[w][lane] = 0;
    bool found = false;
    for (int x = 0; x < 2; ++x)
      for (int j = w; j < HI; j += NW) {
        const u32x4 v = *piece(buf, x, j);
        if (odd_halves(v[0]) | odd_halves(v[1]) | odd_halves(v[2]) | odd_halves(v[3])) {
          found = true;
          atomicOr(&wild[w][x], 1u << ((j * 64 + lane) / CH));
        }
      }
    return __any(found);
  };
  auto take_out = [&](int buf) {
    for (int x = 0; x < 2; ++x)
      for (int j = w; j < HI; j += NW) {
        u32x4 v = *piece(buf, x, j);
#pragma unroll
        for (int y = 0; y < 4; ++y) v[y] &= ~(odd_halves(v[y]) * 0xffffu);
        *piece(buf, x, j) = v;
      }
  };
  // LDS offsets: S's A operand (key 16 kg + r, chunk 4 s + g) for even and odd s, and O's (transposing reads:
  // keys 8 g + [0, 4) and + [4, 8) of 32, elements of block t)
  // (blocks VP apart have the same offset in the chunks that the XOR takes together)
  constexpr int VP = CH % 16 == 8 ? 4 : 2, VN = DTW % VP ? DTW : VP;
  int ka[2];
  uint32_t va[VN] = {};  // (both in one register)
  {
    const int row = 16 * w + r;
#pragma unroll
    for (int x = 0; x < 2; ++x) ka[x] = row * RB + ((4 * x + g) ^ latent_swz<CH>(row)) * 16;
#pragma unroll
    for (int t = 0; t < VN; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int vr = 8 * g + (r >> 2) + 4 * x, c = 2 * (w * DTW + t) + ((r & 3) >> 1);
        va[t] |= (uint32_t)(vr * RB + ((c ^ latent_swz<CH>(vr)) * 16) + (r & 1) * 8) << (16 * x);
      }
  }
  {
    const Copy c = copy_plan(0, 0);
#pragma unroll
    for (int j = 0; j < 2 * J; ++j) copy_one(c, j);
  }
  // Q by way of the second tile's place: whole rows from memory once a workgroup (each wave on its own took four
  // times as long), chunk c of row r where a key's would be.  Rows that are not there repeat the last one:
  // their results are not written.
  u32x4 qf[NB][KS];
  {
    constexpr int PER = 256 / X::ROWS, N = (CH + PER - 1) / PER;  // threads per row, chunks per thread
    const int lr = tid / PER, row = imin(row0 + lr, RT - 1), h = row / p.Sq, i = row - h * p.Sq;
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + u.b * a.qsb + h * a.qsh + i * a.qst;
    const uint16_t* qr = static_cast<const uint16_t*>(a.qr) + u.b * a.rsb + h * a.rsh + i * a.rst;
    u32x4 x[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = imin(tid % PER + PER * k, CH - 1);
      x[k] = *reinterpret_cast<const u32x4*>(c < L / 8 ? q + 8 * c : qr + 8 * c - L);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = tid % PER + PER * k;
      if (CH % PER == 0 || c < CH) *reinterpret_cast<u32x4*>(lds + TILE + lr * RB + ((c ^ latent_swz<CH>(lr)) * 16)) = x[k];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        qf[n][s] = *reinterpret_cast<const u32x4*>(lds + TILE + (16 * n + r) * RB + (((4 * s + g) ^ latent_swz<CH>(r)) * 16));
  }

  auto p_at = [&](int row, int c) { return row * 128 + ((c ^ ((row >> 1) & 7)) * 16); };

  f32x4 acc[DTW][NB];
  float m[NB], l[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -INFINITY;
#pragma unroll
    for (int t = 0; t < DTW; ++t) acc[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) l[n] = 0.f;

  for (int i = 0; i < steps; ++i) {
    const int buf = i & 1, k0 = kfirst + BN * i;
    const char* tile = lds + buf * TILE;
    wait_vmem();
    __syncthreads();  // the tile is whole, and everyone has left the other one
    const bool more = i + 1 < steps;
    Copy next;
    if (more) next = copy_plan(i + 1, buf ^ 1);
    f32x4 s[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    // (an XOR of at most 3 bits stays in its 8 chunks, of 2 bits in its 4)
    auto key_frag = [&](int x) {
      return CH % 16 == 8 ? *reinterpret_cast<const u32x4*>(tile + ka[x & 1] + (x >> 1) * 128)
                          : *reinterpret_cast<const u32x4*>(tile + ka[0] + x * 64);
    };
    {
      u32x4 kf[AHEAD + 1];
#pragma unroll
      for (int x = 0; x < imin(AHEAD, KS); ++x) kf[x] = key_frag(x);
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        if (x + AHEAD < KS) kf[(x + AHEAD) % (AHEAD + 1)] = key_frag(x + AHEAD);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          if constexpr (NB >= 2) {
            if (x < 64 / NB) mma_q<'a'>(s[n], kf[x % (AHEAD + 1)], qf[n][x]);  // (256 AGPRs)
            else mma_q<'v'>(s[n], kf[x % (AHEAD + 1)], qf[n][x]);
          } else {
            s[n] = mma16(kf[x % (AHEAD + 1)], qf[n][x], s[n]);
          }
        }
        if (more) {
#pragma unroll
          for (int j = 0; j < JS; ++j)
            if (j * KS / JS == x) copy_one(next, j);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (NB == 2) mma_q_drain(s[0], s[1]);
    if constexpr (NB == 3) mma_q_drain(s[0], s[1], s[2]);
    if constexpr (NB == 4) mma_q_drain(s[0], s[1], s[2], s[3]);
    // lane: keys k0 + 16 w + 4 g + 0 .. 3
    const bool whole = k0 + BN <= kend && s1.lo <= k0 && s0.hi >= k0 + BN - 1;  // every row sees every key
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        bool live;
        KeySpan see = row_span(n, &live);
        see.hi = imin(see.hi, kend - 1);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int k = k0 + 16 * w + 4 * g + y;
          s[n][y] = k >= see.lo && k <= see.hi ? s[n][y] : -INFINITY;
        }
      }
    }
    // P against the maxima so far; only where a wave finds a score past them by more than kLazy do the waves meet to
    // settle new ones and do it again
    float rs[NB];
    auto weights = [&]() {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const float ref = m[n] == -INFINITY ? 0.f : m[n];
        float x[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] = fast_exp2(fmaf(s[n][y], p.scale_log2, -ref));
        rs[n] = (x[0] + x[1]) + (x[2] + x[3]);
        *reinterpret_cast<u32x2*>(pbuf + p_at(16 * n + r, 2 * w + (g >> 1)) + (g & 1) * 8) =
            u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
      }
    };
    weights();
    float top[NB];
    bool higher = false;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      top[n] = fmaxf(fmaxf(s[n][0], s[n][1]), fmaxf(s[n][2], s[n][3])) * p.scale_log2;
      higher = higher || top[n] > m[n] + kLazy;
    }
    const int any = (__any(higher) ? kHigher : 0) | (note(k0, buf) ? kWild : 0);
    if (lane == 0) over[w] = any;
    __syncthreads();  // every wave's scores are made: nobody reads the tile's keys for S any more
    const i32x4 ov = *reinterpret_cast<const i32x4*>(over);
    const int todo = __builtin_amdgcn_readfirstlane(ov[0] | ov[1] | ov[2] | ov[3]);  // (the same in every wave)
    if (todo & kWild) {
      take_out(buf);
      __syncthreads();
    }
    if (todo & kHigher) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        top[n] = quad_max(top[n]);
        if (g == 0) red[16 * n + r][w] = top[n];
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(red[16 * n + r]);
        const float mnew = fmaxf(m[n], fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        const float alpha = m[n] == -INFINITY ? 0.f : fast_exp2(m[n] - mnew);
        m[n] = mnew;
#pragma unroll
        for (int t = 0; t < DTW; ++t)
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[t][n][y] *= alpha;
        l[n] *= alpha;
      }
      weights();
      __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) l[n] += rs[n];
    {
      // units (kk, t): 32 keys by 16 elements
      u32x4 pf[NB], vf[AHEAD + 1];
      auto val_frag = [&](int x) {
        const int t = x % DTW, at = (x / DTW) * (32 * RB) + (t / VN) * (32 * VN);
        uint32_t off = va[t % VN];
        if constexpr (NB >= 3) asm volatile("" : "+v"(off));
        const uint2 lo = lds_read_tr16(tile + (off & 0xffffu) + at), hi = lds_read_tr16(tile + (off >> 16) + at);
        return u32x4{lo.x, lo.y, hi.x, hi.y};
      };
#pragma unroll
      for (int n = 0; n < NB; ++n) pf[n] = *reinterpret_cast<const u32x4*>(pbuf + p_at(16 * n + r, g));
#pragma unroll
      for (int x = 0; x < imin(AHEAD, 2 * DTW); ++x) vf[x] = val_frag(x);
#pragma unroll
      for (int x = 0; x < 2 * DTW; ++x) {
        if (x + AHEAD < 2 * DTW) vf[(x + AHEAD) % (AHEAD + 1)] = val_frag(x + AHEAD);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          acc[x % DTW][n] = mma16(vf[x % (AHEAD + 1)], pf[n], acc[x % DTW][n]);
          if (x == DTW - 1) pf[n] = *reinterpret_cast<const u32x4*>(pbuf + p_at(16 * n + r, 4 + g));
        }
        if (JS < 2 * J && more) {
#pragma unroll
          for (int j = JS; j < 2 * J; ++j)
            if ((j - JS) * 2 * DTW / (2 * J - JS) == x) copy_one(next, j);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (todo & kWild) {
      // A value that is not finite makes NaN of that element in the rows that see its key (the score that it gave, before
      // it was taken out, is not finite either: nothing else can come out).  From the cache: nothing has to be kept for it.
      for (int x = 0; x < 2; ++x) {
        uint32_t keys = 0u;
        for (int y = 0; y < NW; ++y) keys |= wild[y][x];
        for (keys = __builtin_amdgcn_readfirstlane(keys); keys; keys &= keys - 1) {
          int col = 16 * w * DTW + 4 * g;
          asm volatile("" : "+v"(col));  // (as in row_span)
          const int k = k0 + 32 * x + __builtin_ctz(keys), run = k / kTileKeys, pg = run / p.page_runs;
          const int page = p.page_table ? scalar_load(p.page_table + (size_t)u.b * p.max_pages, pg) : u.b;
          const uint16_t* c = a.cache + (((size_t)page * p.page_runs + (run - pg * p.page_runs)) * kTileKeys + k % kTileKeys) * X::W;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            bool live;
            const KeySpan sp = row_span(n, &live);
            const bool sees = k >= sp.lo && k <= sp.hi;
#pragma unroll
            for (int t = 0; t < DTW; ++t) {
              const u32x2 v = *reinterpret_cast<const u32x2*>(c + col + 16 * t);
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint32_t z = v[y >> 1];
                const bool odd = ((z >> (16 * (y & 1))) & 0x7f80u) == 0x7f80u;
                acc[t][n][y] = sees && odd ? __builtin_nanf("") : acc[t][n][y];
              }
            }
          }
        }
      }
    }
  }

#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const float x = quad_sum(l[n]);
    if (g == 0) red[16 * n + r][w] = x;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    bool live;
    row_span(n, &live);
    const f32x4 sums = *reinterpret_cast<const f32x4*>(red[16 * n + r]);
    const float lt = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const int row = row0 + 16 * n + r;
    if (row >= RT) continue;
    if (u.slot < 0) {
      const size_t at = (size_t)u.b * RT + row;
      const bool none = !live || lt == 0.f;  // (NaN is passed on)
      const float inv = none ? 0.f : 1.0f / lt;
#pragma unroll
      for (int t = 0; t < DTW; ++t) {
        const u32x2 x{pack_bf16x2(acc[t][n][0] * inv, acc[t][n][1] * inv), pack_bf16x2(acc[t][n][2] * inv, acc[t][n][3] * inv)};
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.o) + at * L + 16 * (w * DTW + t) + 4 * g) = none ? u32x2{0u, 0u} : x;
      }
      if (w == 0 && g == 0) p.lse[at] = none ? -INFINITY : (m[n] + log2f(lt)) * kLn2;
    } else {
      const size_t at = (size_t)u.slot * ROWS + 16 * n + r;
#pragma unroll
      for (int t = 0; t < DTW; ++t) *reinterpret_cast<f32x4*>(p.part + at * L + 16 * (w * DTW + t) + 4 * g) = acc[t][n];
      if (w == 0 && g == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = live ? make_float2(m[n], lt) : make_float2(-INFINITY, 0.f);
    }
  }
}

// Items that several workgroups shared: M = max m, L = sum l 2^(m - M), O = sum O 2^(m - M) / L.  A wave per output
// row and 64 C of its elements, of which lane s of 64 holds piece s's factor; kWaves waves take every kWaves-th piece
// of the same elements where few rows would leave one wave's loads one behind another.
template <int L, int kWaves>
__global__ __launch_bounds__(256) void latent_merge(DecodeArgs a, int rt, int rows_per) {
  constexpr int C = L >= 256 ? 4 : 2, DEEP = 8, PARTS = L / (64 * C);
  typedef float vec __attribute__((ext_vector_type(C)));
  const int lane = threadIdx.x & 63, w4 = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), w = kWaves == 1 ? 0 : w4;
  const int RT = a.g * a.Sq;
  const long long unit = kWaves == 1 ? (long long)blockIdx.x * 4 + w4 : blockIdx.x;
  const long long orow = unit / PARTS;
  if (orow >= (long long)a.B * RT) return;
  const int b = (int)(orow / RT), row = (int)(orow - (long long)b * RT);
  const int qb = row / rows_per, in = row - qb * rows_per;
  const int pn = a.head[2 * b + 2] - a.head[2 * b];
  if (pn == 1) return;  // one workgroup had it all
  const int slot = a.head[2 * b + 1];
  const int col = (int)(unit - orow * PARTS) * (64 * C) + C * lane;
  auto at = [&](int p) { return ((size_t)(slot + p) * rt + qb) * rows_per + in; };
  float M = -INFINITY, S = 0.f;
  vec acc = 0.f;
  for (int p0 = 0; p0 < pn; p0 += 64) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (p0 + lane < pn) ml = *reinterpret_cast<const float2*>(a.part_ml + at(p0 + lane) * 2);
    const int np = min(64, pn - p0);
    vec y[DEEP];
    auto load = [&](int i0) {
#pragma unroll
      for (int i = 0; i < DEEP; ++i) y[i] = *reinterpret_cast<const vec*>(a.part + at(p0 + min(i0 + kWaves * i, np - 1)) * L + col);
    };
    load(w);  // ahead of the factors
    float mx = ml.x;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    const float mnew = fmaxf(M, mx), ref = mnew == -INFINITY ? 0.f : mnew;
    const float old = fast_exp2(M - ref), c = fast_exp2(ml.x - ref);
    float ls = ml.y * c;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) ls += __shfl_xor(ls, d);
    S = S * old + ls;
    M = mnew;
    acc *= old;
    for (int i0 = w; i0 < np; i0 += kWaves * DEEP) {
      if (i0 != w) load(i0);
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        const float ci = __shfl(c, (i0 + kWaves * i) & 63);
        const bool there = i0 + kWaves * i < np && !(ci == 0.f);
#pragma unroll
        for (int k = 0; k < C; ++k) acc[k] = there ? fmaf(y[i][k], ci, acc[k]) : acc[k];
      }
    }
  }
  if constexpr (kWaves > 1) {
    __shared__ vec sum[kWaves][64];
    sum[w][lane] = acc;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) acc += sum[i][lane];
  }
  const float inv = S == 0.f ? 0.f : 1.0f / S;
  uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + (size_t)orow * L + col);
#pragma unroll
  for (int k = 0; k < C; k += 2) o[k / 2] = S == 0.f ? 0u : pack_bf16x2(acc[k] * inv, acc[k + 1] * inv);
  if (lane == 0 && col == 0) a.lse[orow] = S == 0.f ? -INFINITY : (M + log2f(S)) * kLn2;
}

}  // namespace fa
