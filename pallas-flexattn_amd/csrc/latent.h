// Latent attention over a paged cache, absorbed form, for gfx950: all heads read one vector c of L
// elements a token, key and value at once, and a rotary part r of R elements that is key only.
//
//   s = scale (q . c + q_r . r),   o = softmax(mask(s)) c      (per head; o has L elements)
//
// (a key W_k c and a value W_v c of a head, with W_k taken into the query and W_v into what follows.)
// A key costs 2 (L + R) bytes and 2 H (2 L + R) operations a query: 16 heads are bound by the
// reads, 128 heads by both. So every key is read from memory once for up to 64 rows (heads x
// queries), and the 64 keys of a tile serve both products from LDS:
//   * S^T = K Q^T (v_mfma_f32_16x16x32_bf16): a wave takes 16 keys of the tile and up to 32 rows, whose
//     Q stays in registers (4 registers per 32 of L + R and 16 rows);
//   * the waves' maxima of a row meet in LDS, then their P (bf16, 2^-9 relative as c is; sums take the
//     unrounded values);
//   * O^T += C^T P^T: a wave takes L / waves of the elements of all rows, so that each value of the
//     tile is read from LDS once for all rows, by transposing reads; O stays in registers.
// Tiles come by LDS DMA, one ahead, two in LDS (147 KB of 160 for L + R = 576: one workgroup per compute unit).
// Chunk c (16 bytes) of key row r sits at chunk c ^ f(r), with f such that 16 rows of one chunk, and
// the 8 rows by 2 chunks of half a transposing read, lie in different banks.
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

// NB: 16-row blocks of an item (1, 2: four waves; 4: eight)
template <int L, int R, int NB>
struct LatentShape {
  static constexpr int NW = NB == 4 ? 8 : 4;
  static constexpr int W = L + R, RB = 2 * W, CH = W / 8, KS = W / 32;
  static constexpr int TILE = kLatentKeys * RB, ROWS = 16 * NB;
  static constexpr int HI = CH / 2;                // copies of 1 KB per run
  static constexpr int J = (HI + NW - 1) / NW;     // of them a wave's
  static constexpr int DTW = L / 16 / NW;          // 16-element blocks of O a wave has
  static constexpr int NBW = NB / (NW / 4);        // 16-row blocks of S a wave has
  static constexpr int LDS = 2 * TILE + ROWS * 128 + 16 * ROWS + 64;
  static_assert(L % (16 * NW) == 0 && W % 32 == 0 && LDS <= 160 * 1024, "shape");
};

template <int L, int R, int NB>
__global__ __launch_bounds__(64 * (NB == 4 ? 8 : 4)) __attribute__((amdgpu_waves_per_eu(
    occupancy_for(LatentShape<L, R, NB>::LDS, LatentShape<L, R, NB>::NW, 2))))
void latent_decode_kernel(LatentArgs a) {
  using X = LatentShape<L, R, NB>;
  constexpr int NW = X::NW, RB = X::RB, CH = X::CH, KS = X::KS, TILE = X::TILE, ROWS = X::ROWS, HI = X::HI, J = X::J;
  constexpr int DTW = X::DTW, NBW = X::NBW, BN = kLatentKeys;
  constexpr float kLazy = 8.0f;  // a maximum may be this stale (log2): P stays under 2^8
  __shared__ __attribute__((aligned(1024))) char lds[2 * TILE];
  __shared__ __attribute__((aligned(16))) char pbuf[ROWS * 128];
  __shared__ float red[4][ROWS];
  __shared__ uint32_t wild[NW][2];  // keys of the tile with values that are not finite, as each wave found them

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int kg = w & 3, rg = w >> 2;  // this wave's keys and rows of S
  const DecodeArgs& p = a.d;
  const DecodeUnit u = decode_unit(p, blockIdx.x, w == 0);
  if (u.b < 0) return;
  const int have = u.have, ql = u.ql, RT = p.g * p.Sq;
  const int row0 = u.item * ROWS;
  const int kfirst = u.t0 * kTileKeys;
  const int kend = imin(have, (u.t0 + u.nt) * kTileKeys);  // this piece's keys: [kfirst, kend)
  const int steps = (u.nt + 1) / 2;

  // rows as lse has them: a head's queries one after another
  auto row_span = [&](int n, bool* live) {
    const int row = row0 + 16 * n + r, i = imin(row, RT - 1) % p.Sq;
    *live = row < RT && i < ql;
    KeySpan k = key_span(have - ql + i, have, p.win_left, p.win_right);
    return *live ? k : KeySpan{0, 0x7fffffff};  // (the results of others are not written)
  };

  u32x4 qf[NBW][KS];
  KeySpan see[NBW];
#pragma unroll
  for (int n = 0; n < NBW; ++n) {
    const int row = row0 + 16 * (NBW * rg + n) + r;
    bool live;
    see[n] = row_span(NBW * rg + n, &live);
    const int h = imin(row, RT - 1) / p.Sq, i = imin(row, RT - 1) - h * p.Sq;
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + u.b * a.qsb + h * a.qsh + i * a.qst;
    const uint16_t* qr = static_cast<const uint16_t*>(a.qr) + u.b * a.rsb + h * a.rsh + i * a.rst;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[n][s] = ld16(32 * s < L ? q + 32 * s + 8 * g : qr + 32 * s - L + 8 * g, live);
  }

  // copies: lane offsets in a run, the same for both runs of a tile
  int dma[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (w + NW * j) * 64 + lane, row = c / CH;
    dma[j] = row * RB + (((c - row * CH) ^ latent_swz<CH>(row)) * 16);
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
  auto copy = [&](int i, int buf) {
    const int t = u.t0 + 2 * i;
    if (t - tab >= 64) table(t);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int run = __builtin_amdgcn_readlane(run_l, t + x - tab);  // (t and tab differ by an even number under 64)
      const uint32_t bytes = run < 0 ? 0u : (uint32_t)imax(imin(kTileKeys, kend - (t + x) * kTileKeys), 0) * RB;
      const i32x4 rs = make_rsrc(a.cache + (size_t)imax(run, 0) * (kTileKeys * X::W), bytes);
#pragma unroll
      for (int j = 0; j < J; ++j)
        if ((j + 1) * NW <= HI || w + NW * j < HI)
          dma16(rs, dma[j], lds + buf * TILE + x * (kTileKeys * RB) + (w + NW * j) * 1024, j == 0);
    }
  };
  // A tile some of whose keys not all rows see: values that are not finite must be kept from
  // those rows (P = 0 times them is NaN).
  const KeySpan s0 = key_span(have - ql, have, p.win_left, p.win_right);
  const KeySpan s1 = key_span(have - 1, have, p.win_left, p.win_right);
  auto cut = [&](int k0) { return s1.lo > k0 || s0.hi < imin(k0 + BN, kend) - 1; };
  auto look = [&](int k0, int buf) {  // between the products: taken out of this wave's part of the tile, and noted by key
    if (!cut(k0)) return;
    if (lane < 2) wild[w][lane] = 0;
    for (int x = 0; x < 2; ++x)
      for (int j = w; j < HI; j += NW) {
        u32x4* at = reinterpret_cast<u32x4*>(lds + buf * TILE + x * (kTileKeys * RB) + j * 1024 + lane * 16);
        u32x4 v = *at;
        uint32_t bad = 0u;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t odd = (((v[y] & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15;  // bits 0 and 16
          bad |= odd;
          v[y] &= ~(odd * 0xffffu);
        }
        if (bad) {
          *at = v;
          atomicOr(&wild[w][x], 1u << ((j * 64 + lane) / CH));
        }
      }
  };
  // LDS offsets: S's A operand (key 16 kg + r, chunk 4 s + g) for even and odd s, and O's (transposing reads:
  // keys 8 g + [0, 4) and + [4, 8) of 32, elements of block t)
  int ka[2], va[DTW][2];
  {
    const int row = 16 * kg + r;
#pragma unroll
    for (int x = 0; x < 2; ++x) ka[x] = row * RB + ((4 * x + g) ^ latent_swz<CH>(row)) * 16;
#pragma unroll
    for (int t = 0; t < DTW; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int vr = 8 * g + (r >> 2) + 4 * x, c = 2 * (w * DTW + t) + ((r & 3) >> 1);
        va[t][x] = vr * RB + ((c ^ latent_swz<CH>(vr)) * 16) + (r & 1) * 8;
      }
  }
  auto p_at = [&](int row, int c) { return row * 128 + ((c ^ ((row >> 1) & 7)) * 16); };

  f32x4 acc[DTW][NB];
  float m[NB], l[NBW];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -INFINITY;
#pragma unroll
    for (int t = 0; t < DTW; ++t) acc[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int n = 0; n < NBW; ++n) l[n] = 0.f;

  copy(0, 0);
  for (int i = 0; i < steps; ++i) {
    const int buf = i & 1, k0 = kfirst + BN * i;
    const char* tile = lds + buf * TILE;
    wait_vmem();
    __syncthreads();  // the tile is whole, and everyone has left the other one
    if (i + 1 < steps) copy(i + 1, buf ^ 1);
    f32x4 s[NBW];
#pragma unroll
    for (int n = 0; n < NBW; ++n) s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      // (an XOR of at most 3 bits stays in its 8 chunks, of 2 bits in its 4)
      const u32x4 kf = CH % 16 == 8 ? *reinterpret_cast<const u32x4*>(tile + ka[x & 1] + (x >> 1) * 128)
                                    : *reinterpret_cast<const u32x4*>(tile + ka[0] + x * 64);
#pragma unroll
      for (int n = 0; n < NBW; ++n) s[n] = mma16(kf, qf[n][x], s[n]);
    }
    const int key = k0 + 16 * kg;  // lane: keys key + 4 g + 0 .. 3
#pragma unroll
    for (int n = 0; n < NBW; ++n) {
      const int hi = imin(see[n].hi, kend - 1);
      float mx = -INFINITY;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int k = key + 4 * g + y;
        s[n][y] = k >= see[n].lo && k <= hi ? s[n][y] * p.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[n][y]);
      }
      mx = quad_max(mx);
      if (g == 0) red[kg][16 * (NBW * rg + n) + r] = mx;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float mx = fmaxf(fmaxf(red[0][16 * n + r], red[1][16 * n + r]), fmaxf(red[2][16 * n + r], red[3][16 * n + r]));
      if (__any(mx > m[n] + kLazy)) {  // (the same in every wave)
        const float mnew = fmaxf(m[n], mx);
        const float alpha = m[n] == -INFINITY ? 0.f : fast_exp2(m[n] - mnew);
        m[n] = mnew;
#pragma unroll
        for (int t = 0; t < DTW; ++t)
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[t][n][y] *= alpha;
#pragma unroll
        for (int k = 0; k < NBW; ++k)
          if (NBW * rg + k == n) l[k] *= alpha;
      }
    }
#pragma unroll
    for (int n = 0; n < NBW; ++n) {
      float ref = m[n];
      if constexpr (NB > NBW) ref = rg ? m[NB - NBW + n] : m[n];
      if (ref == -INFINITY) ref = 0.f;
      float x[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) x[y] = fast_exp2(s[n][y] - ref);
      l[n] += (x[0] + x[1]) + (x[2] + x[3]);
      *reinterpret_cast<u32x2*>(pbuf + p_at(16 * (NBW * rg + n) + r, 2 * kg + (g >> 1)) + (g & 1) * 8) =
          u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
    }
    look(k0, buf);
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      u32x4 pf[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) pf[n] = *reinterpret_cast<const u32x4*>(pbuf + p_at(16 * n + r, 4 * kk + g));
#pragma unroll
      for (int t = 0; t < DTW; ++t) {
        const uint2 lo = lds_read_tr16(tile + va[t][0] + kk * (32 * RB)), hi = lds_read_tr16(tile + va[t][1] + kk * (32 * RB));
        const u32x4 vf{lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[t][n] = mma16(vf, pf[n], acc[t][n]);
      }
    }
    if (cut(k0)) {
      // A value that is not finite makes NaN of that element in the rows that see its key (the score that it gave
      // is not finite either: nothing else can come out).  From the cache: nothing has to be kept for it.
      for (int x = 0; x < 2; ++x) {
        uint32_t keys = 0u;
        for (int y = 0; y < NW; ++y) keys |= wild[y][x];
        for (keys = __builtin_amdgcn_readfirstlane(keys); keys; keys &= keys - 1) {
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
              const u32x2 v = *reinterpret_cast<const u32x2*>(c + 16 * (w * DTW + t) + 4 * g);
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
  for (int n = 0; n < NBW; ++n) {
    const float x = quad_sum(l[n]);
    if (g == 0) red[kg][16 * (NBW * rg + n) + r] = x;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    bool live;
    row_span(n, &live);
    const float lt = (red[0][16 * n + r] + red[1][16 * n + r]) + (red[2][16 * n + r] + red[3][16 * n + r]);
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
// row and 128 of its elements; lane s of 64 holds piece s's factor.
template <int L>
__global__ __launch_bounds__(256) void latent_merge(DecodeArgs a, int rows_per) {
  constexpr int DEEP = 8, PARTS = L / 128;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int RT = a.g * a.Sq;
  const long long unit = (long long)blockIdx.x * 4 + w;
  const long long orow = unit / PARTS;
  if (orow >= (long long)a.B * RT) return;
  const int b = (int)(orow / RT), row = (int)(orow - (long long)b * RT);
  const int qb = row / rows_per, in = row - qb * rows_per;
  const int pn = (a.head[2 * b + 2] - a.head[2 * b]) / a.rt;
  if (pn == 1) return;  // one workgroup had it all
  const int slot = a.head[2 * b + 1] + qb * pn;
  const int col = (int)(unit - orow * PARTS) * 128 + 2 * lane;
  auto at = [&](int p) { return (size_t)(slot + p) * rows_per + in; };
  float M = -INFINITY, S = 0.f, x0 = 0.f, x1 = 0.f;
  for (int p0 = 0; p0 < pn; p0 += 64) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (p0 + lane < pn) ml = *reinterpret_cast<const float2*>(a.part_ml + at(p0 + lane) * 2);
    const int np = min(64, pn - p0);
    float2 y[DEEP];
    auto load = [&](int i0) {
#pragma unroll
      for (int i = 0; i < DEEP; ++i) y[i] = *reinterpret_cast<const float2*>(a.part + at(p0 + min(i0 + i, np - 1)) * L + col);
    };
    load(0);  // ahead of the factors
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
    x0 *= old;
    x1 *= old;
    for (int i0 = 0; i0 < np; i0 += DEEP) {
      if (i0) load(i0);
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        const float ci = __shfl(c, (i0 + i) & 63);
        const bool there = i0 + i < np && !(ci == 0.f);
        x0 = there ? fmaf(y[i].x, ci, x0) : x0;
        x1 = there ? fmaf(y[i].y, ci, x1) : x1;
      }
    }
  }
  const float inv = S == 0.f ? 0.f : 1.0f / S;
  *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + (size_t)orow * L + col) = S == 0.f ? 0u : pack_bf16x2(x0 * inv, x1 * inv);
  if (lane == 0 && col == 0) a.lse[orow] = S == 0.f ? -INFINITY : (M + log2f(S)) * kLn2;
}

}  // namespace fa
