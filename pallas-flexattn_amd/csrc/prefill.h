// Attention of chunks of new tokens over a paged KV cache (bf16, or e4m3 with a
// power-of-two scale per 32 tokens and head), for gfx950.
//
//   o = softmax(mask(mod(scale q k^T))) v,   query i of a row at position keys - queries + i
//
// Bound by the matrix cores from about a hundred rows per kv head on (4 D operations per row
// and key against 4 D or 2 D bytes per key), so it is built around them: a workgroup takes
// 128 rows, 32 a wave, whose Q stays in registers, and walks the keys in tiles of 64, two tiles of K and V in
// LDS (two workgroups per compute unit at D = 128).
//   * S^T = K Q^T (v_mfma_f32_32x32x16_bf16; A = K rows in perm23 order, B = Q): a lane
//     holds scores of one row, so the softmax's state is a scalar per lane;
//   * one pass: exponentials against the reference maximum so far; a wave whose sum over a
//     tile leaves [0, 2^16] (or that has seen no key) takes the tile's maximum and rescales. What
//     reference is used does not change O / l;
//   * O^T += V^T P^T, V^T by transposing LDS reads, P straight from S's registers, rounded to bf16 there
//     (2^-9 relative, as V and O are; l sums the unrounded values).
// A wave brings 16 of a tile's 64 keys, which lie in one run of 32 tokens and so in one page of any
// size: bf16 by LDS DMA, out-of-range rows as zeros; 8-bit codes through registers, converted once per
// workgroup (bf16 holds code x scale exactly) and written to the same layout: the products do not
// know which cache they read.
#pragma once
#include "decode_fp8.h"
#include "dma.h"
#include "fwd.h"
#include "prefill_plan.h"

namespace fa {

// An item's rows [row0, row0 + kPrefillRows) of `rows` = g nq: queries i >= ql see nothing.
struct PrefillItem {
  int b, row0, nq, ql, have, tok;  // tok: the row's first token (packed)
};
template <bool kPacked>
__device__ __forceinline__ PrefillItem prefill_item(const PrefillArgs& a, int rest) {
  PrefillItem it;
  it.tok = 0;
  if constexpr (!kPacked) {  // the last tiles of all rows first: the longest walks
    it.b = rest % a.B;
    it.row0 = (row_tiles(a.Sq, a.g) - 1 - rest / a.B) * kPrefillRows;
    it.nq = a.Sq;
    it.ql = a.q_lens ? clamp_len(scalar_load(a.q_lens, it.b), a.Sq) : a.Sq;
  } else {
    const int lane = threadIdx.x & 63;
    int before = 0;
    it.b = -1;
    for (int b0 = 0; b0 < a.B + 2; b0 += 64) {
      const int b = b0 + lane;
      TokenSpan t{0, 0};
      if (b < a.B + 2) t = packed_span(a.starts, b, a.B, a.Sq);
      const int n = row_tiles(t.e - t.s, a.g);
      const int end = before + wave_scan(n);
      const unsigned long long mine = __ballot(rest >= end - n && rest < end);
      if (mine) {
        const int src = __builtin_ctzll(mine);
        it.b = b0 + src;
        it.tok = __builtin_amdgcn_readlane(t.s, src);
        it.nq = __builtin_amdgcn_readlane(t.e, src) - it.tok;
        it.row0 = (__builtin_amdgcn_readlane(end, src) - 1 - rest) * kPrefillRows;
        break;
      }
      before = __builtin_amdgcn_readlane(end, 63);
    }
    if (it.b < 0) return it;
    it.ql = it.b < a.B ? it.nq : 0;
  }
  it.have = it.b >= a.B ? 0 : a.kv_lens ? clamp_len(scalar_load(a.kv_lens, it.b), a.cap) : a.cap;
  return it;
}

// tanh of a lane's 16 values (tanh8's choice of form)
__device__ __forceinline__ void tanh16(f32x16& x) {
  float lo = INFINITY, hi = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float t = fabsf(x[e]);
    lo = fminf(lo, t);
    hi = fmaxf(hi, t);
  }
  if (!__any(hi >= kTanhSmall)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = tanh_small(x[e]);
  } else if (!__any(lo < kTanhSmall)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = tanh_large(x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float v = x[e];
      x[e] = fabsf(v) < kTanhSmall ? tanh_small(v) : tanh_large(v);
    }
  }
}

// bf16 pairs: bits 15 and 31 set where the half is an infinity or a NaN
__device__ __forceinline__ uint32_t wild_halves(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

template <int D, bool kFp8, bool kMods, bool kPacked>
__global__ __launch_bounds__(256, 2) void prefill_kernel(PrefillArgs a) {
  using E = Elt<uint16_t>;
  using frag = E::frag;
  constexpr int BN = kPrefillKeys, NW = 4;
  constexpr int RB = 2 * D, KCH = D / 8, KSTEPS = D / 16, NSUB = BN / 32, DT = D / 32, NC = BN / 16;
  constexpr int TILE = BN * RB;
  constexpr int IPW = TILE / 1024 / NW;      // LDS DMA instructions per wave and tensor
  constexpr int WR = BN / NW;                // keys that a wave brings
  constexpr int CL = D >= 64 ? D / 64 : 1;   // 16-byte loads of codes per wave and tensor
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];  // K_0, K_1, V_0, V_1
  __shared__ int wild[2][NW];                // a tile holds values that are not finite (where that matters)

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, hh = lane >> 5;
  const int items = a.tiles * a.Hkv;
  const int split = a.n_splits > 1 ? (int)blockIdx.x / items : 0;
  const int item = (int)blockIdx.x - split * items;
  // (kv heads fastest: with eight of them each XCD's L2 holds one head's keys)
  const int rest = item / a.Hkv, hk = item - rest * a.Hkv;
  const PrefillItem it = prefill_item<kPacked>(a, rest);
  if (kPacked && it.b < 0) return;
  const int have = it.have, rows = it.nq * a.g;
  const int i_first = it.row0 / a.g, i_last = imin((it.row0 + kPrefillRows - 1) / a.g, it.ql - 1);
  TileSpan ts = tile_span(have, it.ql, i_first, i_last, a.win_left, a.win_right);
  if (a.n_splits > 1) {
    const SplitRange sr = split_range(ts.t1 - ts.t0, split, a.n_splits, 0);
    ts = TileSpan{ts.t0 + sr.it0, ts.t0 + sr.it1};
  }

  // this lane's row
  const int r = it.row0 + 32 * w + lr;
  const bool valid = r < rows;
  const int qi = (valid ? r : rows - 1) / a.g, hq = (valid ? r : rows - 1) - qi * a.g;
  const int h = hk * a.g + hq;
  const bool live = valid && qi < it.ql;
  const int qpos = have - it.ql + qi;
  KeySpan see = key_span(qpos, have, a.win_left, a.win_right);
  if (!live) see = KeySpan{0, 0x7fffffff};  // (its results are not written: nothing to mask)
  const bool wave_live = __any(live);
  const float slope = kMods && a.alibi ? a.alibi[h] : 0.f;

  frag qf[KSTEPS];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (kPacked ? 0 : it.b) * a.qsb + h * a.qsh + (long long)(it.tok + qi) * a.qst;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) qf[s] = ld16(qp + (2 * s + hh) * 8, live);
  }

  // Where a tile's keys lie: lane i holds, of tile base + i, the run of this wave's 16 keys (-1: none, or a bad page; keys of a
  // run that are past the row's end read as zeros) and its scales.
  int tab_base = ts.t0 - 64, run_l = -1;
  float ks_l = 1.f, vs_l = 1.f;
  auto table = [&](int t0) {
    tab_base = t0;
    run_l = -1;
    ks_l = vs_l = 1.f;
    const long long key = (long long)(t0 + lane) * BN + WR * w;
    if (t0 + lane < ts.t1 && key < have) {
      const int run = (int)(key / kTileKeys), pg = run / a.page_runs;
      const int page = pg >= a.max_pages ? -1 : a.page_table ? a.page_table[(size_t)it.b * a.max_pages + pg] : it.b;
      if (page >= 0 && page < a.num_pages) {
        run_l = (page * a.Hkv + hk) * a.page_runs + (run - pg * a.page_runs);
        if constexpr (kFp8) {
          ks_l = a.ks[run_l];
          vs_l = a.vs[run_l];
        }
      }
    }
  };
  // Byte offset of this wave's 16 keys of tile t (rows of `row` bytes) and how many bytes of them are there.
  struct Place {
    size_t at;
    uint32_t bytes;
    float ksc, vsc;
  };
  auto place = [&](int t, int row) {
    if (t - tab_base >= 64) table(t);
    const int i = t - tab_base;
    const int run = __builtin_amdgcn_readlane(run_l, i);
    Place p;
    p.at = ((size_t)imax(run, 0) * kTileKeys + (WR * w) % kTileKeys) * row;
    p.bytes = run < 0 ? 0u : (uint32_t)imin(WR, have - (t * BN + WR * w)) * row;
    p.ksc = p.vsc = 1.f;
    if constexpr (kFp8) {
      p.ksc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_l), i));
      p.vsc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs_l), i));
    }
    return p;
  };

  // bf16: copies straight to LDS
  [[maybe_unused]] int dma_k[IPW], dma_v[IPW];
  struct Copy {
    i32x4 rk, rv;
    char *kl, *vl;
  };
  [[maybe_unused]] auto copy_plan = [&](int t, int buf) {
    const Place p = place(t, RB);
    return Copy{make_rsrc(a.k + p.at, p.bytes), make_rsrc(a.v + p.at, p.bytes), lds + buf * TILE + w * (IPW * 1024),
                lds + (2 + buf) * TILE + w * (IPW * 1024)};
  };
  [[maybe_unused]] auto copy_one = [&](const Copy& c, int i) {
    if (i < IPW) dma16(c.rk, dma_k[i], c.kl + i * 1024, i == 0);
    else dma16(c.rv, dma_v[i - IPW], c.vl + (i - IPW) * 1024, i == IPW);
  };
  // e4m3: codes in registers, sixteen of a row per load
  [[maybe_unused]] u32x4 kc[CL], vc[CL];
  [[maybe_unused]] float ksc = 1.f, vsc = 1.f;
  constexpr int PR = D / 16;  // loads per row
  [[maybe_unused]] auto codes_load = [&](int t) {
    const Place p = place(t, D);
    const i32x4 rk = make_rsrc(a.k + p.at, p.bytes), rv = make_rsrc(a.v + p.at, p.bytes);
    ksc = p.ksc;
    vsc = p.vsc;
#pragma unroll
    for (int u = 0; u < CL; ++u) {
      kc[u] = buf_load16(rk, (u * 64 + lane) * 16);
      vc[u] = buf_load16(rv, (u * 64 + lane) * 16);
    }
  };
  [[maybe_unused]] auto codes_store = [&](int buf) {
#pragma unroll
    for (int u = 0; u < CL; ++u) {
      const int c = u * 64 + lane, row = WR * w + c / PR, ch = 2 * (c % PR);
      if (D < 64 && lane >= 32) break;  // (D = 32: the 16 rows take 32 loads)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t k0 = kc[u][2 * x], k1 = kc[u][2 * x + 1], v0 = vc[u][2 * x], v1 = vc[u][2 * x + 1];
        *reinterpret_cast<u32x4*>(lds + buf * TILE + row * RB + (((ch + x) ^ chunk_swz<KCH>(row)) * 16)) =
            u32x4{cvt_e4m3_lo(k0, ksc), cvt_e4m3_hi(k0, ksc), cvt_e4m3_lo(k1, ksc), cvt_e4m3_hi(k1, ksc)};
        *reinterpret_cast<u32x4*>(lds + (2 + buf) * TILE + row * RB + (((ch + x) ^ tr_swz<KCH>(row)) * 16)) =
            u32x4{cvt_e4m3_lo(v0, vsc), cvt_e4m3_hi(v0, vsc), cvt_e4m3_lo(v1, vsc), cvt_e4m3_hi(v1, vsc)};
      }
    }
  };
  if constexpr (!kFp8) {
#pragma unroll
    for (int u = 0; u < IPW; ++u) {
      dma_k[u] = tile_dma_offset<D, BN, NW>(lane, w, u) - WR * w * RB;
      dma_v[u] = tile_dma_offset<D, BN, NW, true>(lane, w, u) - WR * w * RB;
    }
  }
  // Keys that all of the item's rows see: a tile with others among its keys has to keep a value that is not finite
  // from the rows that do not see it (P = 0 times it is NaN).
  const KeySpan s0 = key_span(have - it.ql + i_first, have, a.win_left, a.win_right);
  const KeySpan s1 = key_span(have - it.ql + i_last, have, a.win_left, a.win_right);
  auto cut = [&](int t) { return s1.lo > t * BN || s0.hi < imin(t * BN + BN, have) - 1; };
  // (after this wave's part of tile t has come, before the barrier that hands it to the others: they are taken
  // out of the tile here, and noted by key)
  auto look = [&](int t, int buf) {
    if (!cut(t)) return;
    if (lane == 0) wild[buf][w] = 0;
#pragma unroll
    for (int u = 0; u < IPW; ++u) {
      u32x4* at = reinterpret_cast<u32x4*>(lds + (2 + buf) * TILE + (w * IPW + u) * 1024 + lane * 16);
      u32x4 x = *at;
      uint32_t bad = 0u;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t odd = wild_halves(x[y]) >> 15;  // bits 0 and 16
        bad |= odd;
        x[y] &= ~(odd * 0xffffu);
      }
      if (bad) {
        *at = x;
        atomicOr(&wild[buf][w], 1 << ((u * 64 + lane) / KCH));
      }
    }
  };

  RowTileOffsets<D> kt;
  kt.init(lane);
  int voff[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) voff[i] = fwd_voff_t<D>(lane, i);

  f32x16 oacc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[i][e] = 0.f;
#pragma unroll
  for (int i = 0; i < DT; ++i) mfma_drain<'v'>(oacc[i]);
  // Adds what look() took out of a key's value to the rows that see the key: infinities, and NaN.  (From the
  // cache, so that nothing has to be kept for it.)
  auto patch = [&](int key) {
    const int run = key / kTileKeys, pg = run / a.page_runs;  // (of a page that is there: its values were read)
    const int page = a.page_table ? scalar_load(a.page_table + (size_t)it.b * a.max_pages, pg) : it.b;
    const size_t row = ((size_t)(page * a.Hkv + hk) * a.page_runs + (run - pg * a.page_runs)) * kTileKeys + key % kTileKeys;
    const bool sees = key >= see.lo && key <= see.hi;
#pragma unroll
    for (int i = 0; i < DT; ++i) mfma_drain<'v'>(oacc[i]);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const size_t at = row * D + 32 * i + 8 * j + 4 * hh;
        float x[4];
        if constexpr (kFp8) {
          const uint32_t y = nan_codes(*reinterpret_cast<const uint32_t*>(a.v + at));
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = (y >> (8 * e + 7)) & 1u ? __builtin_nanf("") : 0.f;
        } else {
          const u32x2 y = *reinterpret_cast<const u32x2*>(a.v + 2 * at);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t z = y[e >> 1];
            const float v = e & 1 ? bf16_hi(z) : bf16_lo(z);
            x[e] = fabsf(v) < INFINITY ? 0.f : v;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) oacc[i][4 * j + e] += sees ? x[e] : 0.f;
      }
#pragma unroll
    for (int i = 0; i < DT; ++i) mfma_drain<'v'>(oacc[i]);
  };

  constexpr float kSpill = 65536.0f;
  float m = -INFINITY, l = 0.f;
  const float sl2 = kMods ? 1.0f : a.scale_log2;  // (with modifiers the scores are in log2 units already)
  const float mod_in = a.softcap > 0.f ? 1.0f / a.softcap : 1.0f;
  const float mod_out = (a.softcap > 0.f ? a.softcap : 1.0f) * kLog2e;
  auto exps = [&](const f32x16* s, frag* pf, float ref) {
    float r0 = 0.f, r1 = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float x[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) x[t] = fast_exp2(fmaf(s[c >> 1][8 * (c & 1) + t], sl2, -ref));
      pf[c] = E::pack(x);
#pragma unroll
      for (int t = 0; t < 8; t += 2) {
        r0 += x[t];
        r1 += x[t + 1];
      }
    }
    return r0 + r1;
  };
  auto softmax = [&](const f32x16* s, frag* pf) {
    float rs = exps(s, pf, m == -INFINITY ? 0.f : m);
    if (__any(!(rs <= kSpill) || m == -INFINITY)) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < NSUB; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[j][e]);
      const float mnew = fmaxf(m, pair_max(mx) * sl2);
      if (__any(mnew > m)) {
        const float alpha = fast_exp2(m - (mnew == -INFINITY ? 0.f : mnew));
        l *= alpha;
#pragma unroll
        for (int i = 0; i < DT; ++i) mfma_drain<'v'>(oacc[i]);
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) oacc[i][e] *= alpha;
#pragma unroll
        for (int i = 0; i < DT; ++i) mfma_drain<'v'>(oacc[i]);
        m = mnew;
      }
      rs = exps(s, pf, m == -INFINITY ? 0.f : m);
    }
    l += rs;
  };

  if (ts.t0 < ts.t1) {
    if constexpr (kFp8) {
      codes_load(ts.t0);
      codes_store(0);
    } else {
      const Copy c = copy_plan(ts.t0, 0);
#pragma unroll
      for (int i = 0; i < 2 * IPW; ++i) copy_one(c, i);
    }
  }
  wait_vmem();
  if (ts.t0 < ts.t1) look(ts.t0, 0);
  __syncthreads();

  auto step = [&](int t, auto buf_c) {
    constexpr int buf = decltype(buf_c)::value;
    const int kbase = t * BN;
    const bool more = t + 1 < ts.t1;
    [[maybe_unused]] Copy nc;
    if (more) {
      if constexpr (kFp8) codes_load(t + 1);
      else nc = copy_plan(t + 1, buf ^ 1);
    }
    // a tile that no row of this wave sees only passes by
    const bool run = wave_live && __any(live && see.lo < kbase + BN && see.hi >= kbase);
    if (!kFp8 && !run && more) {
#pragma unroll
      for (int i = 0; i < 2 * IPW; ++i) copy_one(nc, i);
    }
    if (run) {  // wave-uniform
      const char* kl = lds + buf * TILE;
      const char* vl = lds + (2 + buf) * TILE;
      f32x16 s[NSUB];
#pragma unroll
      for (int j = 0; j < NSUB; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[j][e] = 0.f;
      constexpr int KPF = 2, KR = KPF + 1;  // K fragments ahead of their products
      frag ka[KR][NSUB];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int x = 0; x < KPF; ++x)
#pragma unroll
        for (int j = 0; j < NSUB; ++j) ka[x][j] = *reinterpret_cast<const u32x4*>(kl + j * 32 * RB + kt.aoff[x]);
#pragma unroll
      for (int x = 0; x < KSTEPS; ++x) {
        if (x + KPF < KSTEPS) {
#pragma unroll
          for (int j = 0; j < NSUB; ++j) ka[(x + KPF) % KR][j] = *reinterpret_cast<const u32x4*>(kl + j * 32 * RB + kt.aoff[x + KPF]);
        }
#pragma unroll
        for (int j = 0; j < NSUB; ++j) s[j] = E::mma(ka[x % KR][j], qf[x], s[j]);
        if constexpr (!kFp8) {  // this step's share of the next tile's copies
#pragma unroll
          for (int i = 0; i < 2 * IPW; ++i)
            if (i * KSTEPS / (2 * IPW) == x && more) copy_one(nc, i);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      if constexpr (kMods) {
#pragma unroll
        for (int j = 0; j < NSUB; ++j) {
          const float first = (float)(kbase + 32 * j + 8 * hh - qpos);
#pragma unroll
          for (int e = 0; e < 16; ++e) s[j][e] = fmaf(slope, first + (float)acc_row(e, 0), s[j][e] * a.scale) * mod_in;
          if (a.softcap > 0.f) tanh16(s[j]);
#pragma unroll
          for (int e = 0; e < 16; ++e) s[j][e] *= mod_out;
        }
      }
      const bool whole = __all(see.lo <= kbase && see.hi >= kbase + BN - 1);
      if (!whole) {
#pragma unroll
        for (int j = 0; j < NSUB; ++j) {
          const int base = kbase + 32 * j + 8 * hh;
          const uint32_t bits = interval_bits(see.lo - base, see.hi - base);
#pragma unroll
          for (int e = 0; e < 16; ++e) s[j][e] = keep_bit(s[j][e], bits, acc_row(e, 0), -INFINITY);
        }
      }
      frag vt[2][NC];
      auto load_vt = [&](int i) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint2 lo = lds_read_tr16(vl + voff[i] + (16 * c) * RB);
          const uint2 hi = lds_read_tr16(vl + voff[i] + (16 * c + 4) * RB);
          vt[i & 1][c] = u32x4{lo.x, lo.y, hi.x, hi.y};
        }
      };
      load_vt(0);
      frag pf[NC];
      softmax(s, pf);
      // the 2 wait states that an MFMA needs after a VALU write of its operand, once for all of P
      static_assert(NC == 4, "P fragments");
      asm volatile("s_nop 1" : "+v"(pf[0]), "+v"(pf[1]), "+v"(pf[2]), "+v"(pf[3]));
      __builtin_amdgcn_s_setprio(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        if (i + 1 < DT) load_vt(i + 1);
#pragma unroll
        for (int c = 0; c < NC; ++c) mfma_acc<'v', false>(oacc[i], vt[i & 1][c], pf[c]);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      if (cut(t)) {
        for (int x = 0; x < NW; ++x) {
          for (int keys = __builtin_amdgcn_readfirstlane(wild[buf][x]); keys; keys &= keys - 1) patch(kbase + WR * x + __builtin_ctz(keys));
        }
      }
    }
    if constexpr (kFp8) {
      if (more) codes_store(buf ^ 1);
    } else {
      wait_vmem();
    }
    if (more) look(t + 1, buf ^ 1);
    __syncthreads();
  };
  int t = ts.t0;
  for (; t + 1 < ts.t1; t += 2) {
    step(t, Int<0>{});
    step(t + 1, Int<1>{});
  }
  if (t < ts.t1) step(t, Int<0>{});

#pragma unroll
  for (int i = 0; i < DT; ++i) mfma_drain<'v'>(oacc[i]);
  const float lt = pair_sum(l);
  // row of lse (and of the partial results)
  const size_t at = ((size_t)(kPacked ? 0 : it.b) * a.Hq + h) * a.Sq + it.tok + qi;
  if (a.n_splits > 1) {
    const size_t all = (size_t)(kPacked ? 1 : a.B) * a.Hq * a.Sq;
    if (valid) {
      float* po = a.part + ((size_t)split * all + at) * D;
      if (ts.t0 < ts.t1 && live) {  // (else m = -inf says that there is no O)
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<f32x4*>(po + 32 * i + 8 * j + 4 * hh) =
                f32x4{oacc[i][4 * j], oacc[i][4 * j + 1], oacc[i][4 * j + 2], oacc[i][4 * j + 3]};
      }
      if (hh == 0)
        *reinterpret_cast<float2*>(a.part + (size_t)a.n_splits * all * D + ((size_t)split * all + at) * 2) =
            live ? make_float2(m, lt) : make_float2(-INFINITY, 0.f);
    }
    return;
  }
  // O through the wave's part of the (now idle) tiles, so that a store writes whole row segments
  const bool none = !live || lt == 0.f;  // (NaN is passed on)
  const float inv = none ? 0.f : 1.0f / lt;
  constexpr int RPI = 64 / KCH;
  char* stage = lds + w * (32 * RB);
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 4 * i + j;
      const u32x2 x{pack_bf16x2(oacc[i][4 * j] * inv, oacc[i][4 * j + 1] * inv),
                    pack_bf16x2(oacc[i][4 * j + 2] * inv, oacc[i][4 * j + 3] * inv)};
      *reinterpret_cast<u32x2*>(stage + lr * RB + ((c ^ (lr % KCH)) * 16) + hh * 8) = none ? u32x2{0u, 0u} : x;
    }
  const int c = lane % KCH;
#pragma unroll
  for (int k = 0; k < 32 / RPI; ++k) {
    const int rr = k * RPI + lane / KCH, row = it.row0 + 32 * w + rr;
    const u32x4 x = *reinterpret_cast<const u32x4*>(stage + rr * RB + ((c ^ (rr % KCH)) * 16));
    if (row < rows) {
      const int i = row / a.g, hr = row - i * a.g;
      uint16_t* o = static_cast<uint16_t*>(a.o) + (kPacked ? 0 : it.b) * a.osb + (hk * a.g + hr) * a.osh + (long long)(it.tok + i) * a.ost;
      *reinterpret_cast<u32x4*>(o + c * 8) = x;
    }
  }
  if (valid && hh == 0) a.lse[at] = none ? -INFINITY : (m + log2f(lt)) * kLn2;
}

// The splits of a row: M = max m_s, L = sum l_s 2^(m_s - M), O = sum O_s 2^(m_s - M) / L.  A wave per row;
// lane s of 64 holds split s's factor, the columns go over the lanes.
template <int D>
__global__ __launch_bounds__(256) void prefill_merge(PrefillArgs a, long long rows) {
  constexpr int CPL = D >= 64 ? D / 64 : 1, DEEP = 8;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const long long row = (long long)blockIdx.x * 4 + w;
  if (row >= rows) return;
  const int n = a.n_splits;
  const float* ml = a.part + (size_t)n * rows * D;
  const int col = lane * CPL < D ? lane * CPL : 0;
  float2 x = make_float2(-INFINITY, 0.f);
  if (lane < n) x = *reinterpret_cast<const float2*>(ml + ((size_t)lane * rows + row) * 2);
  float M = x.x;
#pragma unroll
  for (int d = kPrefillSplits / 2; d >= 1; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
  M = __shfl(M, 0);
  const float c = x.x == -INFINITY ? 0.f : fast_exp2(x.x - M);
  float L = x.y * c;
#pragma unroll
  for (int d = kPrefillSplits / 2; d >= 1; d >>= 1) L += __shfl_xor(L, d);
  L = __shfl(L, 0);
  float acc[CPL];
#pragma unroll
  for (int k = 0; k < CPL; ++k) acc[k] = 0.f;
  for (int s0 = 0; s0 < n; s0 += DEEP) {
    float y[DEEP][CPL];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      const float* p = a.part + ((size_t)imin(s0 + u, n - 1) * rows + row) * D + col;
#pragma unroll
      for (int k = 0; k < CPL; ++k) y[u][k] = p[k];
    }
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      const float cs = __shfl(c, (s0 + u) & 63);
      const bool there = s0 + u < n && !(cs == 0.f);  // (a split without a visible key has no O; NaN is passed on)
#pragma unroll
      for (int k = 0; k < CPL; ++k) acc[k] = there ? fmaf(y[u][k], cs, acc[k]) : acc[k];
    }
  }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  if (lane * CPL < D) {
    const long long tok = row % a.Sq, bh = row / a.Sq;
    uint16_t* o = static_cast<uint16_t*>(a.o) + (bh / a.Hq) * a.osb + (bh % a.Hq) * a.osh + tok * a.ost + col;
    if constexpr (CPL == 2) *reinterpret_cast<uint32_t*>(o) = L == 0.f ? 0u : pack_bf16x2(acc[0] * inv, acc[CPL - 1] * inv);
    else *o = L == 0.f ? (uint16_t)0 : (uint16_t)(pack_bf16x2(acc[0] * inv, 0.f) & 0xffffu);
  }
  if (lane == 0) a.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

}  // namespace fa
