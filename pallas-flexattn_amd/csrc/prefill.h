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
//     (half a step, 2^-8, as for V and O; l sums the unrounded values).
// A wave brings 16 of a tile's 64 keys, which lie in one run of 32 tokens and so in one page of any
// size: bf16 by LDS DMA, out-of-range rows as zeros; 8-bit codes through registers, converted once per
// workgroup (bf16 holds code x scale exactly) and written to the same layout: the products do not
// know which cache they read.
// Measured, 32 heads on 8 of D = 128: 4096 queries behind 28672 keys 1.90 ms, 1080 TFLOP/s, the matrix cores busy half
// the cycles (a library product of 8192^3 1300); 1024 behind 16384 e4m3 keys 285 us and 11 for the join of two ranges, 960: converting, once
// per 128 rows, takes a fifth more VALU instructions and 8 stores to LDS a wave and tile (LDS cycles per product twice those of bf16).  16 heads
// of D = 64, 8 ragged rows, window of 1500, ALiBi and soft-cap: 90 us and 12 for the join; its VALU instructions (39 per MFMA) are
// 36 us of them, the matrix cores' 7: the units idle where a row is shorter than the padded tokens, of whose items half are taken to be
// there and each is cut into as many ranges.
#pragma once
#include "decode_fp8.h"
#include "dma.h"
#include "fwd.h"
#include "prefill_plan.h"

namespace fa {

// inclusive maximum over the lanes of a wave, of numbers that are not negative (as wave_scan)
__device__ __forceinline__ int wave_max_scan(int x) {
  x = imax(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = imax(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = imax(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = imax(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = imax(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  x = imax(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return x;
}

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
    int before = 0, highest = 0;
    it.b = -1;
    for (int b0 = 0; b0 < a.B + 2; b0 += 64) {
      const int b = b0 + lane;
      TokenSpan t = packed_span(a.starts, imin(b, a.B + 1), a.B, a.Sq);
      if (b > a.B + 1) t = TokenSpan{0, 0};
      const int high = imax(wave_max_scan(b <= a.B ? t.s : 0), highest);
      highest = __builtin_amdgcn_readlane(high, 63);
      if (b <= a.B) t = span_behind(t, high);
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

// tanh of a lane's 16 values, in the form that the wave's values allow (tanh8): here also a shorter polynomial below kTanhTiny
// (minimax in x^2 too, within 1.7 2^-24 of the value), where a soft-cap well above the scores leaves them.
constexpr float kTanhTiny = 0.35f;
__device__ __forceinline__ float tanh_tiny(float x) {
  const float y = x * x;
  float p = fmaf(-0.04914850369095802f, y, 0.1329982578754425f);
  p = fmaf(p, y, -0.33332663774490356f);
  return fmaf(x * y, p, x);
}
__device__ __forceinline__ void tanh16(f32x16& x) {
  float hi = 0.f;
#pragma unroll
  for (int e = 0; e < 16; e += 2) hi = fmaxf(fmaxf(hi, fabsf(x[e])), fabsf(x[e + 1]));
  if (!__any(hi >= kTanhTiny)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = tanh_tiny(x[e]);
    return;
  }
  float lo = INFINITY;
#pragma unroll
  for (int e = 0; e < 16; e += 2) lo = fminf(fminf(lo, fabsf(x[e])), fabsf(x[e + 1]));
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

// The rows of a wave, one per lane (the two lane halves hold one row's other elements): Q, the running softmax and O.
template <int D, bool kFp8, bool kMods, bool kPacked>
struct PrefillWave {
  using E = Elt<uint16_t>;
  using frag = E::frag;
  static constexpr int RB = 2 * D, KCH = D / 8, KSTEPS = D / 16, DT = D / 32;
  static constexpr float kSpill = 65536.0f;
  frag qf[KSTEPS];
  f32x16 oacc[DT];
  float m, l;
  KeySpan see;  // keys that the row sees ([0, 2^31 - 1]: a row that is not there, whose results are not written)
  int qpos;
  float mod_scale, mod_slope, sl2;  // scores in log2 units are sl2 times what the products hold (modified: see below)
  int koff[KSTEPS], voff[DT];       // LDS offsets in tiles of keys (K's rows lane % 32 in perm23 order; V's transposing reads)

  struct Row {
    int qi, hq;
    bool valid, live;
  };
  // (Computed again where the walk is over: kept, it would cost the walk registers, and a spilled one is read back only
  // behind all copies under way.)
  __device__ __forceinline__ static Row row(const PrefillArgs& a, const PrefillItem& it, int r) {
    asm volatile("" : "+v"(r));
    const int rows = it.nq * a.g;
    Row x;
    x.valid = r < rows;
    const int c = x.valid ? r : rows - 1;
    x.qi = c / a.g;
    x.hq = c - x.qi * a.g;
    x.live = x.valid && x.qi < it.ql;
    return x;
  }

  // r: the lane's row of the item's batch row and kv head hk
  __device__ __forceinline__ void init(const PrefillArgs& a, const PrefillItem& it, int hk, int r, int lane) {
    const Row x = row(a, it, r);
    const int hh = lane >> 5;
    qpos = it.have - it.ql + x.qi;
    see = key_span(qpos, it.have, a.win_left, a.win_right);
    if (!x.live) see = KeySpan{0, 0x7fffffff};
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (kPacked ? 0 : it.b) * a.qsb + (hk * a.g + x.hq) * a.qsh +
                         (long long)(it.tok + x.qi) * a.qst + 8 * hh;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qp + 16 * s);
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) qf[s] = x.live ? qf[s] : u32x4{0u, 0u, 0u, 0u};  // (padded tokens may be anything)
    const float slope = kMods && a.alibi ? a.alibi[hk * a.g + x.hq] : 0.f;
    const float mod_in = a.softcap > 0.f ? 1.0f / a.softcap : 1.0f;
    mod_scale = a.scale * mod_in;
    mod_slope = slope * mod_in;
    sl2 = kMods ? (a.softcap > 0.f ? a.softcap : 1.0f) * kLog2e : a.scale_log2;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) oacc[i][e] = 0.f;
    drain();
    RowTileOffsets<D> kt;
    kt.init(lane);
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) koff[s] = kt.aoff[s];
#pragma unroll
    for (int i = 0; i < DT; ++i) voff[i] = fwd_voff_t<D>(lane, i);
  }
  __device__ __forceinline__ void drain() {
#pragma unroll
    for (int i = 0; i < DT; ++i) mfma_drain<'v'>(oacc[i]);
  }

  // With modifiers: (scale q k + slope (key - position)) mod_in, of which a soft-cap's tanh; mod_out is taken with the exponent
  template <int NSUB>
  __device__ __forceinline__ void modify(const PrefillArgs& a, f32x16* s, int kbase, int hh) const {
#pragma unroll
    for (int j = 0; j < NSUB; ++j) {
      const float first = mod_slope * (float)(kbase + 32 * j + 8 * hh - qpos);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[j][e] = fmaf(s[j][e], mod_scale, fmaf(mod_slope, (float)acc_row(e, 0), first));
      if (a.softcap > 0.f) tanh16(s[j]);
    }
  }
  template <int NSUB>
  __device__ __forceinline__ void mask(f32x16* s, int kbase, int hh) const {
    if (__all(see.lo <= kbase && see.hi >= kbase + 32 * NSUB - 1)) return;
#pragma unroll
    for (int j = 0; j < NSUB; ++j) {
      const int base = kbase + 32 * j + 8 * hh;
      const uint32_t bits = interval_bits(see.lo - base, see.hi - base);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[j][e] = keep_bit(s[j][e], bits, acc_row(e, 0), -INFINITY);
    }
  }
  template <int NSUB>
  __device__ __forceinline__ float exps(const f32x16* s, frag* pf, float ref) const {
    float r0 = 0.f, r1 = 0.f;
#pragma unroll
    for (int c = 0; c < 2 * NSUB; ++c) {
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
  }
  template <int NSUB>
  __device__ __forceinline__ void softmax(const f32x16* s, frag* pf) {
    float rs = exps<NSUB>(s, pf, m == -INFINITY ? 0.f : m);
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
        drain();
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) oacc[i][e] *= alpha;
        drain();
        m = mnew;
      }
      rs = exps<NSUB>(s, pf, m == -INFINITY ? 0.f : m);
    }
    l += rs;
  }
  // Gives the rows that see the keys (of the 16 from k0 on, as bits) the infinities and NaN that were taken out of their
  // values, read from the cache again so that nothing has to be kept for it: products of the largest finite numbers where they
  // were with 2^16 for each row and visible key overflow to infinity, of both signs to NaN, and leave the other
  // rows as they are.  (As products because any other change of O made the compiler copy it for every tile.)
  __device__ __forceinline__ void patch(const PrefillArgs& a, int b, int hk, int k0, int keys, int lane) {
    const int run = k0 / kTileKeys, pg = run / a.page_runs;  // (of a page that is there: its values were read)
    const int page = a.page_table ? scalar_load(a.page_table + (size_t)b * a.max_pages, pg) : b;
    const int at_run = (page * a.Hkv + hk) * a.page_runs + (run - pg * a.page_runs);
    const size_t row = (size_t)at_run * kTileKeys + k0 % kTileKeys;
    [[maybe_unused]] const float vsc = kFp8 ? __uint_as_float(scalar_load(reinterpret_cast<const int*>(a.vs), at_run)) : 1.f;
    asm volatile("" : "+v"(lane));  // (addresses not kept for the whole walk)
    const int first = 8 * (lane >> 5);
    frag seen;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int key = k0 + first + 2 * y;
      seen[y] = (key >= see.lo && key <= see.hi ? 0x4780u : 0u) | (key + 1 >= see.lo && key + 1 <= see.hi ? 0x47800000u : 0u);
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      frag up = E::zero(), down = E::zero();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool here = (keys >> (first + e)) & 1;  // (a key past the row's end is in the page all the same)
        const size_t at = (row + first + e) * D + 32 * i + (lane & 31);
        uint32_t v;  // as the tile had it, in the upper half: a code is infinite, too, where its scale takes it past bf16
        if constexpr (kFp8) v = cvt_e4m3_lo((uint32_t) static_cast<uint8_t>(a.v[at]) << 8, vsc);
        else v = (uint32_t) * reinterpret_cast<const uint16_t*>(a.v + 2 * at) << 16;
        const bool plus = __builtin_amdgcn_classf(__uint_as_float(v), 0x203), minus = __builtin_amdgcn_classf(__uint_as_float(v), 0x007);
        up[e >> 1] |= (here && plus ? 0x7f7fu : 0u) << (16 * (e & 1));
        down[e >> 1] |= (here && minus ? 0xff7fu : 0u) << (16 * (e & 1));
      }
      mfma_acc<'v', true>(oacc[i], up, seen);
      mfma_acc<'v', true>(oacc[i], down, seen);
    }
  }
};
// Takes infinities and NaN out of 1 KB of a V tile in LDS; returns whether this lane's 16 bytes had any.
__device__ __forceinline__ bool tame(char* at) {
  u32x4 x = *reinterpret_cast<u32x4*>(at);
  uint32_t bad = 0u;
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const uint32_t odd = wild_halves(x[y]) >> 15;  // bits 0 and 16
    bad |= odd;
    x[y] &= ~(odd * 0xffffu);
  }
  if (bad) *reinterpret_cast<u32x4*>(at) = x;
  return bad != 0u;
}

// What a split leaves of a row for the join: m = -inf, nothing (a NaN sum has seen something, whatever the maximum says).
__device__ __forceinline__ float2 split_ml(float m, float l, bool live) {
  return !live ? make_float2(-INFINITY, 0.f) : l == l ? make_float2(m, l) : make_float2(0.f, l);
}

// Row `row` of all `rows` in the join's list of maxima and sums, for the range that x is.  (An item with fewer ranges than others
// says so: one range, whose results are written already, by a negative sum; else by an empty range at the end.)
__device__ __forceinline__ void note_ml(const PrefillArgs& a, const PrefillRange& x, int D, size_t rows, size_t row, float2 ml) {
  if (a.n_splits == 1) return;
  float2* list = reinterpret_cast<float2*>(a.part + (size_t)a.n_splits * rows * D) + row;
  list[x.split * rows] = x.ranges > 1 ? ml : make_float2(0.f, -1.f);
  if (x.split == 0 && x.ranges > 1 && x.ranges < a.n_splits) list[x.ranges * rows] = make_float2(-INFINITY, 0.f);
}

// Where keys lie: lane i holds, for the keys first + step i .. of a batch row, their run (-1: none, or a bad page) and its scales.
template <bool kFp8>
struct RunTable {
  int run = -1;
  float ks = 1.f, vs = 1.f;
  __device__ __forceinline__ void load(const PrefillArgs& a, int b, int hk, int have, long long key, long long end) {
    run = -1;
    ks = vs = 1.f;
    if (key < end && key < have) {
      const int r = (int)(key / kTileKeys), pg = r / a.page_runs;
      const int page = pg >= a.max_pages ? -1 : a.page_table ? a.page_table[(size_t)b * a.max_pages + pg] : b;
      if (page >= 0 && page < a.num_pages) {
        run = (page * a.Hkv + hk) * a.page_runs + (r - pg * a.page_runs);
        if constexpr (kFp8) {
          ks = a.ks[run];
          vs = a.vs[run];
        }
      }
    }
  }
  __device__ __forceinline__ static float lane(float x, int i) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), i));
  }
};

// Items of at most 32 rows (the single tokens of a mixed batch, short chunks): bound by the reads of the cache, so each wave walks
// every fourth 32-key tile by itself, in a quarter of the LDS, without barriers; the waves join at the end.
template <int D, bool kFp8, bool kMods, bool kPacked>
__device__ __forceinline__ void prefill_thin(const PrefillArgs& a, const PrefillItem& it, int hk, const PrefillRange& x0, TileSpan ts, char* lds) {
  using W = PrefillWave<D, kFp8, kMods, kPacked>;
  using frag = typename W::frag;
  constexpr int RB = W::RB, KCH = W::KCH, DT = W::DT, KSTEPS = W::KSTEPS, TB = 32 * RB;
  constexpr int IPT = TB / 1024;               // LDS DMA instructions per tile and tensor
  constexpr int CL = D / 32, PR = D / 16;      // 16-byte loads of codes per lane and tensor, and per row
  __shared__ float2 tml[4][32];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, hh = lane >> 5;
  const int have = it.have;
  char* kl = lds + w * (2 * TB);
  char* vl = kl + TB;
  W x;
  x.init(a, it, hk, it.row0 + lr, lane);
  // this wave's tiles: t0 + w, + 4, ..
  const int t0 = 2 * ts.t0, t1 = imin(2 * ts.t1, (have + 31) / 32);
  const int n = t1 > t0 + w ? (t1 - t0 - w + 3) / 4 : 0;
  RunTable<kFp8> tab;
  int base = -64;
  auto find = [&](int i) {  // -> lane of tile i
    if (i - base >= 64) {
      base = i;
      tab.load(a, it.b, hk, have, (long long)(t0 + w + 4 * (i + lane)) * 32, (long long)t1 * 32);
    }
    return i - base;
  };
  auto rsrc = [&](const char* p, int i, int row_bytes) {
    const int at = find(i), run = __builtin_amdgcn_readlane(tab.run, at);
    const uint32_t bytes = run < 0 ? 0u : (uint32_t)imin(32, have - (t0 + w + 4 * i) * 32) * row_bytes;
    return make_rsrc(p + (size_t)imax(run, 0) * kTileKeys * row_bytes, bytes);
  };
  [[maybe_unused]] uint32_t dma[IPT];
  [[maybe_unused]] u32x4 kc[CL], vc[CL];
  [[maybe_unused]] float ksc = 1.f, vsc = 1.f;
  auto load_k = [&](int i) {
    const i32x4 rs = rsrc(a.k, i, kFp8 ? D : RB);
    if constexpr (kFp8) {
      ksc = RunTable<kFp8>::lane(tab.ks, i - base);
#pragma unroll
      for (int u = 0; u < CL; ++u) kc[u] = buf_load16(rs, (u * 64 + lane) * 16);
    } else {
#pragma unroll
      for (int u = 0; u < IPT; ++u) dma16(rs, (int)(dma[u] & 0xffffu), kl + u * 1024, u == 0);
    }
  };
  auto load_v = [&](int i) {
    const i32x4 rs = rsrc(a.v, i, kFp8 ? D : RB);
    if constexpr (kFp8) {
      vsc = RunTable<kFp8>::lane(tab.vs, i - base);
#pragma unroll
      for (int u = 0; u < CL; ++u) vc[u] = buf_load16(rs, (u * 64 + lane) * 16);
    } else {
#pragma unroll
      for (int u = 0; u < IPT; ++u) dma16(rs, (int)(dma[u] >> 16), vl + u * 1024, u == 0);
    }
  };
  auto store = [&](const u32x4* c, float sc, char* tile, auto val) {  // codes of 16 elements a load, as bf16
#pragma unroll
    for (int u = 0; u < CL; ++u) {
      const int at = u * 64 + lane, row = at / PR, ch = 2 * (at % PR);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t c0 = c[u][2 * y], c1 = c[u][2 * y + 1];
        const int slot = (ch + y) ^ (decltype(val)::value ? tr_swz<KCH>(row) : chunk_swz<KCH>(row));
        *reinterpret_cast<u32x4*>(tile + row * RB + slot * 16) =
            u32x4{cvt_e4m3_lo(c0, sc), cvt_e4m3_hi(c0, sc), cvt_e4m3_lo(c1, sc), cvt_e4m3_hi(c1, sc)};
      }
    }
  };
  if constexpr (!kFp8) {
#pragma unroll
    for (int u = 0; u < IPT; ++u)
      dma[u] = (uint32_t)tile_dma_offset<D, 32, 1>(lane, 0, u) | (uint32_t)tile_dma_offset<D, 32, 1, true>(lane, 0, u) << 16;
  }
  if (n) {
    load_k(0);
    load_v(0);
  }
  for (int i = 0; i < n; ++i) {
    const int kbase = (t0 + w + 4 * i) * 32;
    const bool more = i + 1 < n;
    if constexpr (kFp8) {
      store(kc, ksc, kl, False{});
      if (more) load_k(i + 1);
    } else {
      wait_vmem_but<IPT>();  // (V's copies may still be under way)
    }
    f32x16 s[1];
#pragma unroll
    for (int e = 0; e < 16; ++e) s[0][e] = 0.f;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) s[0] = W::E::mma(*reinterpret_cast<const u32x4*>(kl + x.koff[k]), x.qf[k], s[0]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!kFp8) {
      if (more) load_k(i + 1);  // (K's reads are done: the products have them)
    }
    if constexpr (kMods) x.template modify<1>(a, s, kbase, hh);
    x.template mask<1>(s, kbase, hh);
    frag pf[2];
    x.template softmax<1>(s, pf);
    if constexpr (kFp8) {
      store(vc, vsc, vl, True{});
      if (more) load_v(i + 1);
    } else {
      if (more) wait_vmem_but<IPT>();
      else wait_vmem();
    }
    // values that are not finite, where a row does not see all keys of the tile
    int keys[2] = {0, 0};
    if (!__all(x.see.lo <= kbase && x.see.hi >= imin(kbase + 32, have) - 1)) {
#pragma unroll
      for (int u = 0; u < IPT; ++u) {
        const unsigned long long bad = __ballot(tame(vl + u * 1024 + lane * 16));
        for (unsigned long long z = bad; z; z &= z - 1) {
          const int key = (u * 64 + __builtin_ctzll(z)) / KCH;
          keys[key >> 4] |= 1 << (key & 15);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint2 lo = lds_read_tr16(vl + x.voff[d] + (16 * c) * RB), hi = lds_read_tr16(vl + x.voff[d] + (16 * c + 4) * RB);
        mfma_acc<'v', true>(x.oacc[d], u32x4{lo.x, lo.y, hi.x, hi.y}, pf[c]);
      }
    __builtin_amdgcn_sched_barrier(0);
    if (keys[0]) x.patch(a, it.b, hk, kbase, keys[0], lane);
    if (keys[1]) x.patch(a, it.b, hk, kbase + 16, keys[1], lane);
    if constexpr (!kFp8) {
      if (more) load_v(i + 1);
    }
  }
  x.drain();
  // join: M = max m, L = sum l 2^(m - M), O = sum O 2^(m - M)
  const float lt = pair_sum(x.l);
  if (hh == 0) tml[w][lr] = make_float2(x.m, lt);
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) M = fmaxf(M, tml[i][lr].x);
  const float c = x.m == -INFINITY ? 0.f : fast_exp2(x.m - M);
  constexpr int RC = D / 4;  // 16-byte chunks of a float32 row, swizzled by the row
  char* mine = lds + w * (32 * 4 * D);
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = c == 0.f ? 0.f : x.oacc[i][4 * j + e] * c;
      *reinterpret_cast<f32x4*>(mine + lr * (4 * D) + (((8 * i + 2 * j + hh) ^ (lr & (RC - 1))) * 16)) = y;
    }
  __syncthreads();
  constexpr int CW = D / 8;  // columns of a thread, eight threads a row
  const int orow = tid / 8, col = (tid % 8) * CW;
  float L = 0.f;
  M = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) M = fmaxf(M, tml[i][orow].x);
#pragma unroll
  for (int i = 0; i < 4; ++i) L += tml[i][orow].x == -INFINITY ? tml[i][orow].y : tml[i][orow].y * fast_exp2(tml[i][orow].x - M);
  f32x4 o[CW / 4];
#pragma unroll
  for (int k = 0; k < CW / 4; ++k) {
    const int at = orow * (4 * D) + (((col / 4 + k) ^ (orow & (RC - 1))) * 16);
    const f32x4* p = reinterpret_cast<const f32x4*>(lds + at);
    o[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 y = p[i * (32 * 4 * D) / 16];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[k][e] += y[e];
    }
  }
  const int rows = it.nq * a.g;
  const size_t all = (size_t)(kPacked ? 1 : a.B) * a.Hq * a.Sq;
  const auto me = W::row(a, it, it.row0 + orow);
  if (me.valid) {
    const size_t at = ((size_t)(kPacked ? 0 : it.b) * a.Hq + hk * a.g + me.hq) * a.Sq + it.tok + me.qi;
    if (col == 0) note_ml(a, x0, D, all, at, split_ml(M, L, me.live));
    if (x0.ranges > 1) {
      float* po = a.part + ((size_t)x0.split * all + at) * D + col;
#pragma unroll
      for (int k = 0; k < CW / 4; ++k) *reinterpret_cast<f32x4*>(po + 4 * k) = o[k];
    } else {
      const bool none = !me.live || L == 0.f;  // (NaN is passed on)
      const float inv = none ? 0.f : 1.0f / L;
      uint16_t* po = static_cast<uint16_t*>(a.o) + (kPacked ? 0 : it.b) * a.osb + (hk * a.g + me.hq) * a.osh +
                     (long long)(it.tok + me.qi) * a.ost + col;
#pragma unroll
      for (int k = 0; k < CW / 4; ++k) {
        const u32x2 y{pack_bf16x2(o[k][0] * inv, o[k][1] * inv), pack_bf16x2(o[k][2] * inv, o[k][3] * inv)};
        *reinterpret_cast<u32x2*>(po + 4 * k) = none ? u32x2{0u, 0u} : y;
      }
      if (col == 0) a.lse[at] = none ? -INFINITY : (M + log2f(L)) * kLn2;
    }
  }
  // the item's further rows are padded tokens
  const int left = imin(rows - it.row0, kPrefillRows);
  for (int z = 32 + orow; z < left; z += 32) {
    const auto pad = W::row(a, it, it.row0 + z);
    const size_t at = ((size_t)(kPacked ? 0 : it.b) * a.Hq + hk * a.g + pad.hq) * a.Sq + it.tok + pad.qi;
    if (col == 0) note_ml(a, x0, D, all, at, make_float2(-INFINITY, 0.f));
    if (x0.ranges == 1) {
      uint16_t* po = static_cast<uint16_t*>(a.o) + (kPacked ? 0 : it.b) * a.osb + (hk * a.g + pad.hq) * a.osh +
                     (long long)(it.tok + pad.qi) * a.ost + col;
#pragma unroll
      for (int k = 0; k < CW / 4; ++k) *reinterpret_cast<u32x2*>(po + 4 * k) = u32x2{0u, 0u};
      if (col == 0) a.lse[at] = -INFINITY;
    }
  }
}

template <int D, bool kFp8, bool kMods, bool kPacked>
__global__ __launch_bounds__(256, D == 128 ? 2 : 3) void prefill_kernel(PrefillArgs a) {
  using W = PrefillWave<D, kFp8, kMods, kPacked>;
  using E = typename W::E;
  using frag = typename W::frag;
  constexpr int BN = kPrefillKeys, NW = 4;
  constexpr int RB = W::RB, KCH = W::KCH, KSTEPS = W::KSTEPS, DT = W::DT, NSUB = BN / 32, NC = BN / 16;
  constexpr int TILE = BN * RB;
  constexpr int IPW = TILE / 1024 / NW;      // LDS DMA instructions per wave and tensor
  constexpr int WR = BN / NW;                // keys that a wave brings
  constexpr int CL = D >= 64 ? D / 64 : 1;   // 16-byte loads of codes per wave and tensor
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];  // K_0, K_1, V_0, V_1
  __shared__ int wild[2][NW];                // keys of a tile (of each wave's 16) with values that are not finite, where that matters

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, hh = lane >> 5;
  const PrefillRange range = prefill_range(a, blockIdx.x);
  // (kv heads fastest: with eight of them each XCD's L2 holds one head's keys)
  const int rest = range.item / a.Hkv, hk = range.item - rest * a.Hkv;
  const PrefillItem it = prefill_item<kPacked>(a, rest);
  if (kPacked && it.b < 0) return;
  const int have = it.have, rows = it.nq * a.g;
  const int i_first = it.row0 / a.g, i_last = imin((it.row0 + kPrefillRows - 1) / a.g, it.ql - 1);
  TileSpan ts = tile_span(have, it.ql, i_first, i_last, a.win_left, a.win_right);
  if (range.ranges > 1) {
    const SplitRange sr = split_range(ts.t1 - ts.t0, range.split, range.ranges, 0);
    ts = TileSpan{ts.t0 + sr.it0, ts.t0 + sr.it1};
  }
  if (it.ql * a.g - it.row0 <= 32) {
    prefill_thin<D, kFp8, kMods, kPacked>(a, it, hk, range, ts, lds);
    return;
  }
  W x;
  x.init(a, it, hk, it.row0 + 32 * w + lr, lane);

  // This wave's 16 keys of tile t: their byte offset (rows of `row` bytes) and how many bytes of them are there (the others read as
  // zeros).
  RunTable<kFp8> tab;
  int tab_base = ts.t0 - 64;
  struct Place {
    size_t at;
    uint32_t bytes;
    float ksc, vsc;
  };
  auto place = [&](int t, int row) {
    if (t - tab_base >= 64) {
      tab_base = t;
      tab.load(a, it.b, hk, have, (long long)(t + lane) * BN + WR * w, (long long)ts.t1 * BN);
    }
    const int i = t - tab_base;
    const int run = __builtin_amdgcn_readlane(tab.run, i);
    Place p;
    p.at = ((size_t)imax(run, 0) * kTileKeys + (WR * w) % kTileKeys) * row;
    p.bytes = run < 0 ? 0u : (uint32_t)imin(WR, have - (t * BN + WR * w)) * row;
    p.ksc = p.vsc = 1.f;
    if constexpr (kFp8) {
      p.ksc = RunTable<kFp8>::lane(tab.ks, i);
      p.vsc = RunTable<kFp8>::lane(tab.vs, i);
    }
    return p;
  };

  // bf16: copies straight to LDS
  [[maybe_unused]] uint32_t dma[IPW];  // lane offsets: K's in the lower half, V's in the upper
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
    uint32_t off = dma[i % IPW];
    asm volatile("" : "+v"(off));  // (not unpacked ahead of the loop)
    if (i < IPW) dma16(c.rk, (int)(off & 0xffffu), c.kl + i * 1024, i == 0);
    else dma16(c.rv, (int)(off >> 16), c.vl + (i - IPW) * 1024, i == IPW);
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
  // (in 2 CL parts: load u of K and of V)
  [[maybe_unused]] auto codes_store = [&](int buf, int part) {
    const int u = part >> 1;
    const bool val = part & 1;
    const int c = u * 64 + lane, row = WR * w + c / PR, ch = 2 * (c % PR);
    if (D < 64 && lane >= 32) return;  // (D = 32: the 16 rows take 32 loads)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const uint32_t c0 = val ? vc[u][2 * y] : kc[u][2 * y], c1 = val ? vc[u][2 * y + 1] : kc[u][2 * y + 1];
      const float sc = val ? vsc : ksc;
      const int slot = (ch + y) ^ (val ? tr_swz<KCH>(row) : chunk_swz<KCH>(row));
      *reinterpret_cast<u32x4*>(lds + ((val ? 2 : 0) + buf) * TILE + row * RB + slot * 16) =
          u32x4{cvt_e4m3_lo(c0, sc), cvt_e4m3_hi(c0, sc), cvt_e4m3_lo(c1, sc), cvt_e4m3_hi(c1, sc)};
    }
  };
  if constexpr (!kFp8) {
#pragma unroll
    for (int u = 0; u < IPW; ++u) {
      dma[u] = (uint32_t)(tile_dma_offset<D, BN, NW>(lane, w, u) - WR * w * RB) |
               (uint32_t)(tile_dma_offset<D, BN, NW, true>(lane, w, u) - WR * w * RB) << 16;
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
    int l0 = lane;
    asm volatile("" : "+v"(l0));
#pragma unroll
    for (int u = 0; u < IPW; ++u)
      if (tame(lds + (2 + buf) * TILE + (w * IPW + u) * 1024 + l0 * 16)) atomicOr(&wild[buf][w], 1 << ((u * 64 + l0) / KCH));
  };

  if (ts.t0 < ts.t1) {
    if constexpr (kFp8) {
      codes_load(ts.t0);
#pragma unroll
      for (int i = 0; i < 2 * CL; ++i) codes_store(0, i);
    } else {
      const Copy c = copy_plan(ts.t0, 0);
#pragma unroll
      for (int i = 0; i < 2 * IPW; ++i) copy_one(c, i);
    }
  }
  wait_vmem();
  if (ts.t0 < ts.t1) look(ts.t0, 0);
  __syncthreads();

  // The tiles that some row of this wave sees are [w0, w1): the wave only brings its part of the others.  (Three walks, so that
  // O is in no branch: the compiler kept it twice where it was.)
  const bool sees = x.see.hi >= x.see.lo && x.see.hi != 0x7fffffff;
  const unsigned long long seen = __ballot(sees);  // (spans do not fall from one row to the next)
  int w0 = 0x7fffffff, w1 = 0;
  if (seen) {
    w0 = __builtin_amdgcn_readlane(x.see.lo, __builtin_ctzll(seen)) / BN;
    w1 = __builtin_amdgcn_readlane(x.see.hi, 63 - __builtin_clzll(seen)) / BN + 1;
  }
  w0 = __builtin_amdgcn_readfirstlane(imin(imax(w0, ts.t0), ts.t1));
  w1 = __builtin_amdgcn_readfirstlane(imin(imax(w1, w0), ts.t1));
  int buf = 0;
  // the end of a tile: the next one's keys are there, and everyone has left this one
  auto turn = [&](int t) {
    const bool more = t + 1 < ts.t1;
    if constexpr (!kFp8) wait_vmem();
    if (more) look(t + 1, buf ^ 1);
    __syncthreads();
    buf ^= 1;
  };
  auto pass = [&](int t) {
    if (t + 1 < ts.t1) {
      if constexpr (kFp8) {
        codes_load(t + 1);
#pragma unroll
        for (int i = 0; i < 2 * CL; ++i) codes_store(buf ^ 1, i);
      } else {
        const Copy c = copy_plan(t + 1, buf ^ 1);
#pragma unroll
        for (int i = 0; i < 2 * IPW; ++i) copy_one(c, i);
      }
    }
    turn(t);
  };
  for (int t = ts.t0; t < w0; ++t) pass(t);
  int toggle = buf * TILE;  // of the LDS offsets: the buffers are a power of two apart
  for (int t = w0; t < w1; ++t) {
    const int kbase = t * BN;
    const bool more = t + 1 < ts.t1;
    [[maybe_unused]] Copy nc;
    if (more) {
      if constexpr (kFp8) codes_load(t + 1);
      else nc = copy_plan(t + 1, buf ^ 1);
    }
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) x.koff[k] ^= toggle;
#pragma unroll
    for (int i = 0; i < DT; ++i) x.voff[i] ^= toggle;
    toggle = TILE;
    const char* kl = lds;
    const char* vl = lds + 2 * TILE;
    f32x16 s[NSUB];
#pragma unroll
    for (int j = 0; j < NSUB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[j][e] = 0.f;
    constexpr int KPF = 2, KR = KPF + 1;  // K fragments ahead of their products
    frag ka[KR][NSUB];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int k = 0; k < KPF; ++k)
#pragma unroll
      for (int j = 0; j < NSUB; ++j) ka[k][j] = *reinterpret_cast<const u32x4*>(kl + j * 32 * RB + x.koff[k]);
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      if (k + KPF < KSTEPS) {
#pragma unroll
        for (int j = 0; j < NSUB; ++j) ka[(k + KPF) % KR][j] = *reinterpret_cast<const u32x4*>(kl + j * 32 * RB + x.koff[k + KPF]);
      }
#pragma unroll
      for (int j = 0; j < NSUB; ++j) s[j] = E::mma(ka[k % KR][j], x.qf[k], s[j]);
      if constexpr (!kFp8) {  // this step's share of the next tile's copies
#pragma unroll
        for (int i = 0; i < 2 * IPW; ++i)
          if (i * KSTEPS / (2 * IPW) == k && more) copy_one(nc, i);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (kMods) x.template modify<NSUB>(a, s, kbase, hh);
    x.template mask<NSUB>(s, kbase, hh);
    frag vt[2][NC];
    auto load_vt = [&](int i) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint2 lo = lds_read_tr16(vl + x.voff[i] + (16 * c) * RB);
        const uint2 hi = lds_read_tr16(vl + x.voff[i] + (16 * c + 4) * RB);
        vt[i & 1][c] = u32x4{lo.x, lo.y, hi.x, hi.y};
      }
    };
    load_vt(0);
    frag pf[NC];
    x.template softmax<NSUB>(s, pf);
    // the 2 wait states that an MFMA needs after a VALU write of its operand, once for all of P
    static_assert(NC == 4, "P fragments");
    asm volatile("s_nop 1" : "+v"(pf[0]), "+v"(pf[1]), "+v"(pf[2]), "+v"(pf[3]));
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      if (i + 1 < DT) load_vt(i + 1);
#pragma unroll
      for (int c = 0; c < NC; ++c) mfma_acc<'v', false>(x.oacc[i], vt[i & 1][c], pf[c]);
      if constexpr (kFp8) {  // the next tile's codes have come by now
#pragma unroll
        for (int p = 0; p < 2 * CL; ++p)
          if (p * DT / (2 * CL) == i && more) codes_store(buf ^ 1, p);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    if (cut(t)) {
      for (int y = 0; y < NW; ++y) {
        const int keys = __builtin_amdgcn_readfirstlane(wild[buf][y]);
        if (keys) x.patch(a, it.b, hk, kbase + WR * y, keys, lane);
      }
    }
    turn(t);
  }
  for (int t = w1; t < ts.t1; ++t) pass(t);

  x.drain();
  // (computed again: kept through the walk, it is one register too many at D = 64)
  const int le = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), lre = le & 31, hhe = le >> 5;
  const float lt = pair_sum(x.l);
  const auto me = W::row(a, it, it.row0 + 32 * w + lre);
  // row of lse (and of the partial results)
  const size_t at = ((size_t)(kPacked ? 0 : it.b) * a.Hq + hk * a.g + me.hq) * a.Sq + it.tok + me.qi;
  const size_t all = (size_t)(kPacked ? 1 : a.B) * a.Hq * a.Sq;
  if (me.valid && hhe == 0) note_ml(a, range, D, all, at, split_ml(x.m, lt, me.live));
  if (range.ranges > 1) {
    if (me.valid) {
      float* po = a.part + ((size_t)range.split * all + at) * D;
      if (ts.t0 < ts.t1 && me.live) {  // (else m = -inf says that there is no O)
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<f32x4*>(po + 32 * i + 8 * j + 4 * hhe) =
                f32x4{x.oacc[i][4 * j], x.oacc[i][4 * j + 1], x.oacc[i][4 * j + 2], x.oacc[i][4 * j + 3]};
      }
    }
    return;
  }
  // O through the wave's part of the (now idle) tiles, so that a store writes whole row segments
  const bool none = !me.live || lt == 0.f;  // (NaN is passed on)
  const float inv = none ? 0.f : 1.0f / lt;
  constexpr int RPI = 64 / KCH;
  char* stage = lds + w * (32 * RB);
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 4 * i + j;
      const u32x2 y{pack_bf16x2(x.oacc[i][4 * j] * inv, x.oacc[i][4 * j + 1] * inv),
                    pack_bf16x2(x.oacc[i][4 * j + 2] * inv, x.oacc[i][4 * j + 3] * inv)};
      *reinterpret_cast<u32x2*>(stage + lre * RB + ((c ^ (lre % KCH)) * 16) + hhe * 8) = none ? u32x2{0u, 0u} : y;
    }
  const int c = le % KCH;
#pragma unroll
  for (int k = 0; k < 32 / RPI; ++k) {
    const int rr = k * RPI + le / KCH, row = it.row0 + 32 * w + rr;
    const u32x4 y = *reinterpret_cast<const u32x4*>(stage + rr * RB + ((c ^ (rr % KCH)) * 16));
    if (row < rows) {
      const int i = row / a.g, hr = row - i * a.g;
      uint16_t* o = static_cast<uint16_t*>(a.o) + (kPacked ? 0 : it.b) * a.osb + (hk * a.g + hr) * a.osh + (long long)(it.tok + i) * a.ost;
      *reinterpret_cast<u32x4*>(o + c * 8) = y;
    }
  }
  if (me.valid && hhe == 0) a.lse[at] = none ? -INFINITY : (x.m + log2f(lt)) * kLn2;
}

// The splits of a row: M = max m_s, L = sum l_s 2^(m_s - M), O = sum O_s 2^(m_s - M) / L.  Four columns a thread, D / 4
// threads a row, of which thread j holds split j's factor (and j + D / 4's, ..); kWaves waves take every kWaves-th split of the same
// rows where few rows would leave one wave's loads one behind another.
template <int D, int kWaves>
__global__ __launch_bounds__(256) void prefill_merge(PrefillArgs a, long long rows) {
  constexpr int TPR = D / 4, DEEP = 4, HELD = kPrefillSplits / TPR < 1 ? 1 : kPrefillSplits / TPR;
  const int lane = threadIdx.x & 63, w = kWaves == 1 ? 0 : (int)threadIdx.x >> 6, j = lane % TPR;
  const long long row = ((long long)blockIdx.x * (256 / kWaves) + (kWaves == 1 ? (int)threadIdx.x : lane)) / TPR;
  const bool there = row < rows;
  const long long r = there ? row : rows - 1;
  const int n = a.n_splits, col = 4 * j;
  const float2* ml = reinterpret_cast<const float2*>(a.part + (size_t)n * rows * D) + r;
  const float* part = a.part + (size_t)r * D + col;
  float2 x[HELD];
  f32x4 y[DEEP];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < DEEP; ++u) y[u] = *reinterpret_cast<const f32x4*>(part + (size_t)imin(s0 + kWaves * u, n - 1) * rows * D);
  };
#pragma unroll
  for (int u = 0; u < HELD; ++u) x[u] = ml[(size_t)imin(j + TPR * u, n - 1) * rows];
  load(w);  // ahead of the factors
  const bool whole = __shfl(x[0].y, lane & ~(TPR - 1)) < 0.f;  // (its one range has written it)
  float M = -INFINITY;
#pragma unroll
  for (int u = 0; u < HELD; ++u) M = fmaxf(M, x[u].x);
#pragma unroll
  for (int d = TPR / 2; d >= 1; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
  float c[HELD], L = 0.f;
#pragma unroll
  for (int u = 0; u < HELD; ++u) {
    const bool mine = j + TPR * u < n && x[u].x != -INFINITY;  // (a split without a visible key has no O)
    c[u] = mine ? fast_exp2(x[u].x - M) : -1.f;
    L += mine ? x[u].y * c[u] : 0.f;
  }
#pragma unroll
  for (int d = TPR / 2; d >= 1; d >>= 1) L += __shfl_xor(L, d);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = w; s0 < n; s0 += kWaves * DEEP) {
    if (s0 != w) load(s0);
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      const int s = s0 + kWaves * u;
      float f = -1.f;
#pragma unroll
      for (int h = 0; h < HELD; ++h) f = s / TPR == h ? __shfl(c[h], (lane & ~(TPR - 1)) + s % TPR) : f;
      const bool has = s < n && f >= 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] = has ? fmaf(y[u][k], f, acc[k]) : acc[k];
    }
  }
  if constexpr (kWaves > 1) {
    __shared__ f32x4 sum[kWaves][64];
    sum[w][lane] = acc;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int i = 1; i < kWaves; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += sum[i][lane][k];
  }
  if (!there || whole) return;
  const float inv = L == 0.f ? 0.f : 1.0f / L;  // (NaN is passed on)
  const long long tok = row % a.Sq, bh = row / a.Sq;
  uint16_t* o = static_cast<uint16_t*>(a.o) + (bh / a.Hq) * a.osb + (bh % a.Hq) * a.osh + tok * a.ost + col;
  *reinterpret_cast<u32x2*>(o) =
      L == 0.f ? u32x2{0u, 0u} : u32x2{pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
  if (j == 0) a.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

}  // namespace fa
