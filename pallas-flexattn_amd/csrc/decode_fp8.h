// Attention of a row's newest queries over a paged KV cache in e4m3, one
// power-of-two scale per run of 32 tokens and kv head (decode), for gfx950.
//
//   o = softmax(mask(mod(scale q k~^T))) v~,  k~ = 2^e codes (bf16 holds them exactly)
//
// Bound by the reads of the cache (2 D + 1/4 bytes per key and kv head), so
// everything is laid out for those: a wave takes 32-key tiles (4 + 4 KiB at
// D = 128), its codes go from HBM straight into the registers that feed the
// matrix cores, the next tile's as soon as this one's are used; no LDS and no
// barrier inside the walk.  The g query heads of a kv head and their Sq queries
// are g Sq rows, a head's queries one after another, 16 NQ of them (16 or 32) per work
// item: groups of up to that many rows read the cache once.  Longer chunks of
// queries read it once per item, from the batch row's first visible key to its last
// whatever the item's own rows see: this is a kernel for few queries (B8 Hq32 Hkv8
// 32768 keys D128: 86 us for 538 MB, 6.2 TB/s, 4.7 more for the join; a causal prompt of
// 2000 tokens 170 us, where the bf16 prompt kernel takes 56).
//
// Layouts (v_mfma_f32_16x16x32_bf16; lane l = 16 g + r):
//   * S^T = K Q^T: A = 16 keys, lane (r, g) holds key r's bytes 64 c + 16 g + [0, 16)
//     of every 64-byte piece c: the sum over d may run in any order, so a
//     lane's 16 bytes are two of its k steps; B = Q rows r, the same d.
//   * the C tile gives lane (r, g) the scores of query r and A rows 4 g + i (i =
//     0..3) of both 16-key halves j; row 4 g + i is key 16 j + 4 i + g.  P stays in
//     those lanes as the B operand of O^T += V^T P^T, whose k index may name the keys
//     in that order; the A operand then wants the same eight keys of one d.
//   * V rows: lane (r, g) loads bytes [DV r, DV r + DV) (DV = D / 16) of its eight
//     keys: an instruction reads four consecutive rows, whole cache lines;
//     v_perm_b32 pairs two keys' bytes, the conversion to bf16 makes the
//     operand's words.  MFMA t is then rows d = DV r + t, and a lane ends
//     with 4 DV consecutive d of its query.
// P goes into the product as two bf16 pieces (its value and what that
// rounding left): the matrix cores are idle most of the time anyway, and a
// weight is then off by at most 2^-16, where O's own rounding is 2^-8 (a bf16
// weight would be off by as much).  Maxima may be stale by kLazy, which costs no bits:
// P and its sum scale alike.
#pragma once
#include "common.h"
#include "decode_index.h"

namespace fa {

struct DecodeArgs {
  const void* q;     // (B, Hq, Sq, D) bf16, strides of its first three dimensions
  long long qsb, qsh, qst;
  const uint8_t *k, *v;  // (num_pages, Hkv, page_size, D)
  const float *ks, *vs;  // (num_pages, Hkv, page_size / 32)
  const int* page_table;  // (B, max_pages); null: page b is row b's
  const int *kv_lens, *q_lens;  // (B) or null: every key of the table, Sq
  void* o;           // bf16
  float* lse;
  int B, Hkv, Sq, g;  // g query heads per kv head
  int page_runs, max_pages, num_pages, cap;  // runs per page, keys of the table
  int win_left, win_right;
  float scale, scale_log2, softcap;
  const float* alibi;
  int rt;            // query blocks per kv head
  int pieces, least; // what decode_chunk takes
  // by_item: a workgroup takes one whole item, nothing is shared.  Else the
  // workspace holds the rows' first units and slots (2 (B + 1) ints) and the slots'
  // O (16 NQ, D) and (m, l) (16 NQ, 2)
  int by_item, grid;
  int* head;
  float *part, *part_ml;
};

typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t cvt_e4m3_lo(uint32_t w, float s) {
  const bf16x2v r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false);
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint32_t cvt_e4m3_hi(uint32_t w, float s) {
  const bf16x2v r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true);
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0,
                                                 0);
}
// bit 7 of every byte of w that is a NaN code (S.1111.111)
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// maximum over the four lanes that share a query (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float quad_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// tanh to within 2.4 2^-24 of its value: below kTanhSmall an odd polynomial
// (minimax in x^2), above 1 - 2 / (e^2x + 1), which loses there what it cancels.
constexpr float kTanhSmall = 0.8f;
__device__ __forceinline__ float tanh_small(float x) {
  const float y = x * x;
  float p = fmaf(0.0016673924401402473f, y, -0.007573986891657114f);
  p = fmaf(p, y, 0.02142648957669735f);
  p = fmaf(p, y, -0.053895365446805954f);
  p = fmaf(p, y, 0.13332898914813995f);
  p = fmaf(p, y, -0.3333333432674408f);
  return fmaf(x * y, p, x);
}
__device__ __forceinline__ float tanh_large(float x) {
  return copysignf(fmaf(-2.0f, fast_rcp(fast_exp2(fabsf(x) * (2.0f * kLog2e)) + 1.0f), 1.0f), x);
}
// tanh of a lane's eight values; a wave whose values are all small or all
// large (ALiBi's far keys) takes one form (B16 H16 Sq4 D64, 1500-key window:
// 13.9 us, with both always 14.8, with the second alone, which is not exact, 13.6).
__device__ __forceinline__ void tanh8(f32x4* x) {
  float lo = INFINITY, hi = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = fabsf(x[e >> 2][e & 3]);
    lo = fminf(lo, t);
    hi = fmaxf(hi, t);
  }
  if (!__any(hi >= kTanhSmall)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = tanh_small(x[e >> 2][e & 3]);
  } else if (!__any(lo < kTanhSmall)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = tanh_large(x[e >> 2][e & 3]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = x[e >> 2][e & 3];
      x[e >> 2][e & 3] = fabsf(v) < kTanhSmall ? tanh_small(v) : tanh_large(v);
    }
  }
}

// Loads of the cache.  kStream: past the caches (non-temporal), where every
// load instruction reads whole 128-byte lines (V, and K rows of at most 64 bytes).
template <bool kStream, typename T>
__device__ __forceinline__ T code_load(const uint8_t* p) {
  if constexpr (kStream) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  else return *reinterpret_cast<const T*>(p);
}

// The codes of one tile, as a lane holds them.
template <int D, bool kStream>
struct CodeTile {
  static constexpr int DV = D / 16;               // V bytes per lane and key
  static constexpr int KC = D >= 64 ? D / 64 : 1; // K pieces per key
  static constexpr int KW = D >= 64 ? 4 : 2;      // words of a piece
  static constexpr int VW = DV >= 4 ? DV / 4 : 1; // words of a V row piece
  uint32_t k[2][KC][KW];
  uint32_t v[8][VW];
  __device__ __forceinline__ void load_k(const uint8_t* kp, int r, int g) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint8_t* p = kp + (16 * j + 4 * (r & 3) + (r >> 2)) * D + c * 64 + g * (4 * KW);
        if constexpr (KW == 4) {
          const u32x4 w = code_load<kStream && KC == 1, u32x4>(p);
#pragma unroll
          for (int x = 0; x < 4; ++x) k[j][c][x] = w[x];
        } else {
          const u32x2 w = code_load<kStream, u32x2>(p);
#pragma unroll
          for (int x = 0; x < 2; ++x) k[j][c][x] = w[x];
        }
      }
  }
  __device__ __forceinline__ void load_v(const uint8_t* vp, int r, int g) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint8_t* p = vp + (16 * (e >> 2) + 4 * (e & 3) + g) * D + DV * r;
      if constexpr (DV == 8) {
        const u32x2 w = code_load<kStream, u32x2>(p);
        v[e][0] = w[0];
        v[e][1] = w[1];
      } else if constexpr (DV == 4) {
        v[e][0] = code_load<kStream, uint32_t>(p);
      } else {
        v[e][0] = code_load<kStream, uint16_t>(p);
      }
    }
  }
  __device__ __forceinline__ void zero_k() {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int x = 0; x < KW; ++x) k[j][c][x] = 0u;
  }
};

__device__ __forceinline__ int row_keys(const DecodeArgs& a, int b) {
  return a.kv_lens ? clamp_len(a.kv_lens[b], a.cap) : a.cap;
}
__device__ __forceinline__ int row_queries(const DecodeArgs& a, int b) {
  return a.q_lens ? clamp_len(a.q_lens[b], a.Sq) : a.Sq;
}
// inclusive sum over the lanes of a wave (DPP: no LDS round trips)
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row 0 -> 1, 2 -> 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row 1 -> 2, 3
  return x;
}

// The piece of work of a workgroup (wave-uniform).
struct DecodeUnit {
  int b;                 // batch row; -1: no work left
  int have, ql;          // its keys and queries
  int item;              // kv head * rt + query block
  int t0, nt, slot;      // tiles, and the slot of a part of an item (-1: all of it)
};
// Every wave finds its workgroup's unit by itself: scans over the lanes, each of
// which holds the tiles of up to kRows consecutive rows, give the chunk and the rows' first units.
template <int kRows>
__device__ __forceinline__ DecodeUnit decode_piece_unit(const DecodeArgs& a, int wg, bool first_wave) {
  const int each = a.Hkv * a.rt;
  DecodeUnit u;
  const int lane = threadIdx.x & 63;
  const int per = (a.B + 63) / 64, b0 = lane * per;
  int n[kRows], sum = 0;  // tiles of this lane's rows, 0: no row
  bool same = true;
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int b = b0 + j;
    n[j] = j < per && b < a.B ? decode_span(row_keys(a, b), row_queries(a, b), a.win_left).n : 0;
    sum += n[j];
  }
  const int n0 = __builtin_amdgcn_readfirstlane(n[0]);
#pragma unroll
  for (int j = 0; j < kRows; ++j) same = same && (n[j] == 0 || n[j] == n0);
  // Equal rows make equal pieces, two per compute unit; of unequal ones, whose
  // pieces differ by up to half, twice as many come out more even (GPU time with two / four:
  // 8 equal rows of 32768 keys 97 / 99 us, 32 of 3840 49.8 / 51.7, 32 mixed to 8192 59.8 / 54.9,
  // D = 64 32 mixed to 9000 48 / 42).
  const int pieces = __all(same) ? a.pieces / 2 : a.pieces;
  const int total = __builtin_amdgcn_readlane(wave_scan(sum), 63) * each;
  int chunk = decode_chunk(total, pieces, a.least);
  int p[kRows], units, slots, iu;  // pieces per item, this lane's units and slots
  for (int i = 0;; ++i) {
    units = slots = 0;
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      p[j] = decode_pieces(n[j], chunk);
      decode_next_row(p[j], each, &units, &slots);
    }
    iu = wave_scan(units);
    const int all = __builtin_amdgcn_readlane(iu, 63);
    if (all <= pieces || a.B * each >= pieces || i == decode_tries(kRows)) break;
    chunk = decode_next_chunk(chunk, all, pieces);
  }
  const int is = wave_scan(slots);
  const int fu = iu - units, fs = is - slots;
  if (wg == 0 && first_wave) {  // for the merge
    int f = fu, g = fs;
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      if (n[j]) {
        a.head[2 * (b0 + j)] = f;
        a.head[2 * (b0 + j) + 1] = g;
      }
      decode_next_row(p[j], each, &f, &g);
    }
    if (lane == 63) a.head[2 * a.B] = iu;
  }
  // the lane whose rows hold unit wg, and the row among them
  const unsigned long long mine = __ballot(wg >= fu && wg < iu);
  if (!mine) {
    u.b = -1;
    return u;
  }
  const DecodeRow row = decode_find_row<kRows>(b0, n, p, each, wg, fu, fs);
  const int src = __builtin_ctzll(mine);
  u.b = __builtin_amdgcn_readlane(row.b, src);
  const int pb = __builtin_amdgcn_readlane(row.p, src);
  const int nb = __builtin_amdgcn_readlane(row.n, src);
  const int local = wg - __builtin_amdgcn_readlane(row.unit, src);
  u.have = a.kv_lens ? clamp_len(scalar_load(a.kv_lens, u.b), a.cap) : a.cap;
  u.ql = a.q_lens ? clamp_len(scalar_load(a.q_lens, u.b), a.Sq) : a.Sq;
  u.item = local / pb;
  const int piece = local - u.item * pb;
  const int lo = decode_piece(nb, pb, piece);
  u.t0 = decode_span(u.have, u.ql, a.win_left).lo + lo;
  u.nt = decode_piece(nb, pb, piece + 1) - lo;
  u.slot = pb > 1 ? __builtin_amdgcn_readlane(row.slot, src) + local : -1;
  return u;
}
__device__ __forceinline__ DecodeUnit decode_unit(const DecodeArgs& a, int wg, bool first_wave) {
  DecodeUnit u;
  if (a.by_item) {
    const int each = a.Hkv * a.rt;
    u.b = wg / each;
    u.item = wg - u.b * each;
    u.have = a.kv_lens ? clamp_len(scalar_load(a.kv_lens, u.b), a.cap) : a.cap;
    u.ql = a.q_lens ? clamp_len(scalar_load(a.q_lens, u.b), a.Sq) : a.Sq;
    const DecodeSpan s = decode_span(u.have, u.ql, a.win_left);
    u.t0 = s.lo;
    u.nt = s.n;
    u.slot = -1;
  } else if (a.B <= 64 * kLaneRows) {
    u = decode_piece_unit<kLaneRows>(a, wg, first_wave);
  } else {
    u = decode_piece_unit<kMostLaneRows>(a, wg, first_wave);
  }
  // (the compiler does not see that the branches' values are one per wave: four registers more)
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  return DecodeUnit{uniform(u.b), uniform(u.have), uniform(u.ql), uniform(u.item), uniform(u.t0), uniform(u.nt), uniform(u.slot)};
}

// kGeneral: score modifiers, or windows that differ between an item's rows
template <int D, int NQ, int NW, bool kGeneral, bool kStream>
__global__ __launch_bounds__(64 * NW, 2) void decode_fp8_kernel(DecodeArgs a) {
  using Tile = CodeTile<D, kStream>;
  constexpr int DV = Tile::DV, KC = Tile::KC, KW = Tile::KW;
  constexpr int KS = D / 32;           // k steps of S
  constexpr int OP = D + 4;            // floats per staged O row
  constexpr float kLazy = 8.0f;        // a maximum may be this stale (log2): P stays under 2^8
  __shared__ __attribute__((aligned(16))) float so[NW][16][OP];
  __shared__ float sml[NW][16][2];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g4 = lane >> 4;
  const DecodeUnit u = decode_unit(a, blockIdx.x, w == 0);
  if (u.b < 0) return;
  const int b = u.b, have = u.have, ql = u.ql, t0 = u.t0, nt = u.nt;
  const int hk = u.item / a.rt, qb = u.item - hk * a.rt;
  const int R = a.g * a.Sq;  // query rows of a kv head
  // score mods: s -> mod_out tanh(mod_in s), without a soft-cap mod_out s (log2 units)
  const float mod_in = a.softcap > 0.f ? 1.0f / a.softcap : 1.0f;
  const float mod_out = (a.softcap > 0.f ? a.softcap : 1.0f) * kLog2e;
  const int row0 = qb * (16 * NQ);

  // Q rows as B operands; rows past the group's end repeat its last one
  // (their results are not written)
  u32x4 qf[NQ][KS];
  int qlo[NQ], qhi[NQ];  // keys that this lane's rows see
  float slope[NQ];
  int qpos[NQ];
  const uint16_t* qp = static_cast<const uint16_t*>(a.q) + b * a.qsb + (long long)hk * a.g * a.qsh;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = min(row0 + 16 * n + r, R - 1);
    const int hq = row / a.Sq, i = row - hq * a.Sq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = D >= 64 ? (s >> 1) * 64 + 16 * g4 + 8 * (s & 1) : 8 * g4;
      qf[n][s] = *reinterpret_cast<const u32x4*>(qp + hq * a.qsh + i * a.qst + d);
    }
    qpos[n] = have - ql + i;
    qlo[n] = a.win_left < 0 ? 0 : window_first(qpos[n], a.win_left);
    qhi[n] = a.win_right < 0 ? have - 1 : (int)min((long long)have - 1, (long long)qpos[n] + a.win_right);
    if (i >= ql) qhi[n] = -1;  // a padded query sees nothing
    slope[n] = kGeneral && a.alibi ? a.alibi[hk * a.g + hq] : 0.f;
  }
  const int vlo = a.win_left < 0 ? 0 : window_first(have - ql, a.win_left);  // before it no row sees a key

  f32x4 acc[NQ][DV];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int t = 0; t < DV; ++t) acc[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // This wave's tiles: t0 + w, t0 + w + NW, ...; lane i holds run index (in
  // runs of the cache, -1 for a bad page) and scales of the i-th of them.
  const int mine = nt > w ? (nt - w + NW - 1) / NW : 0;
  int run_l = 0;
  float ks_l = 1.f, vs_l = 1.f;
  auto table = [&](int i0) {
    const int i = i0 + lane;
    run_l = -1;
    ks_l = vs_l = 1.f;
    if (i < mine) {
      const int t = t0 + w + NW * i;
      const int pg = t / a.page_runs;
      // (a row without keys walks one tile that is not there: its scale may be anything)
      const int page = t * kTileKeys >= have || pg >= a.max_pages ? -1 : a.page_table ? a.page_table[(size_t)b * a.max_pages + pg] : b;
      if (page >= 0 && page < a.num_pages) {
        run_l = (page * a.Hkv + hk) * a.page_runs + (t - pg * a.page_runs);
        ks_l = a.ks[run_l];
        vs_l = a.vs[run_l];
      }
    }
  };
  auto code_at = [&](int i) { return (size_t)max(__builtin_amdgcn_readlane(run_l, i & 63), 0) * (kTileKeys * D); };
  Tile x;
  // Tile i; the next one's codes are requested as soon as this one's registers are
  // free: its K behind the S product, its V behind the PV product.
  auto step = [&](int i, bool more) {
    const int run = __builtin_amdgcn_readlane(run_l, i & 63);
    const float ksc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_l), i & 63));
    const float vsc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs_l), i & 63));
    const int k0 = (t0 + w + NW * i) * kTileKeys;
    const size_t next = more ? code_at(i + 1) : 0;
    if (run < 0) x.zero_k();  // a page id outside the cache reads as zero keys
    f32x4 s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) s[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int y = 0; y < KW / 2; ++y) {
          const uint32_t w0 = x.k[j][c][2 * y], w1 = x.k[j][c][2 * y + 1];
          const u32x4 kf{cvt_e4m3_lo(w0, ksc), cvt_e4m3_hi(w0, ksc), cvt_e4m3_lo(w1, ksc), cvt_e4m3_hi(w1, ksc)};
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][j] = mma16(kf, qf[n][KW / 2 * c + y], s[n][j]);
        }
    if (more) x.load_k(a.k + next, r, g4);
    // scores in log2 units
    bool whole = true;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i2 = 0; i2 < 4; ++i2) {
          const float raw = s[n][j][i2];
          if constexpr (kGeneral) {
            s[n][j][i2] = fmaf(slope[n], (float)(k0 + 16 * j + 4 * i2 + g4 - qpos[n]), raw * a.scale) * mod_in;
          } else {
            s[n][j][i2] = raw * a.scale_log2;
          }
        }
      if constexpr (kGeneral) {
        if (a.softcap > 0.f) tanh8(s[n]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) s[n][j][i2] *= mod_out;
      }
      whole = whole && qlo[n] <= k0 && qhi[n] >= k0 + kTileKeys - 1;
    }
    const bool all_whole = __all(whole);
    if (!all_whole) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            const int key = k0 + 16 * j + 4 * i2 + g4;
            s[n][j][i2] = key >= qlo[n] && key <= qhi[n] ? s[n][j][i2] : -INFINITY;
          }
    }
    u32x4 ph[NQ], pl[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float mx = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                       fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
      if (__any(mx > m[n] + kLazy)) {
        const float mnew = fmaxf(m[n], quad_max(mx));
        const float alpha = m[n] == -INFINITY ? 0.f : fast_exp2(m[n] - mnew);
        m[n] = mnew;
        l[n] *= alpha;
#pragma unroll
        for (int t = 0; t < DV; ++t)
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) acc[n][t][i2] *= alpha;
      }
      const float ref = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float p0 = fast_exp2(s[n][y >> 1][2 * (y & 1)] - ref), p1 = fast_exp2(s[n][y >> 1][2 * (y & 1) + 1] - ref);
        l[n] += p0 + p1;
        const uint32_t hi = pack_bf16x2(p0, p1);
        ph[n][y] = hi;
        pl[n][y] = pack_bf16x2(p0 - bf16_lo(hi), p1 - bf16_hi(hi));
      }
    }
    if (run < 0 || k0 < vlo || k0 + kTileKeys > have) {
      // keys that no row sees may hold anything (also NaN codes): P = 0 there must meet V = 0
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = k0 + 16 * (e >> 2) + 4 * (e & 3) + g4;
        const bool ok = run >= 0 && key >= vlo && key < have;
#pragma unroll
        for (int y = 0; y < Tile::VW; ++y) x.v[e][y] = ok ? x.v[e][y] : 0u;
      }
    }
    if (kGeneral && !all_whole) {  // (otherwise a row sees the item's keys or none)
      // A NaN value code of a key that only some rows see must reach those alone, and
      // P = 0 would not keep it from the others: it is taken out, and the rows that see
      // one (a product of its flags and the rows' visible keys counts them) get NaN.
      uint32_t bad = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int y = 0; y < Tile::VW; ++y) bad |= nan_codes(x.v[e][y]);
      if (__any(bad != 0u)) {
        u32x4 seen[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int key = k0 + 16 * (y >> 1) + 8 * (y & 1) + g4;  // and key + 4
            seen[n][y] = (key >= qlo[n] && key <= qhi[n] ? 0x3f80u : 0u) |
                         (key + 4 >= qlo[n] && key + 4 <= qhi[n] ? 0x3f800000u : 0u);
          }
#pragma unroll
        for (int t = 0; t < DV; ++t) {
          u32x4 flag;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int sh = 8 * (t & 3) + 7;
            flag[y] = ((nan_codes(x.v[2 * y][t >> 2]) >> sh) & 1u) * 0x3f80u |
                      ((nan_codes(x.v[2 * y + 1][t >> 2]) >> sh) & 1u) * 0x3f800000u;
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            const f32x4 hits = mma16(flag, seen[n], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) acc[n][t][i2] = hits[i2] > 0.f ? __builtin_nanf("") : acc[n][t][i2];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int y = 0; y < Tile::VW; ++y) x.v[e][y] &= ~((nan_codes(x.v[e][y]) >> 7) * 0xffu);
      }
    }
#pragma unroll
    for (int t2 = 0; t2 < DV / 2; ++t2) {  // d = DV r + 2 t2 and + 1
      const int q = t2 >> 1;               // word of the row piece
      u32x4 v0, v1;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t w0 = x.v[2 * y][q], w1 = x.v[2 * y + 1][q];
        const uint32_t pr = __builtin_amdgcn_perm(w1, w0, (t2 & 1) ? 0x07030602u : 0x05010400u);
        v0[y] = cvt_e4m3_lo(pr, vsc);
        v1[y] = cvt_e4m3_hi(pr, vsc);
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        acc[n][2 * t2] = mma16(v0, ph[n], acc[n][2 * t2]);
        acc[n][2 * t2] = mma16(v0, pl[n], acc[n][2 * t2]);
        acc[n][2 * t2 + 1] = mma16(v1, ph[n], acc[n][2 * t2 + 1]);
        acc[n][2 * t2 + 1] = mma16(v1, pl[n], acc[n][2 * t2 + 1]);
      }
    }
    if (more) x.load_v(a.v + next, r, g4);
  };
  for (int i0 = 0; i0 < mine; i0 += 64) {
    table(i0);
    const int i1 = min(i0 + 64, mine);
    const size_t first = code_at(i0);
    x.load_k(a.k + first, r, g4);
    x.load_v(a.v + first, r, g4);
    for (int i = i0; i < i1; ++i) step(i, i + 1 < i1);
  }

  // join the waves: M = max m, L = sum l 2^(m - M), O = sum O 2^(m - M); TPR
  // threads per row, CW columns each
  constexpr int TPR = 4 * NW < D / 2 ? 4 * NW : D / 2, CW = D / TPR;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    if (n) __syncthreads();  // (the buffer's readers of the block before)
    const float lt = quad_sum(l[n]);
    if (g4 == 0) {
      sml[w][r][0] = m[n];
      sml[w][r][1] = lt;
    }
    // lane (r, g4): d = 4 DV g4 + DV i + t
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < DV; ++t) so[w][r][4 * DV * g4 + DV * i + t] = acc[n][t][i];
    __syncthreads();
    const int orow = tid / TPR, d0 = (tid % TPR) * CW;
    const int row = row0 + 16 * n + orow;
    if (orow < 16 && row < R) {
      float M = sml[0][orow][0];
#pragma unroll
      for (int i = 1; i < NW; ++i) M = fmaxf(M, sml[i][orow][0]);
      const float ref = M == -INFINITY ? 0.f : M;
      float L = 0.f, x[CW];
#pragma unroll
      for (int t = 0; t < CW; ++t) x[t] = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const float c = fast_exp2(sml[i][orow][0] - ref);
        L = fmaf(sml[i][orow][1], c, L);
#pragma unroll
        for (int t = 0; t < CW; ++t) x[t] = fmaf(so[i][orow][d0 + t], c, x[t]);
      }
      if (u.slot < 0) {
        const size_t at = (size_t)(b * a.Hkv + hk) * R + row;
        const float inv = L > 0.f ? 1.0f / L : L;  // (NaN is passed on)
        uint16_t* o = static_cast<uint16_t*>(a.o) + at * D + d0;
#pragma unroll
        for (int t = 0; t < CW; t += 2)  // a row that saw nothing may have met 0 * NaN
          *reinterpret_cast<uint32_t*>(o + t) = L == 0.f ? 0u : pack_bf16x2(x[t] * inv, x[t + 1] * inv);
        if (d0 == 0) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
      } else {
        const size_t at = (size_t)u.slot * (16 * NQ) + 16 * n + orow;
#pragma unroll
        for (int t = 0; t < CW; ++t) a.part[at * D + d0 + t] = x[t];
        if (d0 == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(M, L);
      }
    }
  }
}

// Items that several workgroups shared: a wave per output row adds up their
// pieces.  Lane s of 64 holds piece s's factor, the columns go over the lanes.
template <int D>
__global__ __launch_bounds__(256) void decode_fp8_merge(DecodeArgs a, int rows_per) {
  constexpr int CPL = D >= 64 ? D / 64 : 1, DEEP = 8;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int R = a.g * a.Sq;
  const int rows = a.B * a.Hkv * R;
  const int orow = blockIdx.x * 4 + w;
  if (orow >= rows) return;
  const int bh = orow / R, row = orow - bh * R;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int qb = row / rows_per, in = row - qb * rows_per;
  const int pn = (a.head[2 * b + 2] - a.head[2 * b]) / (a.Hkv * a.rt);
  if (pn == 1) return;  // one workgroup had it all
  const int slot = a.head[2 * b + 1] + (hk * a.rt + qb) * pn;
  const int col = lane * CPL < D ? lane * CPL : 0;
  auto at = [&](int p) { return (size_t)(slot + p) * rows_per + in; };
  float M = -INFINITY, L = 0.f, acc[CPL];
#pragma unroll
  for (int k = 0; k < CPL; ++k) acc[k] = 0.f;
  for (int p0 = 0; p0 < pn; p0 += 64) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (p0 + lane < pn) ml = *reinterpret_cast<const float2*>(a.part_ml + at(p0 + lane) * 2);
    const int np = min(64, pn - p0);
    float x[DEEP][CPL];
    auto load = [&](int i0) {
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        const float* p = a.part + at(p0 + min(i0 + i, np - 1)) * D + col;
#pragma unroll
        for (int k = 0; k < CPL; ++k) x[i][k] = p[k];
      }
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
    L = L * old + ls;
    M = mnew;
#pragma unroll
    for (int k = 0; k < CPL; ++k) acc[k] *= old;
    for (int i0 = 0; i0 < np; i0 += DEEP) {
      if (i0) load(i0);
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        const float ci = __shfl(c, (i0 + i) & 63);
#pragma unroll
        for (int k = 0; k < CPL; ++k) acc[k] = i0 + i < np ? fmaf(x[i][k], ci, acc[k]) : acc[k];
      }
    }
  }
  const size_t out = (size_t)orow;
  const float inv = L > 0.f ? 1.0f / L : L;
#pragma unroll
  for (int k = 0; k < CPL; ++k) acc[k] = L == 0.f ? 0.f : acc[k] * inv;  // (not 0 * NaN)
  if (lane * CPL < D) {
    uint16_t* o = static_cast<uint16_t*>(a.o) + out * D + col;
    if constexpr (CPL == 2) *reinterpret_cast<uint32_t*>(o) = pack_bf16x2(acc[0], acc[CPL - 1]);
    else *o = (uint16_t)(pack_bf16x2(acc[0], 0.f) & 0xffffu);
  }
  if (lane == 0) a.lse[out] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

}  // namespace fa
