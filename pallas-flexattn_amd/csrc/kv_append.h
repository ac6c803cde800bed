// New keys and values into a paged KV cache, keys rotated to their positions
// on the way, in bf16 or in e4m3 with one power-of-two scale per run of
// kRunTokens tokens of a head; the queries of the same tokens rotated by the
// launch's further workgroups (rotary.h).
//
// The scale of a run is 2^e, e the smallest integer in [-126, 127] with
// 448 2^e at least the largest finite |x| of the run's tokens, and never less than
// what tokens appended earlier needed: a run that a call finds begun keeps its
// scale, or takes the larger one and moves its old codes to it (a division by
// a power of two, rounded to nearest even: exact while they stay normal).
// Keys are quantised from their rotated float32 values: one rounding.
//
// A workgroup owns whole runs (D / 16 threads per token, kRunTokens tokens; a
// thread has 16 values of K and of V), so scales need no atomics and results do
// not depend on any order.  Bound by HBM (2 + 2 bytes read, 1 + 1 written per
// element); for single tokens by the launch.
#pragma once
#include "rotary.h"

namespace fa {

constexpr int kRunTokens = 32;

struct AppendArgs {
  const void *k, *v;  // bf16
  long long ksb, ksh, kst, vsb, vsh, vst;
  void *kc, *vc;      // (num_pages, Hkv, page_size, D) bf16 or e4m3
  float *ks, *vs;     // e4m3: (num_pages, Hkv, page_size / kRunTokens)
  const int* page_table;  // (B, max_pages); null: page b is row b's
  int page_size, max_pages, num_pages;
  const int* kv_lens;   // (B) keys before the call
  const int* new_lens;  // (B) or null: T
  int B, Hkv, T;
  const double* freq;  // null: keys are not rotated
  int n, interleaved;
  float scale;
  int runs, groups, per;  // runs per row that T tokens can touch; kv heads in `groups` of `per`
  int kv_blocks;          // workgroups of this part; the following ones rotate queries
  RotaryArgs q;
};

// Largest of a wave's non-negative values, in every lane (DPP row rotations,
// then the swaps across rows: no LDS round trips).
__device__ __forceinline__ float wave_max(float x) {
  auto turn = [](float v, auto ctrl) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  x = fmaxf(x, turn(x, Int<0x121>{}));  // row_ror 1, 2, 4, 8
  x = fmaxf(x, turn(x, Int<0x122>{}));
  x = fmaxf(x, turn(x, Int<0x124>{}));
  x = fmaxf(x, turn(x, Int<0x128>{}));
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

__device__ __forceinline__ float finite_max(float m, float x) {
  const float a = fabsf(x);
  return a < INFINITY ? fmaxf(m, a) : m;  // (NaN and infinities stay out: their codes are NaN)
}
// exponent e of the scale that holds values up to amax: 448 2^e = 1.75 2^(e + 8)
__device__ __forceinline__ int run_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) > 0x600000u ? 7 : 8);
  return e < -126 ? -126 : e;
}
__device__ __forceinline__ int scale_exp(float s) {
  const int e = (int)((__float_as_uint(s) >> 23) & 0xffu) - 127;
  return min(max(e, -126), 127);
}
__device__ __forceinline__ u32x2 pack_e4m3(const float* x, int e) {
  float y[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) y[t] = ldexpf(x[t], -e);
  int w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w0, true);
  int w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], w1, true);
  return u32x2{(uint32_t)w0, (uint32_t)w1};
}
__device__ __forceinline__ u32x2 move_e4m3(u32x2 w, int down) {  // codes x 2^-down
  float x[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = w[i];
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
    x[4 * i] = lo[0];
    x[4 * i + 1] = lo[1];
    x[4 * i + 2] = hi[0];
    x[4 * i + 3] = hi[1];
  }
  return pack_e4m3(x, down);
}

template <int D, bool kFp8>
__global__ __launch_bounds__(2 * D) void kv_append_kernel(AppendArgs a) {
  constexpr int U = D / 16;            // threads per token
  constexpr int NT = U * kRunTokens;   // 2 D
  constexpr int NW = NT / 64;
  static_assert(NT == 2 * D && NW >= 1, "workgroup");
  if ((int)blockIdx.x >= a.kv_blocks) {
    rotary_thread<uint16_t, true>(a.q, (blockIdx.x - a.kv_blocks) * (unsigned)NT + threadIdx.x);
    return;
  }
  [[maybe_unused]] __shared__ float red[2][2][NW];
  const int tid = threadIdx.x, u = tid % U, row = tid / U;
  const int per_b = a.runs * a.groups;
  const int b = blockIdx.x / per_b, rest = blockIdx.x - b * per_b;
  const int grp = rest / a.runs, run = rest - grp * a.runs;
  const int len = a.kv_lens[b];
  const int fresh = a.new_lens ? min(max(a.new_lens[b], 0), a.T) : a.T;
  if (len < 0 || fresh == 0) return;
  // the run's first position; tokens [len, len + fresh) are the new ones
  const long long p0 = ((long long)len / kRunTokens + run) * kRunTokens;
  if (p0 >= (long long)len + fresh) return;
  const long long pg = p0 / a.page_size;
  if (pg >= a.max_pages) return;  // past the table: dropped
  const int page = a.page_table ? a.page_table[(size_t)b * a.max_pages + pg] : b;
  const int off = (int)(p0 - pg * a.page_size);
  const long long pos = p0 + row;
  const int tok = (int)(pos - len);
  const bool mine = pos >= len && tok < fresh;
  const bool begun = p0 < len, old = pos < len;

  const RotaryUnit r = rotary_unit(u, a.freq ? a.n : 0, D, a.interleaved);
  float cs[8], sn[8];
  if (a.freq && mine) rotary_angles(a.freq, r.p0, r.p1, a.n, (double)pos, a.scale, false, cs, sn);
  if (page < 0 || page >= a.num_pages) return;  // (the page's id comes in beside the angles)
  const int h1 = min((grp + 1) * a.per, a.Hkv);
  for (int h = grp * a.per; h < h1; ++h) {
    const size_t first = ((size_t)page * a.Hkv + h) * a.page_size + off;  // the run's first cache row
    const uint16_t* k = static_cast<const uint16_t*>(a.k) + b * a.ksb + h * a.ksh + tok * a.kst;
    const uint16_t* v = static_cast<const uint16_t*>(a.v) + b * a.vsb + h * a.vsh + tok * a.vst;
    float ka[8] = {}, kb[8] = {}, va[8] = {}, vb[8] = {};
    if (mine) {
      load8(k + r.a, ka);
      load8(k + r.b, kb);
      load8(v + r.a, va);
      load8(v + r.b, vb);
      rotary_turn(r, ka, kb, cs, sn);
    }
    if constexpr (!kFp8) {
      if (mine) {
        uint16_t* kd = static_cast<uint16_t*>(a.kc) + (first + row) * D;
        uint16_t* vd = static_cast<uint16_t*>(a.vc) + (first + row) * D;
        store8(kd + r.a, ka);
        store8(kd + r.b, kb);
        store8(vd + r.a, va);
        store8(vd + r.b, vb);
      }
    } else {
      const size_t si = first / kRunTokens;
      int ke0 = 0, ve0 = 0;
      if (begun) {  // (workgroup-uniform; read before the barrier, written behind it)
        ke0 = scale_exp(a.ks[si]);
        ve0 = scale_exp(a.vs[si]);
      }
      float km = 0.f, vm = 0.f;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        km = finite_max(finite_max(km, ka[t]), kb[t]);
        vm = finite_max(finite_max(vm, va[t]), vb[t]);
      }
      km = wave_max(km);
      vm = wave_max(vm);
      if constexpr (NW > 1) {
        // (two buffers: a wave is at most one head ahead of the barrier's slowest)
        float(*m)[NW] = red[h & 1];
        if ((tid & 63) == 0) {
          m[0][tid >> 6] = km;
          m[1][tid >> 6] = vm;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          km = fmaxf(km, m[0][w]);
          vm = fmaxf(vm, m[1][w]);
        }
      }
      int ke = run_exp(km), ve = run_exp(vm);
      if (begun) {
        ke = max(ke, ke0);
        ve = max(ve, ve0);
      }
      if (tid == 0) {
        a.ks[si] = ldexpf(1.f, ke);
        a.vs[si] = ldexpf(1.f, ve);
      }
      uint8_t* kd = static_cast<uint8_t*>(a.kc) + (first + row) * D;
      uint8_t* vd = static_cast<uint8_t*>(a.vc) + (first + row) * D;
      if (mine) {
        *reinterpret_cast<u32x2*>(kd + r.a) = pack_e4m3(ka, ke);
        *reinterpret_cast<u32x2*>(kd + r.b) = pack_e4m3(kb, ke);
        *reinterpret_cast<u32x2*>(vd + r.a) = pack_e4m3(va, ve);
        *reinterpret_cast<u32x2*>(vd + r.b) = pack_e4m3(vb, ve);
      } else if (old) {
        if (ke > ke0) {
          *reinterpret_cast<u32x2*>(kd + r.a) = move_e4m3(*reinterpret_cast<const u32x2*>(kd + r.a), ke - ke0);
          *reinterpret_cast<u32x2*>(kd + r.b) = move_e4m3(*reinterpret_cast<const u32x2*>(kd + r.b), ke - ke0);
        }
        if (ve > ve0) {
          *reinterpret_cast<u32x2*>(vd + r.a) = move_e4m3(*reinterpret_cast<const u32x2*>(vd + r.a), ve - ve0);
          *reinterpret_cast<u32x2*>(vd + r.b) = move_e4m3(*reinterpret_cast<const u32x2*>(vd + r.b), ve - ve0);
        }
      }
    }
  }
}

}  // namespace fa
