// Rotary positions for gfx950: y = s R(pos f) x on the first 2n elements of a
// head, R a rotation of n element pairs; the rest is copied.
//
//   y1 = s (x1 cos a - x2 sin a),  y2 = s (x2 cos a + x1 sin a),  a = pos f_i
//
// The backward is the transpose, the rotation by -a (inverse).  Bound by HBM:
// each element is read once and written once (3 flops), so all that counts is
// that the angles cost little beside that: a thread holds the sines and
// cosines of its eight pairs of one token in registers and takes them through
// several heads.
#pragma once
#include "common.h"

namespace fa {

// One tensor of a rotary call: element strides of (batch, head, token), the
// last dimension dense; the output is dense (B, H, T, D).
struct RotaryTensor {
  const void* x;
  void* y;
  long long sb, sh, st;
  int heads;
};

struct RotaryArgs {
  RotaryTensor t[2];
  int B, T, D;
  const double* freq;  // radians per position of the n pairs
  int n;
  int interleaved, inverse;
  float scale;
  // position of token t of row b: positions[b * pos_stride + t] (32 or 64 bits),
  // or offset + t, or with kv_lens kv_lens[b] + t
  const void* positions;
  int pos64;
  long long pos_stride, offset;
  const int* kv_lens;
  // geometry: a thread takes unit u (of `units`) of one token for `per` heads
  int units, groups, per;
};

// sin and cos of 2 pi turns f radians, turns = pos / (2 pi).  The angle is kept in
// turns in 64 bits (off by pos f 2^-52: 2e-10 at a million radians, where a 32-bit
// product would be off by a hundredth of a turn) until whole turns and the nearest
// quarter are taken off; the Taylor series of sine (to x^9) and cosine (to x^10) on
// |x| <= pi / 4 leave under 2e-9: fp32 rounding is what remains.
__device__ __forceinline__ void sincos_turns(double turns, double f, float* sn, float* cs) {
  double t = turns * f;
  t -= rint(t);
  const float q = rintf(4.0f * (float)t);  // quarter turns, -2 .. 2
  const float x = (float)fma(-0.25, (double)q, t) * 6.2831853f;
  const float z = x * x;
  float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(s, z, 8.3333333e-3f);
  s = fmaf(s, z, -1.6666667e-1f);
  s = fmaf(s * z, x, x);
  float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(c, z, -1.3888889e-3f);
  c = fmaf(c, z, 4.1666667e-2f);
  c = fmaf(c, z, -0.5f);
  c = fmaf(c, z, 1.0f);
  const int k = (int)q;
  const bool swap = k & 1;
  const float a = swap ? c : s, b = swap ? s : c;
  *sn = (k & 2) ? -a : a;
  *cs = ((k + 1) & 2) ? -b : b;
}

// (cos, sin) x scale of pairs p0 .. p0 + 3 and p1 .. p1 + 3 (past the n-th: 1 and 0).
__device__ __forceinline__ void rotary_angles(const double* freq, int p0, int p1, int n, double pos, float scale, bool inverse,
                                              float* cs, float* sn) {
  const double turns = pos * 0.15915494309189533577;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = j < 4 ? p0 + j : p1 + j - 4;
    cs[j] = 1.f;
    sn[j] = 0.f;
    if (p < n) {
      float s, c;
      sincos_turns(turns, freq[p], &s, &c);
      cs[j] = c * scale;
      sn[j] = (inverse ? -s : s) * scale;
    }
  }
}

// Elements of a 16-byte-aligned eight-element chunk as floats, and back.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (sizeof(T) == 2) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t v = w[t];
      x[2 * t] = bf16_lo(v);
      x[2 * t + 1] = bf16_hi(v);
    }
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      x[t] = a[t];
      x[4 + t] = b[t];
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<u32x4*>(p) = Elt<uint16_t>::pack(x);
  } else {
    *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  }
}
__device__ __forceinline__ float load1(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ void store1(uint16_t* p, float x) { *p = (uint16_t)(pack_bf16x2(x, 0.f) & 0xffffu); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }

// Where unit u's two eight-element chunks start (vector form: 2n and D are
// multiples of 16), half of the rotated (or of the copied) elements apart, so that neighbouring
// threads read neighbouring chunks: with 16 consecutive elements per thread float32
// B4 H16 T1000 D64 took 11.5 us, so 9.4.  Half layout: chunk a holds the
// first elements of pairs p0 .. p0 + 7, chunk b the second ones; interleaved:
// chunk a pairs p0 .. p0 + 3, chunk b pairs p1 .. p1 + 3.
struct RotaryUnit {
  int a, b, p0, p1;
  bool turn, half;
};
__device__ __forceinline__ RotaryUnit rotary_unit(int u, int n, int D, bool interleaved) {
  RotaryUnit r;
  const int v = u - n / 8;  // unit of the copied elements
  r.turn = v < 0;
  r.half = r.turn && !interleaved;
  r.a = r.turn ? 8 * u : 2 * n + 8 * v;
  r.b = r.turn ? 8 * u + n : D / 2 + n + 8 * v;
  r.p0 = r.half ? 8 * u : r.turn ? 4 * u : n;
  r.p1 = r.half ? 8 * u + 4 : r.turn ? 4 * u + n / 2 : n;
  return r;
}
// Rotates the unit's 16 values in place.
__device__ __forceinline__ void rotary_turn(const RotaryUnit& r, float* xa, float* xb, const float* cs, const float* sn) {
  if (!r.turn) return;
  if (r.half) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = xa[j], q = xb[j];
      xa[j] = fmaf(p, cs[j], -(q * sn[j]));
      xb[j] = fmaf(q, cs[j], p * sn[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float* x = j < 4 ? xa : xb;
      const int i = 2 * (j & 3);
      const float p = x[i], q = x[i + 1];
      x[i] = fmaf(p, cs[j], -(q * sn[j]));
      x[i + 1] = fmaf(q, cs[j], p * sn[j]);
    }
  }
}

// Flat thread id -> (row, token, head group, unit), the unit fastest (16
// lanes write whole rows), then the token.
template <typename T, bool kVec>
__device__ __forceinline__ void rotary_thread(const RotaryArgs& a, unsigned id) {
  const unsigned per_row = (unsigned)a.units * a.T;  // (B groups units T < 2^31: the host's check)
  const unsigned row = id / per_row;
  if (row >= (unsigned)a.B * a.groups) return;
  const unsigned in_row = id - row * per_row;
  const int tok = (int)(in_row / a.units), u = (int)(in_row - (unsigned)tok * a.units);
  const int b = (int)(row / a.groups), grp = (int)(row - (unsigned)b * a.groups);
  double pos;
  if (a.kv_lens) pos = (double)a.kv_lens[b] + tok;
  else if (!a.positions) pos = (double)(a.offset + tok);
  else if (a.pos64) pos = (double)static_cast<const long long*>(a.positions)[b * a.pos_stride + tok];
  else pos = (double)static_cast<const int*>(a.positions)[b * a.pos_stride + tok];
  float cs[8], sn[8];
  RotaryUnit r{0, 0, 8 * u, 8 * u + 4, true, true};
  if constexpr (kVec) r = rotary_unit(u, a.n, a.D, a.interleaved);
  rotary_angles(a.freq, r.p0, r.p1, a.n, pos, a.scale, a.inverse, cs, sn);
  const int all = a.t[0].heads + a.t[1].heads;
  const int h0 = grp * a.per, h1 = min(h0 + a.per, all);
  for (int hh = h0; hh < h1; ++hh) {
    const int second = hh >= a.t[0].heads;
    const RotaryTensor& R = a.t[second];
    const int h = hh - (second ? a.t[0].heads : 0);
    const T* x = static_cast<const T*>(R.x) + b * R.sb + h * R.sh + tok * R.st;
    T* y = static_cast<T*>(R.y) + (((size_t)b * R.heads + h) * a.T + tok) * a.D;
    if constexpr (kVec) {
      float xa[8], xb[8];
      load8(x + r.a, xa);
      load8(x + r.b, xb);
      rotary_turn(r, xa, xb, cs, sn);
      store8(y + r.a, xa);
      store8(y + r.b, xb);
    } else {
      // any 2n, D and alignment: units [0, ceil(n / 8)) take eight pairs each, the following ones
      // sixteen copied elements each, one element per access (bf16 B4 H32 + 32 T8192 D96, forward
      // and gradient: 24 rotated elements 1566 us, 32 of them in the other form 319)
      const int pair_units = (a.n + 7) / 8;
      if (u < pair_units) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = 8 * u + j;
          if (i < a.n) {
            const int e0 = a.interleaved ? 2 * i : i, e1 = a.interleaved ? 2 * i + 1 : i + a.n;
            const float p = load1(x + e0), q = load1(x + e1);
            store1(y + e0, fmaf(p, cs[j], -(q * sn[j])));
            store1(y + e1, fmaf(q, cs[j], p * sn[j]));
          }
        }
      } else {
        const int e0 = 2 * a.n + 16 * (u - pair_units);
        for (int e = e0; e < min(e0 + 16, a.D); ++e) y[e] = x[e];
      }
    }
  }
}

template <typename T, bool kVec>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  rotary_thread<T, kVec>(a, blockIdx.x * 256u + threadIdx.x);
}

}  // namespace fa
