// New tokens' latent vectors and rotary parts into a paged cache of them, the rotary parts turned to
// their positions on the way (rotary.h); the launch's further workgroups turn the queries' rotary parts.
// A thread takes 16 elements of a token.  Bound by the launch (a few tokens 6 us), for prompts by HBM (2 bytes read and
// 2 written an element): 8 x 4096 tokens of 512 + 64 with 16 heads' queries 43 us, 4.9 TB/s, with 128 heads' 244, 4.7; without
// queries 24, 3.2 TB/s; 1024 tokens 11 and 13.
#pragma once
#include "latent_args.h"

namespace fa {

__global__ __launch_bounds__(256) void latent_append_kernel(LatentAppendArgs a) {
  if ((int)blockIdx.x >= a.kv_blocks) {
    rotary_thread<uint16_t, true>(a.q, (blockIdx.x - a.kv_blocks) * 256u + threadIdx.x);
    return;
  }
  const unsigned id = blockIdx.x * 256u + threadIdx.x;  // (B T units < 2^31: the host's check)
  const unsigned token = id / (unsigned)a.units;
  const int u = (int)(id - token * a.units);
  const int b = (int)(token / (unsigned)a.T), t = (int)(token - (unsigned)b * a.T);
  if (b >= a.B) return;
  const int len = a.kv_lens[b];
  const int fresh = a.new_lens ? min(max(a.new_lens[b], 0), a.T) : a.T;
  if (len < 0 || t >= fresh) return;
  const long long pos = (long long)len + t, pg = pos / a.page_size;
  if (pg >= a.max_pages) return;  // past the table: dropped
  const int page = a.page_table ? a.page_table[(size_t)b * a.max_pages + pg] : b;
  if (page < 0 || page >= a.num_pages) return;
  uint16_t* to = a.cache + ((size_t)page * a.page_size + (size_t)(pos - pg * a.page_size)) * (a.L + a.R);
  if (u < a.L / 16) {
    const u32x4* x = reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.latent) + b * a.lsb + t * a.lst + 16 * u);
    const u32x4 x0 = x[0], x1 = x[1];
    u32x4* y = reinterpret_cast<u32x4*>(to + 16 * u);
    y[0] = x0;
    y[1] = x1;
    return;
  }
  const RotaryUnit r = rotary_unit(u - a.L / 16, a.freq ? a.n : 0, a.R, a.interleaved);
  const uint16_t* x = static_cast<const uint16_t*>(a.rope) + b * a.rsb + t * a.rst;
  float xa[8], xb[8];
  load8(x + r.a, xa);
  load8(x + r.b, xb);
  if (a.freq) {
    float cs[8], sn[8];
    rotary_angles(a.freq, r.p0, r.p1, a.n, (double)pos, a.scale, false, cs, sn);
    rotary_turn(r, xa, xb, cs, sn);
  }
  store8(to + a.L + r.a, xa);
  store8(to + a.L + r.b, xb);
}

}  // namespace fa
