// Instantiations and launches of the kernels around a KV cache: rotary
// positions, appends, and decode over an e4m3 cache.
#include "launch.h"

namespace fa {

static unsigned rotary_threads(const RotaryArgs& a) { return (unsigned)a.B * a.groups * a.units * a.T; }

int launch_rotary(const RotaryArgs& a, bool f32, bool vec, hipStream_t s) {
  const dim3 grid((rotary_threads(a) + 255) / 256);
  if (f32) {
    if (vec) hipLaunchKernelGGL((rotary_kernel<float, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<float, false>), grid, dim3(256), 0, s, a);
  } else {
    if (vec) hipLaunchKernelGGL((rotary_kernel<uint16_t, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<uint16_t, false>), grid, dim3(256), 0, s, a);
  }
  return launch_status();
}

template <int D>
static void run_append(const AppendArgs& a, bool fp8, hipStream_t s) {
  const unsigned turns = a.q.units ? (rotary_threads(a.q) + 2 * D - 1) / (2 * D) : 0;
  const dim3 grid(a.kv_blocks + turns), block(2 * D);
  if (fp8) hipLaunchKernelGGL((kv_append_kernel<D, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((kv_append_kernel<D, false>), grid, block, 0, s, a);
}

int launch_append(const AppendArgs& a, int D, bool fp8, hipStream_t s) {
  switch (D) {
    case 32: run_append<32>(a, fp8, s); break;
    case 64: run_append<64>(a, fp8, s); break;
    case 128: run_append<128>(a, fp8, s); break;
    default: return FA_ERR_UNSUPPORTED;
  }
  return launch_status();
}

template <int D, int NQ, int NW, bool G>
static void run_decode(const DecodeArgs& a, bool stream, hipStream_t s) {
  if (stream) hipLaunchKernelGGL((decode_fp8_kernel<D, NQ, NW, G, true>), dim3(a.grid), dim3(64 * NW), 0, s, a);
  else hipLaunchKernelGGL((decode_fp8_kernel<D, NQ, NW, G, false>), dim3(a.grid), dim3(64 * NW), 0, s, a);
}

template <int D, bool G>
static void decode_nq(const DecodeArgs& a, int nq, bool stream, hipStream_t s) {
  if (nq == 1 && a.by_item) run_decode<D, 1, 8, G>(a, stream, s);
  else if (nq == 1) run_decode<D, 1, 4, G>(a, stream, s);
  else run_decode<D, 2, 4, G>(a, stream, s);
  if (a.by_item) return;
  const int rows = a.B * a.Hkv * a.g * a.Sq;
  hipLaunchKernelGGL((decode_fp8_merge<D>), dim3(cdiv(rows, 4)), dim3(256), 0, s, a, 16 * nq);
}

int launch_decode_fp8(const DecodeArgs& a, int D, int nq, bool general, bool stream, hipStream_t s) {
  switch (D) {
    case 32: general ? decode_nq<32, true>(a, nq, stream, s) : decode_nq<32, false>(a, nq, stream, s); break;
    case 64: general ? decode_nq<64, true>(a, nq, stream, s) : decode_nq<64, false>(a, nq, stream, s); break;
    case 128: general ? decode_nq<128, true>(a, nq, stream, s) : decode_nq<128, false>(a, nq, stream, s); break;
    default: return FA_ERR_UNSUPPORTED;
  }
  return launch_status();
}

__global__ __launch_bounds__(256) void saturate_kernel(const int64_t* x, int32_t* y, unsigned n) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i < n) y[i] = (int32_t)min(max(x[i], (int64_t)INT32_MIN), (int64_t)INT32_MAX);
}

int launch_saturate(const int64_t* x, int32_t* y, long long n, hipStream_t s) {
  hipLaunchKernelGGL(saturate_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, x, y, (unsigned)n);
  return launch_status();
}

}  // namespace fa
