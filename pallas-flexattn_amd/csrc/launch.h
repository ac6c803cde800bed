// Launchers of the tile kernels: the C ABI (capi.hip) validates a call and
// picks its tiles, these pick the instantiation and launch it.  Defined in
// kernels.hip, which is compiled once per head dim and direction (the objects
// build in parallel).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/flexattn.h"
#include "bwd.h"
#include "decode_fp8.h"
#include "fwd.h"
#include "fwd_fp8.h"
#include "kv_append.h"
#include "page_plan.h"
#include "problem.h"

namespace fa {

inline int launch_status() { return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH; }

// Element type T (uint16_t: bf16, float), head dim D, with (M) or without
// the built-in score mods (ALiBi, soft-cap); tiles as chosen by the C ABI.
// A tile with no instantiation returns FA_ERR_UNSUPPORTED.
template <typename T, int D, bool M>
int launch_fwd(const FwdArgs& a, const Tiles& t, hipStream_t s);  // forward (+ split-KV merge)
template <typename T, int D, bool M>
int launch_dq(const BwdArgs& a, const Tiles& t, hipStream_t s);
template <typename T, int D, bool M>
int launch_dkdv(const BwdArgs& a, const Tiles& t, hipStream_t s);
template <typename T, int D>
int launch_delta(const BwdArgs& a, hipStream_t s);  // Delta = rowsum(dO * O)

// fp8 forward (D = 64 or 128, 128 x 64 tiles) and the bf16 -> e4m3 block
// quantiser (kernels_fp8.hip); q16: Q is bf16, quantised in the kernel
int launch_fwd_fp8(const Fp8FwdArgs& a, int D, bool mods, bool q16, hipStream_t s);
int launch_quant_fp8(const QuantArgs& a, hipStream_t s);

// Around a KV cache (kernels_cache.hip): rotary positions (f32 or bf16; vec:
// 16-byte accesses), appends (D = 32, 64 or 128), decode over e4m3 pages
// (nq: 16-row query blocks per work item, 1 or 2; stream: cache reads past the
// caches), and n < 2^31 64-bit lengths or page ids as 32-bit ones
int launch_rotary(const RotaryArgs& a, bool f32, bool vec, hipStream_t s);
int launch_append(const AppendArgs& a, int D, bool fp8, hipStream_t s);
int launch_decode_fp8(const DecodeArgs& a, int D, int nq, bool general, bool stream, hipStream_t s);
struct CopyArgs;
struct LatentAppendArgs;
struct LatentArgs;
struct PrefillArgs;

// Chunks of new tokens over a paged cache (kernels_prefill.hip: D = 32, 64 or 128; mods: ALiBi or a soft-cap), rows
// over a cache of latent vectors (kernels_latent.hip: L = 128, 256 or 512, R = 32 or 64; nb: 16-row blocks per
// work item, 1 to 4), appends to it, and pages (kernels_pages.hip; marks null: the plan of one workgroup)
template <int D>
int launch_prefill(const PrefillArgs& a, bool fp8, bool mods, hipStream_t s);
template <int L>
int launch_latent(const LatentArgs& a, int R, int nb, hipStream_t s);
int launch_latent_append(const LatentAppendArgs& a, hipStream_t s);
constexpr int kCopyGrid = 2048;
int launch_copy_pages(const CopyArgs& a, hipStream_t s);
int launch_page_plan(const PagePlan& a, bool fork, hipStream_t s);
int launch_saturate(const int64_t* x, int32_t* y, long long n, hipStream_t s);

}  // namespace fa
