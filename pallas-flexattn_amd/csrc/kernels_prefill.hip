// Instantiations and launches of attention of chunks over a paged cache, one
// head dim (FA_KERNELS_D) per compilation.
#include "launch.h"
#include "prefill.h"

namespace fa {

template <int D, bool kFp8, bool kMods>
static void run_prefill(const PrefillArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)prefill_grid(a));
  if (a.starts) hipLaunchKernelGGL((prefill_kernel<D, kFp8, kMods, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((prefill_kernel<D, kFp8, kMods, false>), grid, dim3(256), 0, s, a);
}

template <>
int launch_prefill<FA_KERNELS_D>(const PrefillArgs& a, bool fp8, bool mods, hipStream_t s) {
  constexpr int D = FA_KERNELS_D;
  if (fp8) mods ? run_prefill<D, true, true>(a, s) : run_prefill<D, true, false>(a, s);
  else mods ? run_prefill<D, false, true>(a, s) : run_prefill<D, false, false>(a, s);
  const int rc = launch_status();
  if (rc || a.n_splits == 1) return rc;
  const long long rows = (long long)(a.starts ? 1 : a.B) * a.Hq * a.Sq;
  const long long threads = rows * (D / 4);
  if (a.n_splits > 4 && threads <= kMergeWide)
    hipLaunchKernelGGL((prefill_merge<D, 4>), dim3((unsigned)((threads + 63) / 64)), dim3(256), 0, s, a, rows);
  else
    hipLaunchKernelGGL((prefill_merge<D, 1>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, a, rows);
  return launch_status();
}

}  // namespace fa
