// Instantiations and launches around a cache of latent vectors, one length of
// them (FA_KERNELS_L) per compilation.
#include "latent.h"
#include "launch.h"

namespace fa {

template <int L, int R>
static void run_latent(const LatentArgs& a, int nb, hipStream_t s) {
  const dim3 grid(a.d.grid);
  switch (nb) {
    case 1: hipLaunchKernelGGL((latent_decode_kernel<L, R, 1>), grid, dim3(256), 0, s, a); break;
    case 2: hipLaunchKernelGGL((latent_decode_kernel<L, R, 2>), grid, dim3(256), 0, s, a); break;
    case 3: hipLaunchKernelGGL((latent_decode_kernel<L, R, 3>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((latent_decode_kernel<L, R, 4>), grid, dim3(256), 0, s, a); break;
  }
}

template <>
int launch_latent<FA_KERNELS_L>(const LatentArgs& a, int R, int nb, hipStream_t s) {
  constexpr int L = FA_KERNELS_L;
  if (R == 32) run_latent<L, 32>(a, nb, s);
  else run_latent<L, 64>(a, nb, s);
  const int rc = launch_status();
  if (rc || a.d.by_item) return rc;
  const long long units = (long long)a.d.B * a.d.g * a.d.Sq * (L >= 256 ? L / 256 : 1);
  if (units <= kMergeWide / 64)
    hipLaunchKernelGGL((latent_merge<L, 4>), dim3((unsigned)units), dim3(256), 0, s, a.d, a.rt, 16 * nb);
  else
    hipLaunchKernelGGL((latent_merge<L, 1>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, s, a.d, a.rt, 16 * nb);
  return launch_status();
}

}  // namespace fa
