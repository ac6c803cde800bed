// Launches of the kernels on a cache's pages, and of appends to a cache of latent vectors.
#include "kv_pages.h"
#include "latent_append.h"
#include "launch.h"

namespace fa {

int launch_copy_pages(const CopyArgs& a, hipStream_t s) {
  const long long items = (long long)a.pairs * a.first[a.count];
  if (items == 0) return FA_OK;
  hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)(items < kCopyGrid ? items : kCopyGrid)), dim3(256), 0, s, a);
  return launch_status();
}

int launch_page_plan(const PagePlan& a, bool fork, hipStream_t s) {
  if (!a.marks) {
    if (fork) hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    else hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    return launch_status();
  }
  const unsigned rows = (unsigned)((a.N + 3) / 4), wide = rows < 2048u ? rows : 2048u;
  const unsigned pages = (unsigned)((a.num_pages + 255) / 256);
  hipLaunchKernelGGL(page_init_kernel, dim3(pages < 2048u ? pages : 2048u), dim3(256), 0, s, a);
  if (fork) {
    hipLaunchKernelGGL((page_mark_kernel<true>), dim3(wide), dim3(256), 0, s, a);
    hipLaunchKernelGGL((page_assign_kernel<true>), dim3(1), dim3(kPlanThreads), 0, s, a);
  } else {
    hipLaunchKernelGGL((page_mark_kernel<false>), dim3(wide), dim3(256), 0, s, a);
    hipLaunchKernelGGL((page_assign_kernel<false>), dim3(1), dim3(kPlanThreads), 0, s, a);
    hipLaunchKernelGGL(page_write_kernel, dim3(wide), dim3(256), 0, s, a);
  }
  return launch_status();
}

int launch_latent_append(const LatentAppendArgs& a, hipStream_t s) {
  const unsigned turns = a.q.units ? ((unsigned)a.B * a.q.groups * a.q.units * a.T + 255) / 256 : 0;
  hipLaunchKernelGGL(latent_append_kernel, dim3(a.kv_blocks + turns), dim3(256), 0, s, a);
  return launch_status();
}

}  // namespace fa
