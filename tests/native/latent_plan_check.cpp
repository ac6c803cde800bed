// The order of latent attention's workgroups (csrc/latent_plan.h): every block of every piece in one workgroup, and no XCD with
// much more than an eighth of them. Prints "ok" or where it differs.
#include <cstdio>
#include <vector>

#include "latent_plan.h"

using namespace fa;

int main() {
  for (int pieces = 1; pieces < 140; ++pieces)
    for (int rt = 1; rt < 700; rt += rt < 40 ? 1 : 61) {
      const bool near = latent_near(pieces, rt);
      const long long grid = latent_grid(pieces, rt, near);
      std::vector<int> got((size_t)pieces * rt, 0);
      long long load[kXcds] = {};
      for (long long wg = 0; wg < grid; ++wg) {
        const LatentPlace p = latent_place((int)wg, rt, near);
        if (p.block < 0 || p.block >= rt || p.piece < 0) return std::printf("%d pieces of %d blocks: a block %d\n", pieces, rt, p.block), 1;
        if (p.piece >= pieces) continue;  // (nothing to do)
        ++got[(size_t)p.piece * rt + p.block];
        ++load[wg % kXcds];
      }
      for (int n : got)
        if (n != 1) return std::printf("%d pieces of %d blocks: a block in %d workgroups\n", pieces, rt, n), 1;
      for (long long n : load)
        if (n > (long long)pieces * rt / kXcds + 8) return std::printf("%d pieces of %d blocks: %lld on an XCD\n", pieces, rt, n), 1;
    }
  std::printf("ok\n");
}
