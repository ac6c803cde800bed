// The 16-row blocks per item that a decode call takes (csrc/decode_index.h), for "rows heads
// tiles" in the arguments, three for each call.
#include <cstdio>
#include <cstdlib>

#include "decode_index.h"

int main(int argc, char** argv) {
  for (int i = 1; i + 2 < argc; i += 3) std::printf("%d ", fa::decode_blocks(atoll(argv[i]), atoll(argv[i + 1]), atoll(argv[i + 2])));
  return 0;
}
