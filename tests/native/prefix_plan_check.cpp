// The kernel of prefix attention (pz_prefixplan.h) for calls of rows, heads, tiles,
// own units, head_dim, ld and log2(block_size) on 256 CUs, seven arguments each; or
// `splits` with workgroups, tiles, the other part's tiles and the most.
#include <cstdio>
#include <cstdlib>
#include <string>

#include "pz_prefixplan.h"

int main(int argc, char** argv) {
  if (argc == 6 && std::string(argv[1]) == "splits") {
    std::printf("%d\n", pf_wide_splits(256, std::atol(argv[2]), std::atol(argv[3]),
                                       std::atol(argv[4]), std::atol(argv[5])));
    return 0;
  }
  for (int a = 1; a + 6 < argc; a += 7) {
    long v[7];
    for (int i = 0; i < 7; i++) v[i] = std::atol(argv[a + i]);
    std::printf("%d\n", (int)pf_kernel_for(v[0], v[1], v[2], v[3], 256, (int)v[4], v[5], (int)v[6]));
  }
}
