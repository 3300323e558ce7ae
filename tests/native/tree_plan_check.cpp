// The kernel of tree attention (pz_treeplan.h) for calls of rows, heads, tiles,
// head_dim, ld and ld_n on 256 CUs, six arguments each.
#include <cstdio>
#include <cstdlib>

#include "pz_treeplan.h"

int main(int argc, char** argv) {
  for (int a = 1; a + 5 < argc; a += 6) {
    long v[6];
    for (int i = 0; i < 6; i++) v[i] = std::atol(argv[a + i]);
    std::printf("%d\n", (int)tr_kernel_for(v[0], v[1], v[2], 256, (int)v[3], v[4], v[5]));
  }
}
