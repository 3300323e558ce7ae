// The 8-bit LM head's tile for calls of B batch rows and V ids, one per argument
// pair; first the number of tiles.
#include <cstdio>
#include <cstdlib>

#include "pz_lmtile.h"

int main(int argc, char** argv) {
  std::printf("%d\n", I8_TILE_COUNT);
  for (int a = 1; a + 1 < argc; a += 2)
    std::printf("%d\n", i8_tile_for(std::atoi(argv[a + 1]), std::atoi(argv[a]), 256));
}
