// The 8-bit LM head's tile for calls of B batch rows and V ids, one per argument
// pair; first the number of tiles.  After "odd": those of rows off 16 bytes.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "pz_lmtile.h"

int main(int argc, char** argv) {
  const bool odd = argc > 1 && !std::strcmp(argv[1], "odd");
  std::printf("%d\n", odd ? I8_ODD_COUNT : I8_TILE_COUNT);
  for (int a = 1 + odd; a + 1 < argc; a += 2)
    std::printf("%d\n", (odd ? i8_odd_tile_for : i8_tile_for)(std::atoi(argv[a + 1]),
                                                               std::atoi(argv[a]), 256));
}
