// The sizes that the 8-bit LM head refuses (pz_refuse.h), and the workgroups of
// its launches (pz_lmtile.h), which are counted in 64 bits.
#include <cstdint>
#include <cstdio>

#include "pz_lmtile.h"
#include "pz_refuse.h"

static int bad = 0;
static void expect(const char* what, bool ok) {
  if (!ok) bad++;
  std::printf("%s %s\n", ok ? "ok " : "BAD", what);
}

int main() {
  alignas(16) static int8_t w[64];
  alignas(16) static float f[16];
  auto code = [&](int V) { return pz_refuse_i8(w, f, V, 1, w, f, 4, 1, 4).code; };
  expect("2^30 ids", code(1 << 30) == PZ_OK);
  expect("one more", code((1 << 30) + 1) == PZ_ERANGE);
  expect("the largest int", code(INT32_MAX) == PZ_ERANGE);
  expect("one row of one tile", i8_workgroups(1, 1, 16, 16) == 8);
  expect("128256 x 256 in tiles of 256", i8_workgroups(128256, 256, 256, 256) == 504);
  expect("batches in blocks", i8_workgroups(129, 300, 128, 128) == 8 * 3);
  expect("2^30 ids in tiles of 32", i8_workgroups(1 << 30, 1, 32, 16) == 1 << 25);
  expect("past 32 bits", i8_workgroups(1 << 30, 1 << 20, 16, 16) == (int64_t)1 << 42);
  expect("a launch of them all", !pz_launch_fits(i8_workgroups(1 << 30, 1, 32, 16), 256));
  expect("a launch that fits", pz_launch_fits(i8_workgroups(1 << 25, 1, 32, 16), 128));
  return bad != 0;
}
