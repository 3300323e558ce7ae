// The rotation's largest calls (pz_refuse.h): which of its two kernels takes them, and that
// neither is launched with more threads than 32 bits count.
#include <cstdio>

#include "pz_refuse.h"

int main() {
  alignas(16) static uint16_t h[64];
  static float f[8];
  static int32_t pos[1];
  int bad = 0;
  auto check = [&](bool ok, const char* what, long n, int heads) {
    if (!ok) bad++;
    std::printf("%s %s: %ld tokens, %d heads\n", ok ? "ok " : "BAD", what, n, heads);
  };
  const int many[] = {1, 2, 3, 5, 40, 65536};
  for (int heads : many) {
    const long most = ((1L << 26) - 1) / heads;
    for (long n = most + 2; n > most - 6; n--) {
      pz_qk_rope r = {PZ_BF16, heads, 0, 8, nullptr, nullptr, 0.0f, 8, PZ_ROPE_HALVES, f, 1.0f};
      const bool taken = pz_refuse_rope(&r, h, 8L * heads, nullptr, 0, h, 8L * heads, nullptr, 0,
                                        (int)n, pos).code == PZ_OK;
      check(taken == (n <= most), "taken", n, heads);
      if (!taken) continue;
      // a wave for each head: workgroups of four, or of one
      const bool fours = pz_rope_in_fours((int)n, heads);
      const int64_t waves = (int64_t)n * heads;
      const int64_t threads = fours ? (waves + 3) / 4 * 256 : waves * 64;
      check(threads <= (int64_t)UINT32_MAX, "threads", n, heads);
      check(fours == (waves <= (1L << 26) - 4), "in fours", n, heads);
    }
  }
  return bad != 0;
}
