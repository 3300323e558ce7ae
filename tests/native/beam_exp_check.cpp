// The exponential of beam selection (pz_beamexp.h) against the long double one: every table
// entry, the ends of each piece and points between, over the whole range; how far it is off at
// most, in units of 2^-43, goes to the output.  An argument plants a mistake (a table entry
// by its last 8 bits, or a coefficient's) in a copy, which has to be seen.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "pz_beamexp.h"

static be_u32x2 table[32];

static double worst = 0.0, worst_at = 0.0;
static void look(double d) {
  const long double want = expl((long double)d), got = be_add_exp(0.0, d, table);
  const double off = (double)fabsl(got / want - 1.0L);
  if (!(off <= worst)) worst = off, worst_at = d;
}

int main(int argc, char** argv) {
  const int entry = argc > 1 ? std::atoi(argv[1]) : -1;  // planted
  for (int i = 0; i < 32; i++) {
    const uint64_t v = be_roots[i] + (i == entry ? 1ull << 9 : 0ull);
    std::memcpy(&table[i], &v, 8);
    // the definition: 2^(i / 32), rounded once
    uint64_t bits;
    const double root = (double)powl(2.0L, i / 32.0L);
    std::memcpy(&bits, &root, 8);
    if (bits - ((uint64_t)i << 47) != be_roots[i]) {
      std::printf("BAD entry %d\n", i);
      return 1;
    }
  }
  uint64_t state = 12345;
  auto random = [&]() {  // [0, 1)
    state = state * 6364136223846793005ull + 1442695040888963407ull;
    return (double)(state >> 11) * 0x1p-53;
  };
  const double step = std::log(2.0) / 32.0;
  for (int n = -32315; n <= 32315; n++)  // every piece: its middle, its ends, points between
    for (int j = 0; j < 12; j++) {
      const double f = j < 3 ? 0.5 * (j - 1) : random() - 0.5;
      const double d = (n + f) * step;
      if (std::fabs(d) <= 700.0) look(d);
    }
  for (int i = 0; i < 4000000; i++) look((random() - 0.5) * 1400.0);
  for (int i = 0; i < 1000000; i++) look((random() - 0.5) * 40.0);
  look(0.0), look(700.0), look(-700.0), look(-650.0), look(500.0);
  // differences of floats, what lies far below counts as 10^-304, a NaN stays
  for (int i = 0; i < 1000000; i++) {
    const float m = (float)(random() * 60.0 - 30.0), x = m - (float)(random() * 30.0);
    const double got = be_exp(x, m, table);
    const long double want = expl((long double)x - (long double)m);
    const double off = (double)fabsl(got / want - 1.0L);
    if (!(off <= worst)) worst = off, worst_at = x - m;
  }
  const double least = be_exp(-3.0e38f, 3.0e38f, table);
  const double none = be_exp(-__builtin_inff(), 1.0f, table);
  const double nan = be_exp(__builtin_nanf(""), 1.0f, table);
  if (!(least > 0.0 && least < 1e-303 && none == least && std::isnan(nan))) {
    std::printf("BAD ends\n");
    return 1;
  }
  std::printf("%.6f at %.17g\n", worst * 0x1p43, worst_at);
  return 0;
}
