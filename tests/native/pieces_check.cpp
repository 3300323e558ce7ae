// The walk over positions' pieces (pz_pages.h): against numbers counted one by one, and in
// pages whose pieces' numbers pass 32 bits.
#include <cstdio>
#include <initializer_list>

#include "pz_pages.h"

int main() {
  int bad = 0;
  auto check = [&](bool ok, const char* what, long at) {
    if (!ok && bad++ < 20) std::printf("BAD %s at %ld\n", what, at);
  };
  for (int row : {8, 9, 31, 96, 2048})
    for (int step : {1, 7, 8, 256, 1000, 16384})
      for (int from : {0, 1, 255, 300, 16383}) {
        PzPieces w(row, from, step);
        for (long i = from; i < 40000; i += step, w.next())
          check(w.p == i / row && w.j == i % row, "piece", i);
      }
  // the steps that the kernels take, through pages of up to 2^30 positions: 2^33 pieces
  struct {
    int row, positions;
  } far[] = {{144, (1 << 24) - 5}, {128, (1 << 24) + 1}, {16384, (1 << 19) + 3}, {8, (1 << 30) - 1},
             {128, 1 << 26}};
  for (const auto& f : far)
    for (int from : {0, 16383}) {
      PzPieces w(f.row, from, 16384);
      const int64_t all = (int64_t)f.row * f.positions;
      int64_t i = from;
      for (; w.p < f.positions; i += 16384, w.next()) {
        check(i < all, "an end", f.row);
        if (i >= all) break;
        check(w.p >= 0 && w.j >= 0 && w.j < f.row && (int64_t)w.p * f.row + w.j == i, "far piece",
              (long)i);
      }
      check(i >= all, "the last piece", f.row);
    }
  return bad != 0;
}
