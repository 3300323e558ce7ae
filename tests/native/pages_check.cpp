// Slots of a paged cache (pz_pages.h): every position against a table walked
// position by position, page numbers outside the cache, lengths and counts
// outside their range, and offsets past 32 bits.
#include <climits>
#include <cstdio>

#include "pz_pages.h"

int main() {
  int bad = 0;
  auto check = [&](bool ok, const char* what, long at) {
    if (!ok) {
      bad++;
      std::printf("BAD %s at %ld\n", what, at);
    }
  };
  const int32_t table[6] = {3, 0, -1, 6, 7, INT_MIN};
  for (int shift = 3; shift <= 6; shift++) {
    const PzPages P = {7, shift, 6};
    const int size = 1 << shift;
    for (int page = 0; page < 6; page++)
      for (int i = 0; i < size; i++) {
        const int p = page * size + i;
        int64_t slot = -1;
        const bool ok = pz_pages_slot(P, table[p >> shift], p, &slot);
        check(ok == (table[page] >= 0 && table[page] < 7), "validity", p);
        check(slot == (int64_t)(ok ? table[page] : 0) * size + i, "slot", p);
        check(slot >= 0 && slot < 7 * (int64_t)size, "a slot of the cache", p);
      }
    check(pz_pages_len(P, -5) == 0 && pz_pages_len(P, 0) == 0, "no length", shift);
    check(pz_pages_len(P, 6 * size - 1) == 6 * size - 1, "length", shift);
    check(pz_pages_len(P, 6 * size) == 6 * size, "full length", shift);
    check(pz_pages_len(P, 6 * size + 1) == 6 * size, "length past the table", shift);
    check(pz_pages_len(P, INT_MAX) == 6 * size, "largest length", shift);
  }
  // the last page of a cache of 2^31 - 1 pages of 64: past 32 bits
  const int32_t far[1] = {INT_MAX - 1};
  const PzPages F = {INT_MAX, 6, 1};
  int64_t slot = 0;
  check(pz_pages_slot(F, far[0], 63, &slot) && slot == (int64_t)(INT_MAX - 1) * 64 + 63, "far", 63);
  check(pz_pages_most(-1, 5) == 0 && pz_pages_most(0, 5) == 0 && pz_pages_most(4, 5) == 4 &&
            pz_pages_most(6, 5) == 5,
        "counts", 5);
  return bad != 0;
}
