// pz_prefixplan.h -- which kernel a call of prefix attention takes, and in how many splits
// (host only).
#pragma once
#include <stdint.h>

#include <algorithm>

enum PfKernel {
  PF_FEW,   // k_prefix, 16 rows of a prefix a workgroup
  PF_SOME,  // k_prefix, 32
  PF_WIDE   // k_prefix_wide, 256
};
constexpr int PF_ROWS = 256;

// rows: of a key head, of the sequences of a prefix on average (at least a sequence's);
// heads: prefixes with a sequence x key heads; tiles: of 32 keys, of the longest prefix's
// table; own: sequences x key heads; D: head_dim; ld: elements between slots; shift:
// log2(block_size).
//
// Few rows: one tile of rows where it holds them (1 prefix of 4096 positions, rows 16:
// 16.4 us, 17.5 in tiles of 32; 8 prefixes, rows 32: 47.1, 42.2).
// The wide kernel where either of its parts has enough to do (us as it is / without it; 32
// heads over 8, 128 elements, 64 positions of one's own):
//   many sequences, each with a wave of its own: prefixes x sequences x positions
//     32 x 8 x 256 41 / 44, 16 x 8 x 4096 73 / 70, 1 x 128 x 4096 39 / 41, 8 x 24 x 2048
//     43 / 53, 1 x 256 x 4096 51 / 71, 32 x 64 x 256 235 / 299; 1 x 64 x 4096 would be 32 / 27,
//     and with 16 rows 256 x 4 x 256 192 / 185;
//   long prefixes of more than 64 rows: 1 x 24 x 32768 60 / 72, 1 x 64 x 32768 70 / 106, 1 x
//     64 x 16384 57 / 57; 1 x 64 x 8192 would be 42 / 35, 1 x 16 x 32768 58 / 46.
inline PfKernel pf_kernel_for(int64_t rows, int64_t heads, int64_t tiles, int64_t own, int n_cu,
                              int D, long ld, int shift) {
  if (rows <= 16) return PF_FEW;
  const int64_t work = heads * ((rows + PF_ROWS - 1) / PF_ROWS) * tiles;
  // (its registers hold heads of up to 128; offsets within a page's four bytes)
  if (D < 256 && (own >= 4 * (int64_t)n_cu || (rows > 64 && work >= 16 * (int64_t)n_cu)) &&
      ld < (1 << 26) && (int64_t)ld << (shift + 1) <= UINT32_MAX)
    return PF_WIDE;
  return PF_SOME;
}

// Splits of the prefixes' part in k_prefix_wide, a workgroup of which has a CU to itself: wgs
// workgroups over `tiles` tiles of 32 keys, `most` splits at most.  Time in tiles (of 256
// rows, 0.95 us): a workgroup takes its share of the prefix's and six more (its queries' and
// first keys' way in, its results' way out); the sequences' own part, `others` tiles of one CU
// in all, comes after it, fills the CUs that it leaves and has a way of 18 at least.  (As many
// as there are CUs for instead, us before / so: 16 prefixes of 16384 positions x 12 sequences
// 335 / 208, 8 of 16384 x 16 142 / 117, 1 of 2048 x 512 80 / 70, 1 of 131072 x 20 128 / 113, 1
// of 4096 x 256 58 / 51; 1 of 32768 x 256 alike.)
inline int pf_wide_splits(int n_cu, int64_t wgs, int64_t tiles, int64_t others, int64_t most) {
  int64_t best = 1, least = INT64_MAX;
  for (int64_t S = 1; S <= most; S++) {
    const int64_t k = wgs * S, one = (tiles + S - 1) / S + 6;
    const int64_t t = std::max((k + n_cu - 1) / n_cu * one, (k * one + others) / n_cu + 18);
    if (t < least) best = S, least = t;
  }
  return (int)best;
}
