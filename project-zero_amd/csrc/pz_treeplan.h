// pz_treeplan.h -- which kernel a call of tree attention takes (host only).
#pragma once
#include <stdint.h>

enum TrKernel {
  TR_FEW_SHORT,  // k_tree, 16 rows, eight waves, no splits
  TR_FEW,        // k_tree, 16 rows, four waves
  TR_SOME,       // k_tree, 32 rows, four waves
  TR_WIDE16,     // k_tree_wide, 16 rows a wave
  TR_WIDE32      // k_tree_wide, 32 rows a wave
};

// rows: nodes x group; heads: sequences x key heads; tiles: of 32 keys, of the longest
// table and its nodes; D: head_dim; ld, ld_n: elements between slots, between nodes.
//
// Up to 16 rows, few short sequences: eight waves and no launch to join.  (One token
// over 500 positions 11.5 us, 12.0 in splits of four waves, 16 sequences 12.7 / 15.1;
// but over 1000 15.1 / 11.8, and 512 key heads 34.0 / 29.9.)  Heads of 256 spill
// there: 500 positions 20.2 us, in splits 16.1.
//
// The wide kernel (us, narrow / wide of 16 rows a wave / of 32):
//   32 ragged sequences of up to 4096 positions x 8 key heads: 20 rows 73 / 74; 32
//   74 / 76; 48 97 / 78 / 90; 64 - / 78 / 90; 96 - / 95 / 90; 128 - / 105 / 91; 256 -
//   / 181 / 142: from 33 rows on, and 16 a wave while each has a SIMD.
//   256 rows, 8 sequences x 8 key heads, by positions: 500 22 / - / 38; 1000 31 / -
//   / 40; 2000 51 / - / 50; 4000 96 / - / 73; one sequence 2000 18 / - / 25, 8000 33
//   / - / 34, 16000 49 / - / 41; 48 rows 8000 16 / 17, 32768 41 / 36: from 16
//   tiles a CU on, below which k_tree's row blocks fill more CUs; but with a
//   workgroup for each CU at once (32 x 8) 100 47 / - / 35, 48 rows 250 17 / 15.
// Its offsets within a load's rows (7 slots, 63 nodes) are 32 bits, and heads of 256
// do not fit its registers.
inline TrKernel tr_kernel_for(int64_t rows, int64_t heads, int64_t tiles, int n_cu, int D,
                              long ld, long ld_n) {
  if (rows <= 16) return D < 256 && tiles <= 24 && heads <= n_cu ? TR_FEW_SHORT : TR_FEW;
  if (D < 256 && rows > 32 && (heads >= n_cu || heads * tiles >= 16 * (int64_t)n_cu) &&
      ld < (1 << 26) && ld_n < (1 << 24))
    return rows <= 64 ? TR_WIDE16 : TR_WIDE32;
  return TR_SOME;
}
