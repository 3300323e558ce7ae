// pz_prefixplan.h -- which kernel a call of prefix attention takes (host only).
#pragma once
#include <stdint.h>

enum PfKernel {
  PF_FEW,   // k_prefix, 16 rows of a prefix a workgroup
  PF_SOME,  // k_prefix, 32
  PF_WIDE   // k_prefix_wide, 256
};

// rows: of a key head, of the sequences of a prefix on average (at least a sequence's);
// heads: prefixes with a sequence x key heads; tiles: of 32 keys, of the longest prefix's
// table; D: head_dim; ld: elements between slots; shift: log2(block_size).
inline PfKernel pf_kernel_for(int64_t rows, int64_t heads, int64_t tiles, int n_cu, int D, long ld,
                              int shift) {
  if (rows <= 16) return PF_FEW;
  if (D < 256 && rows > 64 && (heads >= n_cu || heads * tiles >= 16 * (int64_t)n_cu) &&
      ld < (1 << 26) && (int64_t)ld << (shift + 1) <= UINT32_MAX)
    return PF_WIDE;
  return PF_SOME;
}
