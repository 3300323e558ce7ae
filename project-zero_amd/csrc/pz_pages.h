// pz_pages.h -- where a position of a sequence lies in a paged cache, and how
// many positions and nodes a sequence has.  Plain integer arithmetic, for the
// kernels and for a test of it without a device.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define PZ_HD __host__ __device__ __forceinline__
#else
#define PZ_HD inline
#endif

struct PzPages {
  int n_blocks, shift;  // pages, log2(block_size)
  int max_blocks;       // entries of a sequence's table
};

// Committed positions of a sequence whose length reads `len`.
PZ_HD int pz_pages_len(const PzPages& P, int len) {
  const int most = P.max_blocks << P.shift;
  return len < 0 ? 0 : (len < most ? len : most);
}

// Slot of position p, whose table entry reads `page`, in *slot; false, and a slot
// of page 0, where that is no page of the cache.
PZ_HD bool pz_pages_slot(const PzPages& P, int32_t page, int p, int64_t* slot) {
  const bool ok = (uint32_t)page < (uint32_t)P.n_blocks;
  *slot = ((int64_t)(ok ? page : 0) << P.shift) + (p & ((1 << P.shift) - 1));
  return ok;
}

// Entries of a list that reads n where T is the most (a count, or the nodes of
// a sequence).
PZ_HD int pz_pages_most(int n, int T) { return n < 0 ? 0 : (n < T ? n : T); }
