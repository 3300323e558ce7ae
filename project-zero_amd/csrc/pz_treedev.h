// pz_treedev.h -- attention of few rows a sequence over a paged cache: the kernels
// that pz_tree_attention and pz_prefix_attention share.
//
//   out[r] = sum_p softmax_p(scale q[r] . k[p]) v[p],  r = (node, head of a key
//   head's group), p over the cached positions and the nodes that r's node sees.
//
// One pass over the keys with a running maximum m and sum l per row.  m is a score
// q . k itself and weights are 2^(c (s - m)), c = scale log2(e): the difference of
// floats that lie close is exact, and the largest score's weight with it, wherever
// fp32 holds the scores.  (One fma(s, c, -c m) moves the weights by half a unit of
// c m, alike for every key of a tile, but from 2^26 on that is 2^8 and more.)  k_tree,
// which memory bounds, always subtracts; k_tree_wide takes the fma where |c m| is at
// most 2^12, half a unit 2^-12 (8 x 64 nodes over 32768 positions: 333 us with the fma
// alone, 336 so, 347 with the difference alone; in k_tree the choice costs heads of
// 256 registers that they lack, 32 ragged x 5 nodes 148 us for 125).  All rows of a key head
// share its keys, so nodes x group rows meet each tile of 32 keys: 16 of them a
// column of v_mfma_f32_16x16x32.  Both kernels compute
//
//   * S^T = K Q^T: A = 16 keys x 32 d, lane l: key l % 16, 8 d from 8 (l / 16).
//     D gives lane l row l % 16 and keys 4 (l / 16) .. +3 of each 16: with two
//     key tiles the 8 weights of one k group of the next product, whose key
//     order (16 t + 4 g + i) V then follows.
//   * O^T = V^T P^T: lane l loads D / 16 neighbouring values of each of its 8
//     keys (l / 16's) from d = (l % 16) D / 16: whole rows of V; a byte permute
//     gathers the 8 keys of one d.  D's rows are d, its columns the rows of q, so
//     m, l and the rescaling are a lane's own.  The weights are rounded to the
//     values' 16 bits for this product; their sum l takes them before it.
//   * m is raised only when a score passes it by 2^TH: the weights stay below
//     2^(TH + OFF), and the cross-lane maximum and the rescaling drop out of
//     most tiles.
//
// k_tree, up to 32 rows or little work: a workgroup owns 16 RT rows of one key head of one
// sequence and a range of its keys; its waves take tiles in turn, each with its
// own m, l and result, which meet in LDS at the end.  Keys and values go from
// memory to registers, with no barrier on the way.  Bound by memory: 32 ragged
// sequences of up to 4096 positions (272 MB), 5 nodes, 32 heads over 8 of 128:
// 73 us, 3.7 TB/s; 55 us (4.9 TB/s) where all are of 2048, since one workgroup a
// CU waits for the longest.
//
// k_tree_wide, many rows over many keys: the waves of a workgroup own 16 RT rows each and share
// the keys, whose tiles come to LDS through a ring of loads.  Bound by issue: 8 x
// 64 nodes over 32768 positions 337 us (275 GFLOP at 0.82 PFLOP/s, 3.2 TB/s of
// keys and values).  Of a tile's 1.3 us a SIMD's two waves take 0.5 for the
// products, 0.6 for the other vector instructions, and LDS 0.55 for the fragments
// and the loads; before the fragments were read a phase ahead it was 363 us, 257 of
// it without loads and barriers.
//
// Few rows and long sequences: the keys are split over S workgroups, whose
// results k_tree_join adds up.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/pz_sampler.h"
#include "pz_device.h"
#include "pz_lmdev.h"
#include "pz_pages.h"

namespace {

typedef uint32_t tr_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t tr_u32x2 __attribute__((ext_vector_type(2)));
typedef float tr_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 tr_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 tr_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 tr_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 tr_f16x2 __attribute__((ext_vector_type(2)));

constexpr int TR_KEYS = 32;         // keys of a tile
constexpr int TR_SHARE = 8;         // tiles that are worth a workgroup
constexpr int TR_ENTRIES = 2048;    // table entries that the wide kernel keeps in LDS
constexpr int TR_STAGES = 6;        // tiles of its ring
constexpr int TR_WIDE = 8;          // its waves
constexpr float TR_LOW = -3.40282346638528859812e38f;  // m before any score (the least float:
                                                       // m - m is 0, and no score lies below)
constexpr float TR_NEAR = 4096.0f;  // largest |c m| whose rounding is none of a weight's business
constexpr float TR_LOG2E = 1.44269504088896340736f;

template <int TYPE>
struct TrType;
template <>
struct TrType<PZ_BF16> {
  // the weights lie around 2^-40, so that the sums of any 2^31 of them times bf16's
  // largest values stay in fp32 (which has as many exponents: down there the small
  // ones keep their bits to 2^-86 of the largest)
  static constexpr float OFF = -40.0f, TH = 8.0f, MUCH = 0x1p-32f;  // 2^(TH + OFF)
  static constexpr uint32_t EXP = 0x7f80u;  // exponent bits of one element
  static constexpr float MOST = 3.38953138925153547590e38f;  // its largest
  __device__ __forceinline__ static tr_f32x4 mfma(tr_u32x4 a, tr_u32x4 b, tr_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(tr_bf16x8, a),
                                                   __builtin_bit_cast(tr_bf16x8, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static uint32_t pack(float x, float y) {
    const tr_bf16x2 v = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, v);
  }
  __device__ __forceinline__ static float widen(uint16_t h) {
    return __uint_as_float((uint32_t)h << 16);
  }
};
template <>
struct TrType<PZ_F16> {
  // the weights lie around 2^8, so that the small ones of a long sequence keep
  // their bits (fp16 has normal numbers down to 2^-14)
  static constexpr float OFF = 8.0f, TH = 6.0f, MUCH = 0x1p14f;
  static constexpr uint32_t EXP = 0x7c00u;
  static constexpr float MOST = 65504.0f;
  __device__ __forceinline__ static tr_f32x4 mfma(tr_u32x4 a, tr_u32x4 b, tr_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(tr_f16x8, a),
                                                  __builtin_bit_cast(tr_f16x8, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static uint32_t pack(float x, float y) {
    const tr_f16x2 v = {(_Float16)x, (_Float16)y};
    return __builtin_bit_cast(uint32_t, v);
  }
  __device__ __forceinline__ static float widen(uint16_t h) {
    return (float)__builtin_bit_cast(_Float16, h);
  }
};

struct TreeArgs {
  const uint16_t* k;
  const uint16_t* v;
  long ld;
  PzPages pages;
  const int32_t* blocks;  // [B, pages.max_blocks]
  const int32_t* len;
  const uint16_t* kn;
  const uint16_t* vn;
  long ld_n;
  int B, T;
  const int32_t* n_nodes;
  const uint64_t* tree;
  int n_kv, group;  // key heads, query heads of each
  float c;          // scale * log2(e)
  const uint16_t* q;
  long ld_q;
  uint16_t* out;
  long ld_out;
  int S, nblk;  // most splits of a sequence, row blocks of a key head
  int chunk;    // tiles of a split of the longest table
  float* part;  // [unit][S] results (a lane's order), then their m and l
  float* ml;
};

// What a launch works on: whole rows of attention (TreeArgs); the part of them that
// is each sequence's own, its cache and its nodes; or the part of a prefix that
// sequences share, whose rows then are those of all these sequences together.
// Parts leave results, m and l row by row: row (b T + t) heads + head, in slot
// `slot` + split of [slots][R].
enum TrWhat { TR_WHOLE, TR_OWN, TR_SHARED };
struct WholeArgs : TreeArgs {
  static constexpr TrWhat WHAT = TR_WHOLE;
};
struct PartArgs : TreeArgs {
  size_t R;  // rows: B T heads
  int slot;
};
struct OwnArgs : PartArgs {
  static constexpr TrWhat WHAT = TR_OWN;
};
// (B, pages, blocks and len are the prefixes'; nblk is the row blocks of all of them)
struct SharedArgs : PartArgs {
  static constexpr TrWhat WHAT = TR_SHARED;
  const int32_t* first;  // [B + 1] sequences, nullptr: `each` of them to a prefix
  int each;
  int run;     // row blocks of a prefix
  int b0, nb;  // the launch takes nb sequences from b0 on, where q and the results begin
};

__device__ __forceinline__ int tr_nodes(const TreeArgs& A, int b) {
  return A.n_nodes ? pz_pages_most(A.n_nodes[b], A.T) : A.T;
}

__device__ __forceinline__ int tr_tiles(const SharedArgs& A, int i) {
  return (pz_pages_len(A.pages, A.len[i]) + TR_KEYS - 1) / TR_KEYS;
}

__device__ __forceinline__ int tr_tiles(const TreeArgs& A, int b) {
  return (pz_pages_len(A.pages, A.len[b]) + TR_KEYS - 1) / TR_KEYS +
         (tr_nodes(A, b) + TR_KEYS - 1) / TR_KEYS;
}

// Tiles of a split: a share of the longest sequence's, which tables that are kept
// larger do not change (A.chunk: the longest table's, the most that it can be).
// (Tables of 32768 positions, us by the table / by the longest sequence: one token
// over 2000 17.7 / 12.4, 8 sequences x 64 nodes over 4000 141 / 64; tight tables the
// same within 0.5.)
template <class ARGS>
__device__ __forceinline__ int tr_chunk(const ARGS& A, int b, int lane) {
  if (A.S == 1) return A.chunk;
  int most;
  if (A.B == 1) {
    most = tr_tiles(A, b);
  } else {
    most = 0;
    for (int i = lane; i < A.B; i += 64) {
      const int n = tr_tiles(A, i);
      most = n > most ? n : most;
    }
    // the wave's maximum in lane 63: within 16 lanes, then over them
    auto step = [&](int o) { most = o > most ? o : most; };
    step(__builtin_amdgcn_update_dpp(0, most, 0x111, 0xf, 0xf, true));  // lane - 1
    step(__builtin_amdgcn_update_dpp(0, most, 0x112, 0xf, 0xf, true));  // lane - 2
    step(__builtin_amdgcn_update_dpp(0, most, 0x114, 0xf, 0xf, true));  // lane - 4
    step(__builtin_amdgcn_update_dpp(0, most, 0x118, 0xf, 0xf, true));  // lane - 8
    step(__builtin_amdgcn_update_dpp(0, most, 0x142, 0xa, 0xf, true));  // row 0's and 2's last to 1, 3
    step(__builtin_amdgcn_update_dpp(0, most, 0x143, 0xc, 0xf, true));  // lane 31 to rows 2, 3
    most = __builtin_amdgcn_readlane(most, 63);
  }
  const int share = (most + A.S - 1) / A.S;
  return share < TR_SHARE ? TR_SHARE : share;
}

// One over the sum l of the weights of node t's row.  A sum of 0 is a row that attends
// nothing, whose result is zeros, or one whose every score is -infinity, which is NaN.
__device__ __forceinline__ float tr_inverse(const TreeArgs& A, int b, int t, float l) {
  if (l != 0.0f) return 1.0f / l;
  const uint64_t sees = A.tree ? A.tree[(size_t)b * A.T + t] : ~0ull;
  if (sees << (64 - tr_nodes(A, b))) return __builtin_nanf("");
  const int ctx = pz_pages_len(A.pages, A.len[b]);
  for (int e = 0; (int64_t)e << A.pages.shift < ctx; e++)
    if ((uint32_t)A.blocks[(size_t)b * A.pages.max_blocks + e] < (uint32_t)A.pages.n_blocks)
      return __builtin_nanf("");
  return 0.0f;
}

// How many of the launch's sequences have prefix i, from *lo on.
__device__ __forceinline__ int tr_sharers(const SharedArgs& A, int i, int* lo) {
  int f = A.first ? A.first[i] : i * A.each, e = A.first ? A.first[i + 1] : f + A.each;
  f = f > A.b0 ? f - A.b0 : 0;
  e = e > A.b0 ? e - A.b0 : 0;
  e = e < A.nb ? e : A.nb;
  *lo = f;
  return e > f ? e - f : 0;
}

// Where a workgroup works: key head h of sequence (or prefix) b, split sp, row block
// `blk` (of `per` times ROWS rows) of `rows`, which start at node node0.
struct TrJob {
  int b, h, sp, blk, rows, node0;
};
template <int ROWS>
__device__ __forceinline__ bool tr_job(const TreeArgs& A, uint32_t block, int lane, int n_blk,
                                       TrJob* J) {
  // the row blocks of one range of keys on one XCD, one after the other
  const int slot = block >> 3, turn = slot / n_blk;
  J->blk = slot - turn * n_blk;
  const int grp = turn * 8 + (block & 7);
  if (grp >= A.B * A.n_kv * A.S) return false;
  // (split by split, so that those that short sequences lack are spread over the
  // XCDs: 32 ragged sequences of up to 4096 positions in 4 splits 89 us, 75 so)
  const int units = A.B * A.n_kv;
  J->sp = grp / units;
  const int bh = grp - J->sp * units;
  J->h = bh % A.n_kv;
  J->b = bh / A.n_kv;
  J->rows = tr_nodes(A, J->b) * A.group;
  J->node0 = J->b * A.T;
  return J->blk * ROWS < J->rows;
}
// A prefix's row blocks (`run` of them; with ranges, on average) follow each other on one
// XCD.  Units of a run and a key head go to the XCDs in turn, split by split, and one further
// with every turn, so that splits that short prefixes lack leave no XCD idle (16 prefixes of
// 16384 positions x 16 sequences 196 us in the units' own order, an eighth to each XCD; 186
// so)
template <int ROWS>
__device__ __forceinline__ bool tr_job(const SharedArgs& A, uint32_t block, int lane, int n_blk,
                                       TrJob* J) {
  const int slot = block >> 3, turn = slot / A.run, unit = turn * 8 + ((block + turn) & 7);
  const int v = unit / A.n_kv, runs = (n_blk + A.run - 1) / A.run;
  J->h = unit - v * A.n_kv;
  J->sp = v / runs;
  int blk = (v - J->sp * runs) * A.run + (slot - turn * A.run);
  if (J->sp >= A.S || blk >= n_blk) return false;
  if (!A.first) {  // (as many row blocks each)
    const int each = ((A.each < A.nb ? A.each : A.nb) * A.T * A.group + ROWS - 1) / ROWS;
    int lo;
    J->b = blk / each;
    J->blk = blk - J->b * each;
    J->rows = tr_sharers(A, J->b, &lo) * A.T * A.group;
    J->node0 = lo * A.T;
    return J->blk * ROWS < J->rows;
  }
  for (int i0 = 0; i0 < A.B; i0 += 64) {
    int lo = 0, n = 0;
    if (i0 + lane < A.B) n = tr_sharers(A, i0 + lane, &lo);
    const int mine = (n * A.T * A.group + ROWS - 1) / ROWS;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      sum += lane >= o ? v : 0;
    }
    const uint64_t past = __ballot(sum > blk);
    if (past) {
      const int at = __ffsll((unsigned long long)past) - 1;
      J->b = i0 + at;
      J->blk = blk - __builtin_amdgcn_readlane(sum - mine, at);
      J->rows = __builtin_amdgcn_readlane(n, at) * A.T * A.group;
      J->node0 = __builtin_amdgcn_readlane(lo, at) * A.T;
      return true;
    }
    blk -= __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// What results taken against the maximum m count for against the maximum top.
__device__ __forceinline__ float tr_lift(float m, float top, float c) {
  return __builtin_amdgcn_exp2f((m - top) * c);
}

// A lane's results of one row: d = NT (4 g + i) + 4 f + 0..3 in o (i, f).  A mean of
// finite values does not pass the type's largest; the rounded weights, whose sum is
// taken before, can make it do so by 2^-11 (fp16) or 2^-8, which would be an infinity.
template <int TYPE>
__device__ __forceinline__ void tr_store4(uint16_t* o, tr_f32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; i++)
    v[i] = fabsf(v[i]) > TrType<TYPE>::MOST && fabsf(v[i]) < __builtin_inff()
               ? __builtin_copysignf(TrType<TYPE>::MOST, v[i])
               : v[i];
  tr_u32x2 w;
  w[0] = TrType<TYPE>::pack(v[0], v[1]);
  w[1] = TrType<TYPE>::pack(v[2], v[3]);
  *reinterpret_cast<tr_u32x2*>(o) = w;
}

// Four results of a row of a part, from d on, and (with the first four) its m and l.
template <int D>
__device__ __forceinline__ void tr_part(const PartArgs& A, int sp, size_t row, int d, tr_f32x4 v,
                                        float m, float l) {
  const size_t at = (size_t)(A.slot + sp) * A.R + row;
  *reinterpret_cast<tr_f32x4*>(A.part + at * D + d) = v;
  if (d == 0) {
    A.ml[2 * at] = m;
    A.ml[2 * at + 1] = l;
  }
}

// The running state of 16 RT rows in one wave, and the steps of one tile of keys.
// CHOOSE: weights by one fma where every |c m| is small, else always from s - m.
template <int TYPE, int D, int RT, bool CHOOSE>
struct TrRows {
  typedef TrType<TYPE> Y;
  static constexpr int KS = D / 32, NT = D / 16, NW = NT / 2;  // k steps, d tiles, words of V
  tr_f32x4 o[RT][NT];
  float mx[RT], l[RT];
  bool far;      // (CHOOSE) some row's |c m| is above TR_NEAR: s - m first (wave-uniform)
  float nb[RT];  // (CHOOSE) what the fma adds
  tr_f32x4 s[RT][2];  // scores, then weights: keys 16 t + 4 g + i of row m
  int m, g;
  float c;  // scale log2(e)

  __device__ __forceinline__ void clear(int lane, float scale) {
    m = lane & 15;
    g = lane >> 4;
    c = scale;
    far = true;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      mx[rt] = TR_LOW;
      nb[rt] = Y::OFF;
      l[rt] = 0.0f;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) o[rt][nt] = tr_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  // kf(t, ks): keys 16 t + m, 8 d from 32 ks + 8 g; qf(rt, ks): row m, the same d
  template <class K, class Q>
  __device__ __forceinline__ void scores(K kf, Q qf) {
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int t = 0; t < 2; t++) s[rt][t] = tr_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const tr_u32x4 a = kf(t, ks);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) s[rt][t] = Y::mfma(a, qf(rt, ks), s[rt][t]);
      }
  }
  // scores of keys that do not exist (`on`, bit e: key 16 (e / 4) + 4 g + e % 4) or
  // that the row does not see
  template <class F>
  __device__ __forceinline__ void drop(uint32_t on, F seen) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const bool there = on >> e & 1u;
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
        s[rt][e >> 2][e & 3] =
            there && seen(rt, 16 * (e >> 2) + 4 * g + (e & 3)) ? s[rt][e >> 2][e & 3]
                                                               : -__builtin_inff();
    }
  }
  // what lies in the place of a key that does not exist may be anything
  __device__ __forceinline__ static void blank(uint32_t on, uint32_t (&vr)[8][NW]) {
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int i = 0; i < NW; i++) vr[e][i] = on >> e & 1u ? vr[e][i] : 0u;
  }
  // the largest score of each row tile in this lane (a NaN stays: its row's result is
  // one, and the plain maximum would first quiet every operand)
  __device__ __forceinline__ static float most(float a, float b) {
    return __builtin_elementwise_maximum(a, b);
  }
  __device__ __forceinline__ static void tops(const tr_f32x4 (&s)[RT][2], float (&tm)[RT]) {
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
      tm[rt] = most(most(most(s[rt][0][0], s[rt][0][1]), most(s[rt][0][2], s[rt][0][3])),
                    most(most(s[rt][1][0], s[rt][1][1]), most(s[rt][1][2], s[rt][1][3])));
  }
  // raises m where a score passes it by 2^TH, and readies the scores for their weights
  __device__ __forceinline__ void raise(const float (&tm)[RT]) {
    bool up = false;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) up |= (tm[rt] - mx[rt]) * c > Y::TH;
    if (__ballot(up)) {
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        float t = tm[rt];
        t = fmaxf(t, __shfl_xor(t, 16, 64));
        t = fmaxf(t, __shfl_xor(t, 32, 64));
        const float mn = fmaxf(mx[rt], t);
        const float al = tr_lift(mx[rt], mn, c);
        mx[rt] = mn;
        l[rt] *= al;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) o[rt][nt] *= al;
      }
      if (CHOOSE) {
        bool out = false;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) out |= !(fabsf(mx[rt] * c) <= TR_NEAR);
        far = __ballot(out) != 0;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) nb[rt] = far ? Y::OFF : Y::OFF - mx[rt] * c;
      }
    }
    if (CHOOSE && far)
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int e = 0; e < 8; e++) s[rt][e >> 2][e & 3] -= mx[rt];
  }
  // weight e of row tile rt from its score, which raise() has seen
  __device__ __forceinline__ void weigh(int rt, int e) {
    const float d = CHOOSE ? s[rt][e >> 2][e & 3] : s[rt][e >> 2][e & 3] - mx[rt];
    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(d, c, CHOOSE ? nb[rt] : Y::OFF));
    s[rt][e >> 2][e & 3] = p;
    l[rt] += p;
  }
  __device__ __forceinline__ void weights() {
    float tm[RT];
    tops(s, tm);
    raise(tm);
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int e = 0; e < 8; e++) weigh(rt, e);
  }
  // the weights as the next product takes them
  __device__ __forceinline__ void pack(tr_u32x4 (&pf)[RT]) const {
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        pf[rt][j] = Y::pack(s[rt][j >> 1][2 * (j & 1)], s[rt][j >> 1][2 * (j & 1) + 1]);
  }
  // adds the values of one d tile: v[e] the word of key e that holds d tile nt, high
  // its upper half
  __device__ __forceinline__ void value(int nt, const uint32_t (&v)[8], bool high,
                                        const tr_u32x4 (&pf)[RT]) {
    tr_u32x4 vt;
#pragma unroll
    for (int j = 0; j < 4; j++)
      vt[j] = __builtin_amdgcn_perm(v[2 * j + 1], v[2 * j], high ? 0x07060302u : 0x05040100u);
#pragma unroll
    for (int rt = 0; rt < RT; rt++) o[rt][nt] = Y::mfma(vt, pf[rt], o[rt][nt]);
  }
  // vr: values of the 8 keys of `on`'s bits, NT d from NT m
  __device__ __forceinline__ void values(const uint32_t (&vr)[8][NW]) {
    tr_u32x4 pf[RT];
    pack(pf);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      uint32_t v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = vr[e][nt >> 1];
      value(nt, v, nt & 1, pf);
    }
  }
  // A value that is not finite must reach the rows that see its node and no other
  // (0 * NaN is NaN): such nodes leave the product and are added row by row.  vn:
  // the tile's first node's values, ps: LDS for [16 RT][TR_KEYS + 1] weights.
  __device__ __forceinline__ void odd_values(uint32_t (&vr)[8][NW], const uint64_t (&sees)[RT],
                                             const uint16_t* vn, long ld_n, float* ps) {
    uint32_t odd = 0u;  // bit 4 e + g': key 16 (e / 4) + 4 g' + e % 4
#pragma unroll
    for (int e = 0; e < 8; e++) {
      bool nf = false;
#pragma unroll
      for (int i = 0; i < NW; i++)
        nf |= (vr[e][i] & Y::EXP) == Y::EXP || (vr[e][i] >> 16 & Y::EXP) == Y::EXP;
      const uint64_t any = __ballot(nf);
#pragma unroll
      for (int gg = 0; gg < 4; gg++)
        if (any >> (16 * gg) & 0xffffull) odd |= 1u << (4 * e + gg);
    }
    if (odd) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool z = odd >> (4 * e + g) & 1u;
#pragma unroll
        for (int i = 0; i < NW; i++) vr[e][i] = z ? 0u : vr[e][i];
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
          ps[(rt * 16 + m) * (TR_KEYS + 1) + 4 * e + g] = s[rt][e >> 2][e & 3];
      }
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // (one wave's own LDS)
#pragma clang loop unroll(disable)
      for (int j = 0; j < TR_KEYS; j++) {
        if (!(odd >> j & 1u)) continue;
        const int key = 16 * (j >> 4) + 4 * (j & 3) + (j >> 2 & 3);
        const uint16_t* vrow = vn + (size_t)key * ld_n + 4 * NT * g;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
          const float p = ps[(rt * 16 + m) * (TR_KEYS + 1) + j];
          if (!(sees[rt] >> key & 1ull)) continue;
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
              o[rt][nt][i] = __builtin_fmaf(p, Y::widen(vrow[NT * i + nt]), o[rt][nt][i]);
        }
      }
    }
  }
};

// LDS of tr_narrow.
template <int D, int RT, int WAVES>
struct TrLds {
  static constexpr int CH = RT * (D / 16);  // float4s of a lane's results
  static constexpr int QF = RT * (D / 32) * 1024, LDS_P = 16 * RT * (TR_KEYS + 1) * 4;
  // the waves' results meet HALF of them at a time
  static constexpr int HALF = RT > 1 && CH * WAVES > 64 ? 2 : 1;
  static constexpr int BUF = CH * 1024 / HALF;  // bytes of a wave's
  static constexpr int SH = WAVES * BUF > QF + WAVES * LDS_P ? WAVES * BUF : QF + WAVES * LDS_P;
  __align__(16) char sh[SH];
  float mls[WAVES][16 * RT][2];
};

// A workgroup of k_tree (thread tid of it, block its number), or with WAVES = 1 a wave by
// itself, whatever the others of its workgroup do.
template <int TYPE, int D, int RT, int WAVES, class ARGS>
__device__ __forceinline__ void tr_narrow(const ARGS& A, uint32_t block, int tid,
                                          TrLds<D, RT, WAVES>& lds) {
  typedef TrLds<D, RT, WAVES> Lds;
  constexpr int KS = D / 32, NT = D / 16, NW = NT / 2;  // k steps of S, d tiles, words of V
  constexpr int ROWS = 16 * RT, CH = Lds::CH, QF = Lds::QF, LDS_P = Lds::LDS_P, HALF = Lds::HALF,
                BUF = Lds::BUF;
  char* const sh = lds.sh;
  auto& mls = lds.mls;
  auto sync = [&]() {
    if constexpr (WAVES == 1) {
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  };
  const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  TrJob J;
  if (!tr_job<ROWS>(A, block, lane, A.nblk, &J)) return;
  const int b = J.b, h = J.h, sp = J.sp, rows = J.rows, row0 = J.blk * ROWS;
  const int node0 = J.node0;
  const int ctx = pz_pages_len(A.pages, A.len[b]),
            nn = ARGS::WHAT == TR_SHARED ? 0 : tr_nodes(A, b);
  const int nc = (ctx + TR_KEYS - 1) / TR_KEYS, ntl = nc + (nn + TR_KEYS - 1) / TR_KEYS;
  const int chunk = tr_chunk(A, b, lane);
  const int tl0 = sp * chunk, tl1 = ntl - tl0 < chunk ? ntl : tl0 + chunk;
  if (tl0 >= ntl) return;
  const int ns = (ntl + chunk - 1) / chunk;  // splits that this sequence has
  const int32_t* table = A.blocks + (size_t)b * A.pages.max_blocks;
  const uint16_t* kc = A.k + (size_t)h * D;
  const uint16_t* vc = A.v + (size_t)h * D;
  const uint16_t* kn = A.kn + (size_t)b * A.T * A.ld_n + (size_t)h * D;
  const uint16_t* vn = A.vn + (size_t)b * A.T * A.ld_n + (size_t)h * D;

  tr_u32x4 kf[2][KS];   // a tile's keys: 16 t + m, 8 d from 32 ks + 8 g
  uint32_t vr[8][NW];   // its values: keys 16 (e / 4) + 4 g + e % 4, NT d from NT m
  auto load_k = [&](int t, const uint16_t* p) {
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
      kf[t][ks] = *reinterpret_cast<const tr_u32x4*>(p + ks * 32 + 8 * g);
  };
  auto load_v = [&](int e, const uint16_t* p) {
    p += m * NT;
    if constexpr (NW == 2) {
      const tr_u32x2 x = *reinterpret_cast<const tr_u32x2*>(p);
      vr[e][0] = x[0];
      vr[e][1] = x[1];
    } else {
#pragma unroll
      for (int i = 0; i < NW; i += 4) {
        const tr_u32x4 x = *reinterpret_cast<const tr_u32x4*>(p + 2 * i);
#pragma unroll
        for (int c = 0; c < 4; c++) vr[e][i + c] = x[c];
      }
    }
  };
  // A tile of the cache: the pages of key 16 t + m (k[t]) and of keys 16 t + 4 g .. +3
  // (v[t]: four positions from a multiple of four share a page).  Positions past
  // the last: the last one's (or its four's) again.  The pages are looked at a
  // tile later, since waiting for them waits for every load before them.
  struct Pages {
    int32_t k[2], v[2];
  };
  auto pos_k = [&](int tl, int t) {
    const int p = tl * TR_KEYS + 16 * t + m;
    return p < ctx ? p : ctx - 1;
  };
  auto pos_v = [&](int tl, int t) {
    const int p = tl * TR_KEYS + 16 * t + 4 * g, last = (ctx - 1) & ~3;
    return p < last ? p : last;
  };
  auto pages_of = [&](int tl) {
    Pages f;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      f.k[t] = table[pos_k(tl, t) >> A.pages.shift];
      f.v[t] = table[pos_v(tl, t) >> A.pages.shift];
    }
    return f;
  };
  // its keys and values, and bit e where key 16 (e / 4) + 4 g + e % 4 exists
  auto fetch_k = [&](int tl, const Pages& f) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
      int64_t slot;
      pz_pages_slot(A.pages, f.k[t], pos_k(tl, t), &slot);
      load_k(t, kc + slot * A.ld);
    }
  };
  auto fetch_v = [&](int tl, const Pages& f) {
    uint32_t on = 0u;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      int64_t slot;
      const bool ok = pz_pages_slot(A.pages, f.v[t], pos_v(tl, t), &slot);
      const uint16_t* p = vc + slot * A.ld;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        load_v(4 * t + i, p + i * A.ld);
        if (ok && tl * TR_KEYS + 16 * t + 4 * g + i < ctx) on |= 1u << (4 * t + i);
      }
    }
    return on;
  };
  // the wave's first tile before anything else
  int tl = tl0 + w;
  const int tc = tl1 < nc ? tl1 : nc;  // the cache's tiles end here
  uint32_t on = 0u;
  Pages nx = {};
  if (tl < tc) {
    const Pages at = pages_of(tl);
    nx = pages_of(tl + WAVES < tc ? tl + WAVES : tl);
    fetch_k(tl, at);
    on = fetch_v(tl, at);
  }

  // Q as fragments: lane l: row l % 16, 8 d from 8 (l / 16) of 32
  for (int f = w; f < RT * KS; f += WAVES) {
    const int rt = f / KS, ks = f - rt * KS, r = row0 + rt * 16 + m;
    tr_u32x4 x = {0u, 0u, 0u, 0u};
    if (r < rows) {
      const int t = r / A.group, hq = h * A.group + (r - t * A.group);
      x = *reinterpret_cast<const tr_u32x4*>(A.q + (size_t)(node0 + t) * A.ld_q + (size_t)hq * D +
                                             ks * 32 + 8 * g);
    }
    *reinterpret_cast<tr_u32x4*>(sh + (f * 64 + lane) * 16) = x;
  }
  sync();

  TrRows<TYPE, D, RT, false> R;
  R.clear(lane, A.c);
  auto scores = [&]() {
    R.scores([&](int t, int ks) { return kf[t][ks]; },
             [&](int rt, int ks) {
               return *reinterpret_cast<const tr_u32x4*>(sh + ((rt * KS + ks) * 64 + lane) * 16);
             });
  };

  // The cache's tiles: the next one's keys are on their way from this one's scores
  // on, its values from this one's last use of them, its pages a tile earlier.
  for (; tl < tc; tl += WAVES) {
    const int t1 = tl + WAVES < tc ? tl + WAVES : tl, t2 = t1 + WAVES < tc ? t1 + WAVES : t1;
    scores();
    const Pages at = nx;
    fetch_k(t1, at);
    nx = pages_of(t2);
    if (__ballot(on != 0xffu)) {
      R.drop(on, [](int, int) { return true; });
      R.blank(on, vr);
    }
    R.weights();
    R.values(vr);
    on = fetch_v(t1, at);
  }
  // the nodes' tiles
  for (; ARGS::WHAT != TR_SHARED && tl < tl1; tl += WAVES) {
    const int first = (tl - nc) * TR_KEYS;
    // (past the last node: the last one again)
    auto node = [&](int i) { return (size_t)(first + i < nn ? first + i : nn - 1) * A.ld_n; };
    on = 0u;
    load_k(0, kn + node(m));
    load_k(1, kn + node(16 + m));
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int key = 16 * (e >> 2) + 4 * g + (e & 3);
      load_v(e, vn + node(key));
      on |= first + key < nn ? 1u << e : 0u;
    }
    uint64_t sees[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      const int r = row0 + rt * 16 + m, t = r < rows ? r / A.group : 0;
      sees[rt] = (A.tree ? A.tree[node0 + t] : ~0ull >> (63 - t)) >> first;
    }
    scores();
    R.drop(on, [&](int rt, int key) { return sees[rt] >> key & 1ull; });
    R.blank(on, vr);
    R.weights();
    R.odd_values(vr, sees, vn + (size_t)first * A.ld_n, A.ld_n,
                 reinterpret_cast<float*>(sh + QF + w * LDS_P));
    R.values(vr);
  }

  // the waves' results meet: common maximum, then the sums
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    R.l[rt] += __shfl_xor(R.l[rt], 16, 64);
    R.l[rt] += __shfl_xor(R.l[rt], 32, 64);
    if (g == 0) {
      mls[w][rt * 16 + m][0] = R.mx[rt];
      mls[w][rt * 16 + m][1] = R.l[rt];
    }
  }
  sync();  // (and Q is done with)
  float mt[RT], lt[RT];
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    mt[rt] = mls[0][rt * 16 + m][0];
#pragma unroll
    for (int i = 1; i < WAVES; i++) mt[rt] = fmaxf(mt[rt], mls[i][rt * 16 + m][0]);
    lt[rt] = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; i++)
      lt[rt] += mls[i][rt * 16 + m][1] * tr_lift(mls[i][rt * 16 + m][0], mt[rt], A.c);
    const float al = tr_lift(R.mx[rt], mt[rt], A.c);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) R.o[rt][nt] *= al;
  }
  const size_t unit = ((size_t)b * A.n_kv + h) * A.nblk + J.blk;
  if (ARGS::WHAT == TR_WHOLE && ns > 1 && w == 0 && g == 0)
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      float* ml = A.ml + ((unit * A.S + sp) * ROWS + rt * 16 + m) * 2;
      ml[0] = mt[rt];
      ml[1] = lt[rt];
    }
  // float4 (i, f) of row tile rt: d = NT (4 g + i) + 4 f + 0..3 of row m
  auto buf = [&](int wave, int c) {
    return reinterpret_cast<tr_f32x4*>(sh + wave * BUF + (c * 64 + lane) * 16);
  };
#pragma unroll
  for (int half = 0; half < HALF; half++) {
    constexpr int RH = RT / HALF, PER = (CH / HALF + WAVES - 1) / WAVES;  // row tiles, float4s of a wave's share
    if (half) sync();
#pragma unroll
    for (int rt = 0; rt < RH; rt++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int f = 0; f < NT / 4; f++) {
          const tr_f32x4* v = &R.o[half * RH + rt][4 * f];
          *buf(w, (rt * 4 + i) * (NT / 4) + f) = tr_f32x4{v[0][i], v[1][i], v[2][i], v[3][i]};
        }
    sync();
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int c = w * PER + j, ch = half * (CH / HALF) + c;
      if (c >= CH / HALF) break;
      tr_f32x4 v = *buf(0, c);
#pragma unroll
      for (int i = 1; i < WAVES; i++) v += *buf(i, c);
      if (ARGS::WHAT == TR_WHOLE && ns > 1) {
        reinterpret_cast<tr_f32x4*>(A.part)[((unit * A.S + sp) * CH + ch) * 64 + lane] = v;
        continue;
      }
      const int rt = ch / NT, i = ch % NT / (NT / 4), f = ch % (NT / 4);
      const int r = row0 + rt * 16 + m;
      if (r >= rows) continue;
      float lr = lt[0];
#pragma unroll
      for (int k = 1; k < RT; k++) lr = rt == k ? lt[k] : lr;
      const int t = r / A.group, hq = h * A.group + (r - t * A.group);
      if constexpr (ARGS::WHAT != TR_WHOLE) {
        float lm = mt[0];
#pragma unroll
        for (int k = 1; k < RT; k++) lm = rt == k ? mt[k] : lm;
        tr_part<D>(A, sp, (size_t)(node0 + t) * (A.n_kv * A.group) + hq, 4 * NT * g + NT * i + 4 * f, v,
                   lm, lr);
      } else {
        const float inv = tr_inverse(A, b, t, lr);
        tr_store4<TYPE>(A.out + (size_t)(node0 + t) * A.ld_out + (size_t)hq * D + 4 * NT * g + NT * i +
                            4 * f,
                        v * inv);
      }
    }
  }
}

}  // namespace
