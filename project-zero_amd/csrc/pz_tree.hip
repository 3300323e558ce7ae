// pz_tree.hip -- attention of drafted tokens over a paged cache and over each
// other along a tree (pz_tree_attention), and the accepted tokens' way into the
// pages (pz_cache_append).
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
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/pz_sampler.h"
#include "pz_device.h"
#include "pz_lmdev.h"
#include "pz_pages.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"
#include "pz_treeplan.h"

namespace {

typedef uint32_t tr_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t tr_u32x2 __attribute__((ext_vector_type(2)));
typedef float tr_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 tr_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 tr_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 tr_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 tr_f16x2 __attribute__((ext_vector_type(2)));

constexpr int TR_JOIN = 4;          // waves of a joining workgroup
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
  static constexpr float OFF = -40.0f, TH = 8.0f;
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
  static constexpr float OFF = 8.0f, TH = 6.0f;
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

__device__ __forceinline__ int tr_nodes(const TreeArgs& A, int b) {
  return A.n_nodes ? pz_pages_most(A.n_nodes[b], A.T) : A.T;
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
__device__ __forceinline__ int tr_chunk(const TreeArgs& A, int b, int lane) {
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

template <int TYPE, int D, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(D * (1 + RT) >= 512 ? 1 : 2, 8))) void
k_tree(const TreeArgs A) {
  constexpr int KS = D / 32, NT = D / 16, NW = NT / 2;  // k steps of S, d tiles, words of V
  constexpr int ROWS = 16 * RT;
  constexpr int CH = RT * NT;  // float4s of a lane's results
  constexpr int QF = RT * KS * 1024;
  constexpr int LDS_P = ROWS * (TR_KEYS + 1) * 4;
  // the waves' results meet HALF of them at a time
  constexpr int HALF = RT > 1 && CH * WAVES > 64 ? 2 : 1, BUF = CH * 1024 / HALF;  // bytes of a wave's
  constexpr int SH = WAVES * BUF > QF + WAVES * LDS_P ? WAVES * BUF : QF + WAVES * LDS_P;
  __shared__ __align__(16) char sh[SH];
  __shared__ float mls[WAVES][ROWS][2];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  // the row blocks of one range of keys on one XCD, one after the other
  const int slot = blockIdx.x >> 3, turn = slot / A.nblk, blk = slot - turn * A.nblk;
  const int grp = turn * 8 + (blockIdx.x & 7);
  if (grp >= A.B * A.n_kv * A.S) return;
  // (split by split, so that those that short sequences lack are spread over the
  // XCDs: 32 ragged sequences of up to 4096 positions in 4 splits 89 us, 75 so)
  const int units = A.B * A.n_kv, sp = grp / units, bh = grp - sp * units, h = bh % A.n_kv,
            b = bh / A.n_kv;
  const int ctx = pz_pages_len(A.pages, A.len[b]), nn = tr_nodes(A, b);
  const int rows = nn * A.group, row0 = blk * ROWS;
  if (row0 >= rows) return;
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
      x = *reinterpret_cast<const tr_u32x4*>(A.q + ((size_t)b * A.T + t) * A.ld_q +
                                             (size_t)hq * D + ks * 32 + 8 * g);
    }
    *reinterpret_cast<tr_u32x4*>(sh + (f * 64 + lane) * 16) = x;
  }
  __syncthreads();

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
  for (; tl < tl1; tl += WAVES) {
    const int node0 = (tl - nc) * TR_KEYS;
    // (past the last node: the last one again)
    auto node = [&](int i) { return (size_t)(node0 + i < nn ? node0 + i : nn - 1) * A.ld_n; };
    on = 0u;
    load_k(0, kn + node(m));
    load_k(1, kn + node(16 + m));
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int key = 16 * (e >> 2) + 4 * g + (e & 3);
      load_v(e, vn + node(key));
      on |= node0 + key < nn ? 1u << e : 0u;
    }
    uint64_t sees[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      const int r = row0 + rt * 16 + m, t = r < rows ? r / A.group : 0;
      sees[rt] = (A.tree ? A.tree[(size_t)b * A.T + t] : ~0ull >> (63 - t)) >> node0;
    }
    scores();
    R.drop(on, [&](int rt, int key) { return sees[rt] >> key & 1ull; });
    R.blank(on, vr);
    R.weights();
    R.odd_values(vr, sees, vn + (size_t)node0 * A.ld_n, A.ld_n,
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
  __syncthreads();  // (and Q is done with)
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
  const size_t unit = (size_t)bh * A.nblk + blk;
  if (ns > 1 && w == 0 && g == 0)
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
    if (half) __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RH; rt++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int f = 0; f < NT / 4; f++) {
          const tr_f32x4* v = &R.o[half * RH + rt][4 * f];
          *buf(w, (rt * 4 + i) * (NT / 4) + f) = tr_f32x4{v[0][i], v[1][i], v[2][i], v[3][i]};
        }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int c = w * PER + j, ch = half * (CH / HALF) + c;
      if (c >= CH / HALF) break;
      tr_f32x4 v = *buf(0, c);
#pragma unroll
      for (int i = 1; i < WAVES; i++) v += *buf(i, c);
      if (ns > 1) {
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
      const float inv = tr_inverse(A, b, t, lr);
      tr_store4<TYPE>(A.out + ((size_t)b * A.T + t) * A.ld_out + (size_t)hq * D + 4 * NT * g +
                          NT * i + 4 * f,
                      v * inv);
    }
  }
}

// Many rows: the waves of a workgroup own 16 RT rows each and share the keys,
// whose tiles come straight to LDS through a ring of TR_STAGES -- whole rows of
// keys and of values, one barrier per tile -- instead of to every wave's
// registers.  Waves past the last row load only, which is worth having: 48 rows
// in 8 waves 83 us, in 4 111 (32 ragged sequences of up to 4096 positions; 78
// since fragments are read a phase before their products).  The
// 16-byte pieces of a key's row are permuted so that the 16 rows that one cycle
// reads lie in 16 places.
template <int TYPE, int D, int RT>
__global__ __launch_bounds__(64 * TR_WIDE) __attribute__((amdgpu_waves_per_eu(TR_WIDE / 4, 8))) void
k_tree_wide(const TreeArgs A) {
  constexpr int WAVES = TR_WIDE, NS = TR_STAGES;
  typedef TrRows<TYPE, D, RT, true> Rows;
  constexpr int KS = D / 32, NT = D / 16, NW = NT / 2, ROWS = 16 * RT, CH = RT * NT;
  constexpr int TILE = TR_KEYS * D * 2;            // bytes of a tile's keys, or of its values
  constexpr int LN = TILE / 1024, PER = 2 * LN / WAVES;  // 1 KiB loads: of a tile's keys, of a wave
  constexpr int PR = D / 8, RPI = 64 / PR;         // 16-byte pieces of a row, rows of a load
  constexpr int LDS_P = ROWS * (TR_KEYS + 1) * 4;
  static_assert(2 * LN % WAVES == 0 && RPI <= 8, "");
  constexpr int STG = 2 * TILE;  // a stage: a tile's keys, then its values
  __shared__ __align__(16) char sh[NS * STG + WAVES * LDS_P];
  __shared__ int32_t tab[TR_ENTRIES];
  __shared__ int broken;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  // the row blocks of one range of keys on one XCD, one after the other
  const int nwg = A.nblk / WAVES;
  const int slot = blockIdx.x >> 3, turn = slot / nwg, wg = slot - turn * nwg;
  const int grp = turn * 8 + (blockIdx.x & 7);
  if (grp >= A.B * A.n_kv * A.S) return;
  const int units = A.B * A.n_kv, sp = grp / units, bh = grp - sp * units, h = bh % A.n_kv,
            b = bh / A.n_kv;
  const int ctx = pz_pages_len(A.pages, A.len[b]), nn = tr_nodes(A, b);
  const int rows = nn * A.group, row0 = (wg * WAVES + w) * ROWS;
  if (wg * WAVES * ROWS >= rows) return;
  const int nc = (ctx + TR_KEYS - 1) / TR_KEYS, ntl = nc + (nn + TR_KEYS - 1) / TR_KEYS;
  const int chunk = tr_chunk(A, b, lane);
  const int tl0 = sp * chunk, tl1 = ntl - tl0 < chunk ? ntl : tl0 + chunk;
  if (tl0 >= ntl) return;
  const int ns = (ntl + chunk - 1) / chunk;  // splits that this sequence has
  const bool idle = row0 >= rows;                // (a wave past the last row loads only)
  const uint16_t* kc = A.k + (size_t)h * D;
  const uint16_t* vc = A.v + (size_t)h * D;
  const uint16_t* kn = A.kn + (size_t)b * A.T * A.ld_n + (size_t)h * D;
  const uint16_t* vn = A.vn + (size_t)b * A.T * A.ld_n + (size_t)h * D;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)sh;
  const int lr = lane / PR, place = lane % PR;

  // load i of this wave for a tile: of keys or values, rows qk * RPI ..
  auto swizzle = [](int key) { return D == 64 ? key >> 1 & 7 : key & (PR - 1); };
  // (where a wave has an even number of loads, the keys and the values of one place)
  constexpr int PK = PER % 2 == 0 ? PER / 2 : PER;  // places of a wave
  auto of_v = [&](int i) { return PER % 2 == 0 ? i >= PK : w * PER + i >= LN; };
  auto qk_of = [&](int i) { return PER % 2 == 0 ? w * PK + i % PK : (w * PER + i) % LN; };
  uint32_t off[PER], pc[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    pc[i] = 16u * (of_v(i) ? place : place ^ swizzle(qk_of(i) * RPI + lr));
    off[i] = (uint32_t)lr * (uint32_t)A.ld * 2u + pc[i];
  }
  // the page of load i (positions past the last: the last one's rows again)
  auto pos_of = [&](int tl, int i) {
    const int p = tl * TR_KEYS + qk_of(i) * RPI, last = (ctx - 1) & ~(RPI - 1);
    return p < last ? p : last;
  };
  // The range's part of the table in LDS: a scalar load per tile would make every
  // wait for LDS one for it, too (8 x 64 nodes over 32768 positions 403 us, 344
  // without).
  const int e0 = tl0 * TR_KEYS >> A.pages.shift;
  bool whole = true;  // whether the range's pages are all there
  {
    const int e1 = ((tl1 < nc ? tl1 * TR_KEYS : ctx) - 1) >> A.pages.shift;
    if (tl0 < nc)
      for (int e = e0 + tid; e <= e1; e += 64 * WAVES) {
        const int32_t id = A.blocks[(size_t)b * A.pages.max_blocks + e];
        if (e - e0 < TR_ENTRIES) tab[e - e0] = id;
        whole = whole && (uint32_t)id < (uint32_t)A.pages.n_blocks;
      }
    if (tid == 0) broken = 0;
    __syncthreads();
    if (!whole) broken = 1;
    __syncthreads();
    whole = broken == 0;
  }
  // (Entries past those that LDS holds: with a wait of their own, which is one for the
  // ring's loads, too.)
  auto entry = [&](int p) {
    const int e = p >> A.pages.shift;
    int32_t id;
    if (e - e0 < TR_ENTRIES) {
      id = tab[e - e0];
    } else {
      id = A.blocks[(size_t)b * A.pages.max_blocks + e];
      __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    }
    return id;
  };
  struct Ids {
    int32_t v[PK];
  };
  auto ids_of = [&](int tl) {
    Ids r;
#pragma unroll
    for (int i = 0; i < PK; i++) r.v[i] = tl < nc ? entry(pos_of(tl, i)) : 0;
    return r;
  };
  auto issue = [&](int tl, const Ids& ids, int buf) {
    const uint32_t to = lds0 + buf * STG;
    if (tl < nc) {
#pragma unroll
      for (int i = 0; i < PK; i++) {
        int64_t at;
        pz_pages_slot(A.pages, __builtin_amdgcn_readfirstlane(ids.v[i]), pos_of(tl, i), &at);
        at *= A.ld;
#pragma unroll
        for (int j = i; j < PER; j += PK)
          lm_lds_load16<false>((of_v(j) ? vc : kc) + at, off[j],
                               to + ((of_v(j) ? LN : 0) + qk_of(j)) * 1024);
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const int n = (tl - nc) * TR_KEYS + qk_of(i) * RPI + lr;
        lm_lds_load16<false>(of_v(i) ? vn : kn,
                             (uint32_t)(n < nn ? n : nn - 1) * (uint32_t)A.ld_n * 2u + pc[i],
                             to + ((of_v(i) ? LN : 0) + qk_of(i)) * 1024);
      }
    }
  };
  // bit e where key 16 (e / 4) + 4 g + e % 4 of a tile of the cache exists
  auto held = [&](int tl) {
    uint32_t on = 0u;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int p = tl * TR_KEYS + 16 * (e >> 2) + 4 * g + (e & 3);
      const int32_t id = entry(p < ctx ? p : ctx - 1);
      if (p < ctx && (uint32_t)id < (uint32_t)A.pages.n_blocks) on |= 1u << e;
    }
    return on;
  };
  auto clip = [&](int tl) { return tl < tl1 ? tl : tl1 - 1; };  // (past the last: read again)
  tr_u32x4 qf[RT][KS];  // lane l: row l % 16, 8 d from 8 (l / 16) of 32
  uint64_t sees[RT];
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    const int r = row0 + rt * 16 + m, rr = r < rows ? r : 0, t = rr / A.group,
              hq = h * A.group + (rr - t * A.group);
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
      qf[rt][ks] = *reinterpret_cast<const tr_u32x4*>(A.q + ((size_t)b * A.T + t) * A.ld_q +
                                                      (size_t)hq * D + ks * 32 + 8 * g);
    sees[rt] = A.tree ? A.tree[(size_t)b * A.T + t] : ~0ull >> (63 - t);
  }
  // (arrived before the ring's loads, which the compiler does not see, are under
  // way: a wait for them in the loop would be one for those, too)
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
#pragma unroll
  for (int i = 0; i < NS - 1; i++) issue(clip(tl0 + i), ids_of(clip(tl0 + i)), i);
  Ids ids = ids_of(clip(tl0 + NS - 1));

  Rows R;
  R.clear(lane, A.c);
  int buf = 0, nbuf = NS - 1;
  // Tiles tl to tl + 2 have arrived, in every wave; and every wave is done with the
  // slot of the tile before, which is filled next.
  auto step = [&](int tl) {
    lm_wait<(NS - 4) * PER>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue(clip(tl + NS - 1), ids, nbuf);
    ids = ids_of(clip(tl + NS));
  };
  auto next = [&]() {
    asm volatile("" ::: "memory");
    buf = buf + 1 == NS ? 0 : buf + 1;
    nbuf = nbuf + 1 == NS ? 0 : nbuf + 1;
  };
  auto kf = [&](int at, int t, int ks) {
    const int key = 16 * t + m;
    return *reinterpret_cast<const tr_u32x4*>(sh + at * STG + key * D * 2 +
                                              ((ks * 4 + g) ^ swizzle(key)) * 16);
  };
  auto scores = [&](int at) {
    R.scores([&](int t, int ks) { return kf(at, t, ks); },
             [&](int rt, int ks) { return qf[rt][ks]; });
  };
  // the words of a key's values in this lane
  auto fetch = [&](const char* p, uint32_t(&v)[NW]) {
    if constexpr (NW == 2) {
      const tr_u32x2 x = *reinterpret_cast<const tr_u32x2*>(p);
      v[0] = x[0];
      v[1] = x[1];
    } else {
      static_assert(NW == 4, "");
      const tr_u32x4 x = *reinterpret_cast<const tr_u32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = x[i];
    }
  };
  int tl = tl0;
  const int tc = tl1 < nc ? tl1 : nc;  // the cache's tiles end here
  lm_wait<(NS - 3) * PER>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  constexpr int NQ = 2 * KS;  // fragments of a tile's keys
  tr_u32x4 kr[NQ];            // those of tile tl + 1
  float tm[RT] = {};
  if (!idle && tl < tc) {
    scores(0);
    R.tops(R.s, tm);
#pragma unroll
    for (int q = 0; q < NQ; q++) kr[q] = kf(1, q & 1, q >> 1);
  }
  // The weights of a tile beside the scores of the next, its values beside that
  // one's keys, each fragment read a phase before its product.
#pragma clang loop unroll(disable)
  for (; tl < tc; tl++) {
    step(tl);
    const bool full = whole && (tl + 1) * TR_KEYS <= ctx;
    if (!full) {
      // what lies in the place of a position that does not exist may be anything
      for (int i = tid; i < TILE / 16; i += 64 * WAVES) {
        const int p = tl * TR_KEYS + i / PR;
        if (p >= ctx || (uint32_t)entry(p) >= (uint32_t)A.pages.n_blocks)
          *reinterpret_cast<tr_u32x4*>(sh + buf * STG + TILE + i * 16) = tr_u32x4{0u, 0u, 0u, 0u};
      }
      __syncthreads();
    }
    if (!idle) {
      if (!full) {
        R.drop(held(tl), [](int, int) { return true; });
        R.tops(R.s, tm);
      }
      R.raise(tm);
      const int ahead = buf + 2 >= NS ? buf + 2 - NS : buf + 2;
      const char* vt = sh + buf * STG + TILE + 4 * g * D * 2 + m * NT * 2;
      uint32_t vr[8][NW];
      tr_f32x4 sn[RT][2];  // (of whatever lies there after the last of them: unused)
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int t = 0; t < 2; t++) sn[rt][t] = tr_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        constexpr int EQ = 8 / NQ;  // weights and keys' values beside each
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
          sn[rt][q & 1] = TrType<TYPE>::mfma(kr[q], qf[rt][q >> 1], sn[rt][q & 1]);
#pragma unroll
        for (int e = q * EQ; e < (q + 1) * EQ; e++) {
#pragma unroll
          for (int rt = 0; rt < RT; rt++) R.weigh(rt, e);
          fetch(vt + (16 * (e >> 2) + (e & 3)) * D * 2, vr[e]);
        }
      }
      tr_u32x4 pf[RT];
      R.pack(pf);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = vr[e][nt >> 1];
        R.value(nt, v, nt & 1, pf);
#pragma unroll
        for (int q = nt * NQ / NT; q < (nt + 1) * NQ / NT; q++) kr[q] = kf(ahead, q & 1, q >> 1);
      }
      R.tops(sn, tm);
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int t = 0; t < 2; t++) R.s[rt][t] = sn[rt][t];
    }
    next();
  }
  // the nodes' tiles
#pragma clang loop unroll(disable)
  for (; tl < tl1; tl++) {
    step(tl);
    if (!idle) {
      const int node0 = (tl - nc) * TR_KEYS;
      uint32_t on = 0u, vr[8][NW];
#pragma unroll
      for (int e = 0; e < 8; e++)
        on |= node0 + 16 * (e >> 2) + 4 * g + (e & 3) < nn ? 1u << e : 0u;
      uint64_t of_tile[RT];
#pragma unroll
      for (int rt = 0; rt < RT; rt++) of_tile[rt] = sees[rt] >> node0;
      scores(buf);
#pragma unroll
      for (int e = 0; e < 8; e++)
        fetch(sh + buf * STG + TILE + (16 * (e >> 2) + 4 * g + (e & 3)) * D * 2 + m * NT * 2, vr[e]);
      R.drop(on, [&](int rt, int key) { return of_tile[rt] >> key & 1ull; });
      R.blank(on, vr);
      R.weights();
      R.odd_values(vr, of_tile, vn + (size_t)node0 * A.ld_n, A.ld_n,
                   reinterpret_cast<float*>(sh + NS * STG + w * LDS_P));
      R.values(vr);
    }
    next();
  }
  lm_wait<0>();
  if (idle) return;
  const size_t unit = (size_t)bh * A.nblk + wg * WAVES + w;
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    float l = R.l[rt];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const int r = row0 + rt * 16 + m;
    if (ns > 1) {
      if (g == 0) {
        float* ml = A.ml + ((unit * A.S + sp) * ROWS + rt * 16 + m) * 2;
        ml[0] = R.mx[rt];
        ml[1] = l;
      }
    } else if (r >= rows) {
      continue;
    }
    const int t = r / A.group, hq = h * A.group + (r - t * A.group);
    const float inv = ns > 1 ? 0.0f : tr_inverse(A, b, t, l);
    uint16_t* out = A.out + ((size_t)b * A.T + t) * A.ld_out + (size_t)hq * D + 4 * NT * g;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int f = 0; f < NT / 4; f++) {
        const tr_f32x4* o = &R.o[rt][4 * f];
        const tr_f32x4 v = {o[0][i], o[1][i], o[2][i], o[3][i]};
        if (ns > 1)
          reinterpret_cast<tr_f32x4*>(
              A.part)[((unit * A.S + sp) * CH + (rt * 4 + i) * (NT / 4) + f) * 64 + lane] = v;
        else
          tr_store4<TYPE>(out + NT * i + 4 * f, v * inv);
      }
  }
}

// Adds up the splits of one unit (key head and row block): for each float4 of a
// lane's results WAVES waves, which take the splits in turn; TR_JOIN / WAVES of
// them in a workgroup.  (One wave where the splits are few enough to be under way
// together: 512 units of 4 splits of 32 rows 20
// -> 11 us.)
template <int TYPE, int D, int RT, int WAVES>
__global__ __launch_bounds__(64 * TR_JOIN) void k_tree_join(const TreeArgs A) {
  constexpr int NT = D / 16, ROWS = 16 * RT, CH = RT * NT, PER = TR_JOIN / WAVES;
  static_assert(CH % PER == 0 && (WAVES == 1 || PER == 1), "a workgroup's work is one unit's");
  __shared__ tr_f32x4 sum[WAVES][64];
  __shared__ float mls[WAVES][16][2];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4, w = wv % WAVES, at = blockIdx.x * PER + wv / WAVES;
  const int unit = at / CH, ch = at - unit * CH;
  const int blk = unit % A.nblk, bh = unit / A.nblk, h = bh % A.n_kv, b = bh / A.n_kv;
  const int nn = tr_nodes(A, b), rows = nn * A.group;
  if (blk * ROWS >= rows) return;  // (its workgroups wrote nothing)
  const int chunk = tr_chunk(A, b, lane), ns = (tr_tiles(A, b) + chunk - 1) / chunk;
  if (ns <= 1) return;  // (its workgroup wrote the results)
  const int rt = ch / NT, i = ch % NT / (NT / 4), f = ch % (NT / 4);
  const float* ml = A.ml + ((size_t)unit * A.S * ROWS + rt * 16 + m) * 2;
  const tr_f32x4* part =
      reinterpret_cast<const tr_f32x4*>(A.part) + ((size_t)unit * A.S * CH + ch) * 64 + lane;
  constexpr int U = 4;  // splits of a wave whose results are on their way together
  float mt = TR_LOW, lt = 0.0f;
  tr_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = w; s0 < ns; s0 += WAVES * U) {
    float ms[U], ls[U];
    tr_f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int s = s0 + u * WAVES < ns ? s0 + u * WAVES : s0;  // (past the last: the first,
      ms[u] = ml[(size_t)s * ROWS * 2];                             // for nothing)
      ls[u] = s0 + u * WAVES < ns ? ml[(size_t)s * ROWS * 2 + 1] : 0.0f;
      v[u] = part[(size_t)s * CH * 64];
    }
    float mn = mt;
#pragma unroll
    for (int u = 0; u < U; u++) mn = fmaxf(mn, ms[u]);
    const float al = tr_lift(mt, mn, A.c);
    mt = mn;
    lt *= al;
    o *= al;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const float e = tr_lift(ms[u], mt, A.c);
      lt += ls[u] * e;
      if (s0 + u * WAVES < ns) o += v[u] * e;
    }
  }
  const int r = blk * ROWS + rt * 16 + m;
  if constexpr (WAVES > 1) {
    sum[w][lane] = o;
    if (g == 0) {
      mls[w][m][0] = mt;
      mls[w][m][1] = lt;
    }
    __syncthreads();
    if (w != 0) return;
    float mx = mt;
#pragma unroll
    for (int k = 1; k < WAVES; k++) mx = fmaxf(mx, mls[k][m][0]);
    const float a0 = tr_lift(mt, mx, A.c);
    lt *= a0;
    o *= a0;
#pragma unroll
    for (int k = 1; k < WAVES; k++) {
      const float e = tr_lift(mls[k][m][0], mx, A.c);
      lt += mls[k][m][1] * e;
      o += sum[k][lane] * e;
    }
  }
  if (r >= rows) return;
  const int t = r / A.group, hq = h * A.group + (r - t * A.group);
  const float inv = tr_inverse(A, b, t, lt);
  tr_store4<TYPE>(A.out + ((size_t)b * A.T + t) * A.ld_out + (size_t)hq * D + 4 * NT * g + NT * i +
                      4 * f,
                  o * inv);
}

// Plans the splits of `units` row blocks of 16 RT rows over sequences of up to
// `tiles` tiles, about `want` of each.
template <int D, int RT>
int plan(pz_sampler* s, TreeArgs& A, int64_t units, int64_t tiles, int64_t want) {
  constexpr int ROWS = 16 * RT;
  const int64_t room = (int64_t)(PZ_TREE_WS / ((size_t)ROWS * (D + 2) * sizeof(float))) / units;
  int64_t S = want < room ? want : room;
  S = S < 64 ? S : 64;
  S = S < 1 ? 1 : S;
  // every sequence takes as many splits as it has chunks: short ones write their
  // results at once
  A.chunk = (int)((tiles + S - 1) / S);
  A.S = (int)((tiles + A.chunk - 1) / A.chunk);
  A.part = static_cast<float*>(s->tree_dev);
  A.ml = A.part + (size_t)units * A.S * ROWS * D;
  if (!pz_launch_fits(((int64_t)A.B * A.n_kv * A.S + 7) * A.nblk, 512) ||
      !pz_launch_fits(units * RT * (D / 16), A.S > 1 ? 64 * TR_JOIN : 1))
    return fail(s, PZ_ERANGE, "B=%d sequences of T=%d nodes", A.B, A.T);
  return PZ_OK;
}

template <int TYPE, int D, int RT>
int join(pz_sampler* s, const TreeArgs& A, int64_t units) {
  PZ_HIP(s, hipGetLastError());
  if (A.S > 1) {
    const unsigned parts = (unsigned)(units * RT * (D / 16));
    if (A.S <= 4)
      hipLaunchKernelGGL((k_tree_join<TYPE, D, RT, 1>), dim3(parts / TR_JOIN), dim3(64 * TR_JOIN),
                         0, s->stream, A);
    else
      hipLaunchKernelGGL((k_tree_join<TYPE, D, RT, TR_JOIN>), dim3(parts), dim3(64 * TR_JOIN), 0,
                         s->stream, A);
    PZ_HIP(s, hipGetLastError());
  }
  return PZ_OK;
}

template <int TYPE, int D, int RT, int WAVES>
int narrow(pz_sampler* s, TreeArgs& A, int64_t tiles, int64_t want) {
  A.nblk = (A.T * A.group + 16 * RT - 1) / (16 * RT);
  const int64_t units = (int64_t)A.B * A.n_kv * A.nblk;
  const int rc = plan<D, RT>(s, A, units, tiles, want);
  if (rc != PZ_OK) return rc;
  const int64_t groups = ((int64_t)A.B * A.n_kv * A.S + 7) / 8 * 8;
  hipLaunchKernelGGL((k_tree<TYPE, D, RT, WAVES>), dim3((unsigned)(groups * A.nblk)),
                     dim3(64 * WAVES), 0, s->stream, A);
  return join<TYPE, D, RT>(s, A, units);
}

template <int TYPE, int D, int RT>
int wide(pz_sampler* s, TreeArgs& A, int64_t tiles, int64_t want) {
  const int nwg = (A.T * A.group + 16 * RT * TR_WIDE - 1) / (16 * RT * TR_WIDE);
  A.nblk = nwg * TR_WIDE;
  const int64_t units = (int64_t)A.B * A.n_kv * A.nblk;
  const int rc = plan<D, RT>(s, A, units, tiles, want);
  if (rc != PZ_OK) return rc;
  const int64_t groups = ((int64_t)A.B * A.n_kv * A.S + 7) / 8 * 8;
  hipLaunchKernelGGL((k_tree_wide<TYPE, D, RT>), dim3((unsigned)(groups * nwg)),
                     dim3(64 * TR_WIDE), 0, s->stream, A);
  return join<TYPE, D, RT>(s, A, units);
}

template <int TYPE, int D>
int run_rows(pz_sampler* s, TreeArgs& A) {
  const int rows = A.T * A.group;
  const int64_t tiles = ((int64_t)A.pages.max_blocks << A.pages.shift) / TR_KEYS + 1 +
                        (A.T + TR_KEYS - 1) / TR_KEYS;
  const int64_t heads = (int64_t)A.B * A.n_kv;
  // A workgroup a CU, and two tiles a wave at least.  (More only add a launch and
  // its traffic: 32 x 5 nodes, 256 key heads, over 2048 positions whole 55 us, in
  // two splits 67.)
  auto splits = [&](int64_t wgs) {
    const int64_t want = (s->n_cu + wgs - 1) / wgs, most = tiles / TR_SHARE;
    return want < most ? want : most;
  };
  const TrKernel kernel = tr_kernel_for(rows, heads, tiles, s->n_cu, D, A.ld, A.ld_n);
  if constexpr (D < 256) {
    if (kernel == TR_FEW_SHORT) return narrow<TYPE, D, 1, 8>(s, A, tiles, 1);
    if (kernel == TR_WIDE16) return wide<TYPE, D, 1>(s, A, tiles, splits(heads));
    if (kernel == TR_WIDE32)
      return wide<TYPE, D, 2>(s, A, tiles, splits(heads * ((rows + 255) / 256)));
  }
  if (kernel == TR_FEW) return narrow<TYPE, D, 1, 4>(s, A, tiles, splits(heads));
  return narrow<TYPE, D, 2, 4>(s, A, tiles, splits(heads * ((rows + 31) / 32)));
}

template <int TYPE>
int run(pz_sampler* s, TreeArgs& A, int D) {
  if (D == 64) return run_rows<TYPE, 64>(s, A);
  if (D == 128) return run_rows<TYPE, 128>(s, A);
  return run_rows<TYPE, 256>(s, A);
}

// ---- append --------------------------------------------------------------------
// One workgroup per node: its row of keys and its row of values, 16 bytes a
// thread.
__global__ __launch_bounds__(256) void k_append(const TreeArgs A, int row, const int32_t* take,
                                                const int32_t* count) {
  const int b = blockIdx.x / A.T, i = blockIdx.x - b * A.T;
  if (count && i >= pz_pages_most(count[b], A.T)) return;
  const int node = take ? take[blockIdx.x] : i;
  if (node < 0 || node >= A.T) return;
  const int64_t p = (int64_t)pz_pages_len(A.pages, A.len[b]) + i;
  if (p >= (int64_t)A.pages.max_blocks << A.pages.shift) return;
  int64_t slot;
  const int32_t page = A.blocks[(size_t)b * A.pages.max_blocks + (p >> A.pages.shift)];
  if (!pz_pages_slot(A.pages, page, (int)p, &slot)) return;
  const size_t to = (size_t)slot * A.ld;
  const size_t from = ((size_t)b * A.T + node) * A.ld_n;
  const int n = row / 8;  // 16-byte pieces
  for (int j = threadIdx.x; j < 2 * n; j += 256) {
    const bool val = j >= n;
    const int d = (val ? j - n : j) * 8;
    *reinterpret_cast<tr_u32x4*>(const_cast<uint16_t*>(val ? A.v : A.k) + to + d) =
        *reinterpret_cast<const tr_u32x4*>((val ? A.vn : A.kn) + from + d);
  }
}

TreeArgs args_of(const pz_kv_cache* c, const void* d_kn, const void* d_vn, long ld_n, int B,
                 int T) {
  TreeArgs A = {};
  A.k = static_cast<const uint16_t*>(c->d_k);
  A.v = static_cast<const uint16_t*>(c->d_v);
  A.ld = c->ld;
  A.pages = {c->n_blocks, __builtin_ctz((unsigned)c->block_size), c->max_blocks};
  A.blocks = c->d_blocks;
  A.len = c->d_len;
  A.n_kv = c->n_kv_heads;
  A.kn = static_cast<const uint16_t*>(d_kn);
  A.vn = static_cast<const uint16_t*>(d_vn);
  A.ld_n = ld_n;
  A.B = B;
  A.T = T;
  return A;
}

}  // namespace

extern "C" int pz_tree_attention(pz_sampler* s, const pz_kv_cache* cache, const void* d_kn,
                                 const void* d_vn, long ld_n, int B, int T,
                                 const int32_t* d_n_nodes, const uint64_t* d_tree, int n_heads,
                                 float scale, const void* d_q, long ld_q, void* d_out,
                                 long ld_out) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no =
      pz_refuse_tree(cache, d_kn, d_vn, ld_n, B, T, n_heads, scale, d_q, ld_q, d_out, ld_out);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (B == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  if (!s->tree_dev && hipMalloc(&s->tree_dev, PZ_TREE_WS) != hipSuccess) {
    s->tree_dev = nullptr;
    (void)hipGetLastError();
    return fail(s, PZ_ENOMEM, "tree attention's workspace");
  }
  TreeArgs A = args_of(cache, d_kn, d_vn, ld_n, B, T);
  A.n_nodes = d_n_nodes;
  A.tree = d_tree;
  A.group = n_heads / cache->n_kv_heads;
  A.c = scale * TR_LOG2E;
  A.q = static_cast<const uint16_t*>(d_q);
  A.ld_q = ld_q;
  A.out = static_cast<uint16_t*>(d_out);
  A.ld_out = ld_out;
  return cache->type == PZ_BF16 ? run<PZ_BF16>(s, A, cache->head_dim)
                                : run<PZ_F16>(s, A, cache->head_dim);
}

extern "C" int pz_cache_append(pz_sampler* s, const pz_kv_cache* cache, const void* d_kn,
                               const void* d_vn, long ld_n, int B, int T, const int32_t* d_take,
                               const int32_t* d_count) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no = pz_refuse_cache(cache, d_kn, d_vn, ld_n, B, T);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (B == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  const TreeArgs A = args_of(cache, d_kn, d_vn, ld_n, B, T);
  hipLaunchKernelGGL(k_append, dim3((unsigned)B * (unsigned)T), dim3(256), 0, s->stream, A,
                     cache->n_kv_heads * cache->head_dim, d_take, d_count);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}
