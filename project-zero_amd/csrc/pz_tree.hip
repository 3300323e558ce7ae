// pz_tree.hip -- attention of drafted tokens over a paged cache and over each
// other along a tree (pz_tree_attention), and the accepted tokens' way into the
// pages (pz_cache_append).
//
//   out[r] = sum_p softmax_p(scale q[r] . k[p]) v[p],  r = (node, head of a key
//   head's group), p over the cached positions and the nodes that r's node sees.
//
// One pass over the keys with a running maximum m and sum l per row; the
// scores' exponentials are taken to base 2 of scale log2(e) s - m.  All rows of
// a key head share its keys, so nodes x group rows meet each key: 16 of them a
// column of v_mfma_f32_16x16x32.
//
//   * A workgroup of 4 waves owns 16 RT rows of one key head of one sequence
//     and a range of its keys; its waves take tiles of 32 keys in turn, each
//     with its own m, l and result, which meet in LDS at the end.  No barrier
//     and no LDS traffic for keys or values on the way: both go from memory to
//     registers in the order the matrix cores take them.
//   * S^T = K Q^T: A = 16 keys x 32 d, lane l: key l % 16, 8 d from 8 (l / 16).
//     D gives lane l row l % 16 and keys 4 (l / 16) .. +3 of each 16: with two
//     key tiles the 8 weights of one k group of the next product, whose key
//     order (16 t + 4 g + i) V then follows.
//   * O^T = V^T P^T: lane l loads D / 16 neighbouring values of each of its 8
//     keys (l / 16's) from d = (l % 16) D / 16: whole rows of V, coalesced; a
//     byte permute gathers the 8 keys of one d.  D's rows are d, its columns the
//     rows of q, so m, l and the rescaling are a lane's own.
//   * m is raised only when a score passes it by 2^TH_: the weights stay below
//     2^(TH_ + OFF_), and the cross-lane maximum and the rescaling drop out of
//     most tiles.
//   * Few rows and long sequences: the keys are split over S workgroups, whose
//     results k_tree_join adds up.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/pz_sampler.h"
#include "pz_device.h"
#include "pz_pages.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"

namespace {

typedef uint32_t tr_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t tr_u32x2 __attribute__((ext_vector_type(2)));
typedef float tr_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 tr_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 tr_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 tr_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 tr_f16x2 __attribute__((ext_vector_type(2)));

constexpr int TR_WAVES = 4;
constexpr int TR_KEYS = 32;         // keys of a tile
constexpr float TR_LOW = -3.0e38f;  // m before any score (finite: m - m is 0)
constexpr float TR_LOG2E = 1.44269504088896340736f;

template <int TYPE>
struct TrType;
template <>
struct TrType<PZ_BF16> {
  static constexpr float OFF = 0.0f, TH = 8.0f;
  static constexpr uint32_t EXP = 0x7f80u;  // exponent bits of one element
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
  int S, nblk;  // splits, row blocks of a key head
  float* part;  // [unit][S] results (TR result order), then their m and l
  float* ml;
};

__device__ __forceinline__ int tr_nodes(const TreeArgs& A, int b) {
  return A.n_nodes ? pz_pages_most(A.n_nodes[b], A.T) : A.T;
}

// A lane's results of one row: d = NT (4 g + i) + 4 f + 0..3 in o (i, f).
template <int TYPE>
__device__ __forceinline__ void tr_store4(uint16_t* o, const tr_f32x4 v) {
  tr_u32x2 w;
  w[0] = TrType<TYPE>::pack(v[0], v[1]);
  w[1] = TrType<TYPE>::pack(v[2], v[3]);
  *reinterpret_cast<tr_u32x2*>(o) = w;
}

template <int TYPE, int D, int RT>
__global__ __launch_bounds__(64 * TR_WAVES) void k_tree(const TreeArgs A) {
  typedef TrType<TYPE> Y;
  constexpr int KS = D / 32, NT = D / 16, NW = NT / 2;  // k steps of S, d tiles, words of V
  constexpr int ROWS = 16 * RT;
  constexpr int CH = RT * NT;  // float4s of a lane's results
  constexpr int QF = RT * KS * 1024;
  constexpr int BUF = CH * 64 * 16;  // one wave's results
  constexpr int LDS_P = ROWS * (TR_KEYS + 1) * 4;
  constexpr int SH = 2 * BUF > QF + TR_WAVES * LDS_P ? 2 * BUF : QF + TR_WAVES * LDS_P;
  __shared__ __align__(16) char sh[SH];
  __shared__ float mls[TR_WAVES][ROWS][2];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  // the row blocks of one range of keys on one XCD, one after the other
  const int slot = blockIdx.x >> 3;
  const int grp = (slot / A.nblk) * 8 + (blockIdx.x & 7), blk = slot % A.nblk;
  if (grp >= A.B * A.n_kv * A.S) return;
  const int sp = grp % A.S, bh = grp / A.S, h = bh % A.n_kv, b = bh / A.n_kv;
  const int ctx = pz_pages_len(A.pages, A.len[b]), nn = tr_nodes(A, b);
  const int rows = nn * A.group, row0 = blk * ROWS;
  if (row0 >= rows) return;
  const int nc = (ctx + TR_KEYS - 1) / TR_KEYS, ntl = nc + (nn + TR_KEYS - 1) / TR_KEYS;
  const int tl0 = (int)((int64_t)ntl * sp / A.S), tl1 = (int)((int64_t)ntl * (sp + 1) / A.S);

  // Q as fragments: lane l: row l % 16, 8 d from 8 (l / 16) of 32
  for (int f = w; f < RT * KS; f += TR_WAVES) {
    const int rt = f / KS, ks = f - rt * KS, r = row0 + rt * 16 + m;
    tr_u32x4 x = {0u, 0u, 0u, 0u};
    if (r < rows) {
      const int t = r / A.group, hq = h * A.group + (r - t * A.group);
      x = *reinterpret_cast<const tr_u32x4*>(A.q + ((size_t)b * A.T + t) * A.ld_q +
                                             (size_t)hq * D + ks * 32 + 8 * g);
    }
    *reinterpret_cast<tr_u32x4*>(sh + (f * 64 + lane) * 16) = x;
  }
  uint64_t sees[RT];
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    const int r = row0 + rt * 16 + m, t = r < rows ? r / A.group : 0;
    sees[rt] = A.tree ? A.tree[(size_t)b * A.T + t] : ~0ull >> (63 - t);
  }
  __syncthreads();

  tr_f32x4 o[RT][NT];
  float mx[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    mx[rt] = TR_LOW;
    l[rt] = 0.0f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) o[rt][nt] = tr_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int32_t* table = A.blocks + (size_t)b * A.pages.max_blocks;
  const uint16_t* kc = A.k + (size_t)h * D;
  const uint16_t* vc = A.v + (size_t)h * D;
  const uint16_t* kn = A.kn + (size_t)b * A.T * A.ld_n + (size_t)h * D;
  const uint16_t* vn = A.vn + (size_t)b * A.T * A.ld_n + (size_t)h * D;

  // one tile: key 16 t + m at kp[t], the values of key 16 (e / 4) + 4 g + e % 4 at
  // vp(e); `on`: bit e set where that key exists, `all`: wherever there is one.
  // NODE: of nodes, the first of them node0
  auto tile = [&](auto node_tag, const uint16_t* const(&kp)[2], auto vp, uint32_t on, bool all,
                  int node0) {
    constexpr bool NODE = decltype(node_tag)::value;
    tr_u32x4 kf[2][KS];
    uint32_t vr[8][NW];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
        kf[t][ks] = *reinterpret_cast<const tr_u32x4*>(kp[t] + ks * 32 + 8 * g);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint16_t* p = vp(e) + m * NT;
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
    }
    tr_f32x4 s[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        s[rt][t] = tr_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
          s[rt][t] = Y::mfma(kf[t][ks],
                             *reinterpret_cast<const tr_u32x4*>(
                                 sh + ((rt * KS + ks) * 64 + lane) * 16),
                             s[rt][t]);
      }
    if (NODE || !all) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool there = on >> e & 1u;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
          bool seen = there;
          if (NODE) seen = there && (sees[rt] >> (node0 + 16 * (e >> 2) + 4 * g + (e & 3)) & 1ull);
          s[rt][e >> 2][e & 3] = seen ? s[rt][e >> 2][e & 3] : -__builtin_inff();
        }
        // what lies in the place of a key that does not exist may be anything
#pragma unroll
        for (int i = 0; i < NW; i++) vr[e][i] = there ? vr[e][i] : 0u;
      }
    }
    float tm[RT];
    bool up = false;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      tm[rt] = fmaxf(fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), fmaxf(s[rt][0][2], s[rt][0][3])),
                     fmaxf(fmaxf(s[rt][1][0], s[rt][1][1]), fmaxf(s[rt][1][2], s[rt][1][3]))) *
               A.c;
      up |= tm[rt] > mx[rt] + Y::TH;
    }
    if (__ballot(up)) {
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        float t = fmaxf(tm[rt], __shfl_xor(tm[rt], 16, 64));
        t = fmaxf(t, __shfl_xor(t, 32, 64));
        const float mn = fmaxf(mx[rt], t);
        const float al = __builtin_amdgcn_exp2f(mx[rt] - mn);
        mx[rt] = mn;
        l[rt] *= al;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) o[rt][nt] *= al;
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      const float sub = mx[rt] - Y::OFF;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float p =
            __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][e >> 2][e & 3], A.c, -sub));
        s[rt][e >> 2][e & 3] = p;
        l[rt] += p;
      }
    }
    if (NODE) {
      // A value that is not finite must reach the rows that see its node and no
      // other (0 * NaN is NaN): such nodes leave the product and are added row
      // by row.
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
        float* ps = reinterpret_cast<float*>(sh + QF + w * LDS_P);  // [ROWS][TR_KEYS + 1]
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
          const int node = node0 + 16 * (j >> 4) + 4 * (j & 3) + (j >> 2 & 3);
          const uint16_t* vrow = vn + (size_t)node * A.ld_n + 4 * NT * g;
#pragma unroll
          for (int rt = 0; rt < RT; rt++) {
            const float p = ps[(rt * 16 + m) * (TR_KEYS + 1) + j];
            if (!(sees[rt] >> node & 1ull)) continue;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
              for (int nt = 0; nt < NT; nt++)
                o[rt][nt][i] = __builtin_fmaf(p, Y::widen(vrow[NT * i + nt]), o[rt][nt][i]);
          }
        }
      }
    }
    tr_u32x4 pf[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        pf[rt][j] = Y::pack(s[rt][j >> 1][2 * (j & 1)], s[rt][j >> 1][2 * (j & 1) + 1]);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      tr_u32x4 vt;
#pragma unroll
      for (int j = 0; j < 4; j++)
        vt[j] = __builtin_amdgcn_perm(vr[2 * j + 1][nt >> 1], vr[2 * j][nt >> 1],
                                      nt & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int rt = 0; rt < RT; rt++) o[rt][nt] = Y::mfma(vt, pf[rt], o[rt][nt]);
    }
  };
  int tl = tl0 + w;
  for (; tl < tl1 && tl < nc; tl += TR_WAVES) {
    const int p0 = tl * TR_KEYS;
    const uint16_t* kp[2];
    const uint16_t* vp[2];
    uint32_t on = 0u;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      // positions past the last: the last one's (or its four's) again
      const int pk = p0 + 16 * t + m < ctx ? p0 + 16 * t + m : ctx - 1;
      const int v0 = p0 + 16 * t + 4 * g, v1 = (ctx - 1) & ~3, pv = v0 < v1 ? v0 : v1;
      // (four positions from a multiple of four share a page)
      int64_t ks, vs;
      pz_pages_slot(A.pages, table, pk, &ks);
      const bool vok = pz_pages_slot(A.pages, table, pv, &vs);
      kp[t] = kc + ks * A.ld;
      vp[t] = vc + vs * A.ld;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (vok && v0 + i < ctx) on |= 1u << (4 * t + i);
    }
    tile(std::false_type{}, kp, [&](int e) { return vp[e >> 2] + (e & 3) * A.ld; }, on,
         __ballot(on != 0xffu) == 0ull, 0);
  }
  for (; tl < tl1; tl += TR_WAVES) {
    const int node0 = (tl - nc) * TR_KEYS;
    // (past the last node: the last one again)
    auto node = [&](int i) { return (size_t)(node0 + i < nn ? node0 + i : nn - 1) * A.ld_n; };
    const uint16_t* kp[2] = {kn + node(m), kn + node(16 + m)};
    auto key = [&](int e) { return 16 * (e >> 2) + 4 * g + (e & 3); };
    uint32_t on = 0u;
#pragma unroll
    for (int e = 0; e < 8; e++) on |= node0 + key(e) < nn ? 1u << e : 0u;
    tile(std::true_type{}, kp, [&](int e) { return vn + node(key(e)); }, on, false, node0);
  }

  // the waves' results meet: common maximum, then the sums
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    l[rt] += __shfl_xor(l[rt], 16, 64);
    l[rt] += __shfl_xor(l[rt], 32, 64);
    if (g == 0) {
      mls[w][rt * 16 + m][0] = mx[rt];
      mls[w][rt * 16 + m][1] = l[rt];
    }
  }
  __syncthreads();  // (and Q is done with)
  float mt[RT], lt[RT];
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    mt[rt] = mls[0][rt * 16 + m][0];
#pragma unroll
    for (int i = 1; i < TR_WAVES; i++) mt[rt] = fmaxf(mt[rt], mls[i][rt * 16 + m][0]);
    lt[rt] = 0.0f;
#pragma unroll
    for (int i = 0; i < TR_WAVES; i++)
      lt[rt] += mls[i][rt * 16 + m][1] * __builtin_amdgcn_exp2f(mls[i][rt * 16 + m][0] - mt[rt]);
    const float al = __builtin_amdgcn_exp2f(mx[rt] - mt[rt]);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) o[rt][nt] *= al;
  }
  auto at = [&](int buf, int ch) {
    return reinterpret_cast<tr_f32x4*>(sh + buf * BUF + (ch * 64 + lane) * 16);
  };
#pragma unroll
  for (int half = 2; half >= 1; half >>= 1) {
    if (w >= half && w < 2 * half)
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) *at(w - half, rt * NT + nt) = o[rt][nt];
    __syncthreads();
    if (w < half)
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) o[rt][nt] += *at(w, rt * NT + nt);
    __syncthreads();
  }
  if (w != 0) return;
  const size_t unit = (size_t)bh * A.nblk + blk;
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    const int r = row0 + rt * 16 + m;
    if (A.S > 1) {
      if (g == 0) {
        float* ml = A.ml + ((unit * A.S + sp) * ROWS + rt * 16 + m) * 2;
        ml[0] = mt[rt];
        ml[1] = lt[rt];
      }
      tr_f32x4* part = reinterpret_cast<tr_f32x4*>(A.part) + (unit * A.S + sp) * CH * 64;
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int f = 0; f < NT / 4; f++)
          part[((rt * 4 + i) * (NT / 4) + f) * 64 + lane] =
              tr_f32x4{o[rt][4 * f][i], o[rt][4 * f + 1][i], o[rt][4 * f + 2][i],
                       o[rt][4 * f + 3][i]};
    } else if (r < rows) {
      // nothing seen: l is 0 and so is the result
      const float inv = lt[rt] == 0.0f ? 0.0f : 1.0f / lt[rt];
      const int t = r / A.group, hq = h * A.group + (r - t * A.group);
      uint16_t* out = A.out + ((size_t)b * A.T + t) * A.ld_out + (size_t)hq * D + 4 * NT * g;
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int f = 0; f < NT / 4; f++)
          tr_store4<TYPE>(out + NT * i + 4 * f,
                          tr_f32x4{o[rt][4 * f][i], o[rt][4 * f + 1][i], o[rt][4 * f + 2][i],
                                   o[rt][4 * f + 3][i]} *
                              inv);
    }
  }
}

// Adds up the splits of one unit (key head and row block): a wave per float4 of
// every lane's results.
template <int TYPE, int D, int RT>
__global__ __launch_bounds__(64 * TR_WAVES) void k_tree_join(const TreeArgs A) {
  constexpr int NT = D / 16, ROWS = 16 * RT, CH = RT * NT;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int64_t job = (int64_t)blockIdx.x * TR_WAVES + w;
  const int64_t unit = job / CH;
  const int ch = (int)(job - unit * CH);
  if (unit >= (int64_t)A.B * A.n_kv * A.nblk) return;
  const int blk = (int)(unit % A.nblk), bh = (int)(unit / A.nblk), h = bh % A.n_kv,
            b = bh / A.n_kv;
  const int rows = tr_nodes(A, b) * A.group;
  const int rt = ch / NT, i = ch % NT / (NT / 4), f = ch % (NT / 4);
  const int r = blk * ROWS + rt * 16 + m;
  if (blk * ROWS >= rows) return;  // (its workgroups wrote nothing)
  const float* ml = A.ml + ((size_t)unit * A.S * ROWS + rt * 16 + m) * 2;
  float mt = TR_LOW;
  for (int s = 0; s < A.S; s++) mt = fmaxf(mt, ml[(size_t)s * ROWS * 2]);
  float lt = 0.0f;
  tr_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  const tr_f32x4* part =
      reinterpret_cast<const tr_f32x4*>(A.part) + ((size_t)unit * A.S * CH + ch) * 64 + lane;
#pragma unroll 4
  for (int s = 0; s < A.S; s++) {
    const float f2 = __builtin_amdgcn_exp2f(ml[(size_t)s * ROWS * 2] - mt);
    lt += ml[(size_t)s * ROWS * 2 + 1] * f2;
    o += part[(size_t)s * CH * 64] * f2;
  }
  if (r >= rows) return;
  const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
  const int t = r / A.group, hq = h * A.group + (r - t * A.group);
  tr_store4<TYPE>(A.out + ((size_t)b * A.T + t) * A.ld_out + (size_t)hq * D + 4 * NT * g + NT * i +
                      4 * f,
                  o * inv);
}

template <int TYPE, int D, int RT>
int launch(pz_sampler* s, TreeArgs& A) {
  constexpr int ROWS = 16 * RT;
  A.nblk = (A.T * A.group + ROWS - 1) / ROWS;
  const int64_t units = (int64_t)A.B * A.n_kv * A.nblk;
  // splits: four workgroups a CU, each with two tiles a wave at least, and
  // results that fit the workspace
  const int64_t tiles = ((int64_t)A.pages.max_blocks << A.pages.shift) / TR_KEYS + (A.T + TR_KEYS - 1) / TR_KEYS;
  int64_t S = (4 * (int64_t)s->n_cu + units - 1) / units;
  const int64_t most = tiles / (2 * TR_WAVES);
  S = S < most ? S : most;
  const int64_t room = (int64_t)(PZ_TREE_WS / ((size_t)ROWS * (D + 2) * sizeof(float))) / units;
  S = S < room ? S : room;
  S = S < 64 ? S : 64;
  A.S = S < 1 ? 1 : (int)S;
  const int64_t groups = (int64_t)A.B * A.n_kv * A.S;
  const int64_t grid = (groups + 7) / 8 * 8 * A.nblk;
  if (grid > INT32_MAX) return fail(s, PZ_ERANGE, "B=%d sequences of T=%d nodes", A.B, A.T);
  A.part = static_cast<float*>(s->tree_dev);
  A.ml = A.part + (size_t)units * A.S * ROWS * D;
  hipLaunchKernelGGL((k_tree<TYPE, D, RT>), dim3((unsigned)grid), dim3(64 * TR_WAVES), 0,
                     s->stream, A);
  PZ_HIP(s, hipGetLastError());
  if (A.S > 1) {
    const int64_t jobs = units * RT * (D / 16);
    hipLaunchKernelGGL((k_tree_join<TYPE, D, RT>), dim3((unsigned)((jobs + TR_WAVES - 1) / TR_WAVES)),
                       dim3(64 * TR_WAVES), 0, s->stream, A);
    PZ_HIP(s, hipGetLastError());
  }
  return PZ_OK;
}

template <int TYPE, int D>
int run_rows(pz_sampler* s, TreeArgs& A) {
  const int rows = A.T * A.group;
  if (rows <= 16) return launch<TYPE, D, 1>(s, A);
  if (rows <= 32 || D == 256) return launch<TYPE, D, 2>(s, A);
  return launch<TYPE, D, D == 256 ? 2 : 4>(s, A);
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
  if (!pz_pages_slot(A.pages, A.blocks + (size_t)b * A.pages.max_blocks, (int)p, &slot)) return;
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
  if ((int64_t)B * T > INT32_MAX) return fail(s, PZ_ERANGE, "B=%d sequences of T=%d nodes", B, T);
  if (B == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  const TreeArgs A = args_of(cache, d_kn, d_vn, ld_n, B, T);
  hipLaunchKernelGGL(k_append, dim3((unsigned)B * (unsigned)T), dim3(256), 0, s->stream, A,
                     cache->n_kv_heads * cache->head_dim, d_take, d_count);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}
