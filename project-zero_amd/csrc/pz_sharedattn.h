// pz_sharedattn.h -- the prefix's part of pz_prefix_attention where many rows share it.
//
// As k_tree_wide (pz_treedev.h): S^T = K Q^T and O^T = V^T P^T on 16x16x32 matrix
// instructions, keys and values through LDS, running maximum and sum of a row in the lanes
// that hold it.  What is different, since nothing but one prefix's positions comes by:
//
//   * a tile is 64 keys, and a step of it has two phases: the products (the last tile's
//     weights with its values, this one's keys with the queries) and the weights.  The
//     eight waves are two groups, one wave of each on every SIMD, that work half a step
//     apart: while one is at its products, the other is at its weights.  (In one phase
//     together the matrix cores and the vector unit take turns.)
//   * the values come out of LDS transposed (ds_read_b64_tr_b16: 16 lanes read 4 keys x 16
//     d and get 4 keys of one d each) in place of byte permutes.  The 32-byte pieces of a
//     row are exchanged by the row's number, so that 8 rows lie in 8 places.
//
// Stage j of the ring holds the keys of tile j and the values of tile j - 1, which the
// products of step j take.  With intervals between barriers, group 0 makes the products of
// step t in interval 2 t and its weights in 2 t + 1, group 1 in 2 t + 1 and 2 t + 2.  So a
// stage's slot is free from interval 2 t + 2 on, and every wave asks for its share of stage
// t + SH_STAGES among its products of step t + 1; and it waits for its share of stage t + 1
// before the barrier that interval 2 t + 2 begins with.
//
// Bound by issue: a tile of 64 keys x 256 rows takes a CU 1.9 us, some 4000 cycles, 2048 of
// them products and 1570 weights on each SIMD.  The vector instructions of one wave run at
// little more than half their rate while another's products keep the matrix cores busy, so
// that the two phases hide each other only in part.  1 prefix of 32768 positions, 256
// sequences of one token, 32 heads over 8 of 128 (137 GFLOP): 169 us with the maximum of every
// tile's scores, 155 with it looked for only where the weights' sum tells.  (256 sequences
// that have up to 512 positions of their own, too: 229 us with one phase and a launch for
// either part, 181 so.)
#pragma once
#include "pz_treedev.h"

namespace {

constexpr int SH_KEYS = 64;    // keys of a tile
constexpr int SH_STAGES = 4;   // of the ring
constexpr int SH_ROWS = 32;    // rows of a wave
constexpr int SH_WAVES = 8;
constexpr int SH_AHEAD = 6;    // fragments that are read ahead of their products

typedef short sh_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char* sh_lds;

// Four keys of one d: keys from p's row on (lane l: row l / 4 % 4, 8 bytes at l % 4).
__device__ __forceinline__ tr_u32x2 sh_transposed(sh_lds p) {
  return __builtin_bit_cast(
      tr_u32x2,
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sh_s16x4*)p));
}

// No instruction crosses this, nor the barrier within.
__device__ __forceinline__ void sh_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int D>
struct ShLds {
  __align__(16) char sh[SH_STAGES * 2 * SH_KEYS * D * 2];
  int64_t tab[TR_ENTRIES];
  int broken;
};

// Workgroup `block` of 64 SH_WAVES threads.
template <int TYPE, int D>
__device__ __forceinline__ void sh_attend(const SharedArgs& A, uint32_t block, ShLds<D>& buf) {
  typedef TrType<TYPE> Y;
  constexpr int RT = SH_ROWS / 16, KS = D / 32, NT = D / 16, KT = SH_KEYS / 16, NS = SH_STAGES;
  constexpr int TILE = SH_KEYS * D * 2, STG = 2 * TILE;  // bytes: of a tile's keys, of a stage
  constexpr int LN = TILE / 1024, PK = LN / SH_WAVES;    // 1 KiB loads of a tile's keys, of a wave
  constexpr int PR = D / 8, RPI = 64 / PR;               // 16-byte pieces of a row, rows of a load
  static_assert(LN % SH_WAVES == 0 && RPI <= 8 && D <= 128, "");
  char* const sh = buf.sh;
  int64_t* const tab = buf.tab;
  int& broken = buf.broken;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  TrJob J;
  if (!tr_job<SH_WAVES * SH_ROWS>(A, block, lane, A.nblk, &J)) return;
  const int h = J.h, sp = J.sp, rows = J.rows, row0 = (J.blk * SH_WAVES + w) * SH_ROWS;
  const bool idle = row0 >= rows;  // (a wave past the last row loads only)
  const int ctx = pz_pages_len(A.pages, A.len[J.b]);
  // (splits are counted in tiles of TR_KEYS; where a share is an odd number of them, the last
  // tile here of every split is half full, as that of a prefix may be)
  const int chunk = tr_chunk(A, J.b, lane), ntl = tr_tiles(A, J.b);
  const int tl0 = sp * chunk, tl1 = ntl - tl0 < chunk ? ntl : tl0 + chunk;
  if (tl0 >= ntl) return;
  const int p0 = tl0 * TR_KEYS, p1 = tl1 * TR_KEYS < ctx ? tl1 * TR_KEYS : ctx;
  const int n = (p1 - p0 + SH_KEYS - 1) / SH_KEYS;  // tiles
  const uint16_t* kc = A.k + (size_t)h * D;
  const uint16_t* vc = A.v + (size_t)h * D;
  const int32_t* table = A.blocks + (size_t)J.b * A.pages.max_blocks;
  const sh_lds lds = (sh_lds)sh;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;

  // Where the range's pages begin, in bytes from the first one, in LDS; and whether they
  // are all there.
  const int e0 = p0 >> A.pages.shift;
  const uint32_t row_bytes = (uint32_t)A.ld * 2u;
  auto there = [&](int32_t id) { return (uint32_t)id < (uint32_t)A.pages.n_blocks; };
  auto page_at = [&](int32_t id) {
    return ((int64_t)(there(id) ? id : 0) << A.pages.shift) * (int64_t)row_bytes;
  };
  bool whole = true;
  for (int e = e0 + tid; e <= (p1 - 1) >> A.pages.shift; e += 64 * SH_WAVES) {
    const int32_t id = table[e];
    if (e - e0 < TR_ENTRIES) tab[e - e0] = page_at(id);
    whole = whole && there(id);
  }
  if (tid == 0) broken = 0;
  __syncthreads();
  if (!whole) broken = 1;
  __syncthreads();
  whole = broken == 0;
  // (a tile that is not: an entry from memory, whose wait is one for the ring's loads, too)
  auto exists = [&](int p) { return p < p1 && there(table[p >> A.pages.shift]); };
  auto full = [&](int t) { return whole && p0 + (t + 1) * SH_KEYS <= p1; };

  // Load i of this wave: rows (w PK + i) RPI .. of a tile.  Keys: piece ^ the row's number,
  // so that the 16 rows that are read together lie in 16 places; values: 32 bytes ^ it.
  const int lr = lane / PR, place = lane % PR;
  uint32_t koff[PK], voff[PK];
#pragma unroll
  for (int i = 0; i < PK; i++) {
    const int row = (w * PK + i) * RPI + lr;
    const int ks = D == 64 ? row >> 1 & 7 : row & 15;
    const int vs = D == 64 ? row >> 1 & 3 : row & 7;
    koff[i] = (uint32_t)lr * (uint32_t)A.ld * 2u + 16u * (uint32_t)(place ^ ks);
    voff[i] = (uint32_t)lr * (uint32_t)A.ld * 2u + 16u * (uint32_t)(place ^ (vs << 1));
  }
  // (positions past the last: the last one's rows again)
  auto pos_of = [&](int t, int i) {
    const int p = p0 + t * SH_KEYS + (w * PK + i) * RPI, last = (p1 - 1) & ~(RPI - 1);
    return p < last ? p : last;
  };
  auto clip = [&](int t) { return t < n ? t : n - 1; };
  // of the next stage to ask for: its keys' and its values' places, in bytes
  int64_t kpl[PK] = {}, vpl[PK] = {};
  uint32_t to = lds0;  // its slot
  auto ask = [&](int i) {  // load i of 2 PK
    const int k = i % PK;
    if (i < PK)
      lm_lds_load16<false>(reinterpret_cast<const char*>(kc) + kpl[k], koff[k],
                           to + (w * PK + k) * 1024);
    else
      lm_lds_load16<false>(reinterpret_cast<const char*>(vc) + vpl[k], voff[k],
                           to + TILE + (w * PK + k) * 1024);
  };
  // its pages' places, and on to the stage after it, which holds the keys of tile t
  auto pages_of = [&](int t, int64_t(&at)[PK]) {
#pragma unroll
    for (int i = 0; i < PK; i++) {
      const int e = (pos_of(clip(t), i) >> A.pages.shift) - e0;
      if (e < TR_ENTRIES) {
        at[i] = tab[e];
      } else {  // (past those in LDS)
        at[i] = page_at(table[e0 + e]);
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
      }
    }
  };
  auto go_on = [&](int t, const int64_t(&at)[PK]) {
#pragma unroll
    for (int i = 0; i < PK; i++) {
      const uint32_t low = __builtin_amdgcn_readfirstlane((int)(uint32_t)at[i]),
                     high = __builtin_amdgcn_readfirstlane((int)(at[i] >> 32));
      const uint32_t in = (uint32_t)pos_of(clip(t), i) & ((1u << A.pages.shift) - 1u);
      vpl[i] = kpl[i];
      kpl[i] = (int64_t)((uint64_t)high << 32 | low) + (int64_t)(uint64_t)(in * row_bytes);
    }
    to = to == lds0 + (NS - 1) * STG ? lds0 : to + STG;
  };

  tr_u32x4 qf[RT][KS];  // lane l: row l % 16, 8 d from 8 (l / 16) of 32
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    const int r = row0 + rt * 16 + m, rr = r < rows ? r : 0, t = rr / A.group,
              hq = h * A.group + (rr - t * A.group);
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
      qf[rt][ks] = *reinterpret_cast<const tr_u32x4*>(A.q + (size_t)(J.node0 + t) * A.ld_q +
                                                      (size_t)hq * D + ks * 32 + 8 * g);
  }
  // (arrived before the ring's loads, which the compiler does not see, are under way)
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  {
    int64_t at[PK];
    pages_of(0, at);
    go_on(0, at);
    to = lds0;
#pragma unroll
    for (int i = 0; i < PK; i++) vpl[i] = kpl[i];
    for (int j = 0; j < NS; j++) {
#pragma unroll
      for (int i = 0; i < 2 * PK; i++) ask(i);
      pages_of(j + 1, at);
      go_on(j + 1, at);
    }
  }

  tr_f32x4 o[RT][NT], s[RT][KT];
  tr_u32x4 pf[RT][KT / 2];  // weights: keys 32 c + 16 (j / 2) + 4 g + 2 (j % 2) .. + 1
  float mx[RT], l[RT], nb[RT];
  bool far = true;
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    mx[rt] = TR_LOW;
    nb[rt] = Y::OFF;
    l[rt] = 0.0f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) o[rt][nt] = tr_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kt = 0; kt < KT; kt++) s[rt][kt] = tr_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < KT / 2; c++) pf[rt][c] = tr_u32x4{0u, 0u, 0u, 0u};
  }
  // a lane's place in a tile: key 16 t + m, pieces ks * 4 + g; key 16 t + 4 g + l / 4 % 4
  const int vrow = 4 * g + (lane >> 2 & 3);
  const uint32_t vat = (uint32_t)vrow * D * 2 + ((D == 64 ? vrow >> 1 & 3 : vrow & 7) << 5) +
                       (lane & 3) * 8;
  const uint32_t kat = (uint32_t)m * D * 2 + ((g ^ (D == 64 ? m >> 1 & 7 : m)) << 4);

  auto tie = [&]() {  // (what a phase made is made before the next)
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      asm volatile("" : "+v"(s[rt][0]), "+v"(s[rt][1]), "+v"(s[rt][2]), "+v"(s[rt][3]));
      asm volatile("" : "+v"(pf[rt][0]), "+v"(pf[rt][1]));
#pragma unroll
      for (int nt = 0; nt < NT; nt++) asm volatile("" : "+v"(o[rt][nt]));
    }
  };
  // The products of a step: with the values, fragment (nt, c), then with the keys, fragment
  // (kt, ks), each read SH_AHEAD fragments before its products; those that add up to one
  // result as far apart as can be.
  // (A step with both also asks for a stage, one load now and then.)
  auto products = [&](int slot, auto pv, auto qk) {
    constexpr bool PV = decltype(pv)::value, QK = decltype(qk)::value;
    constexpr int NV = PV ? NT * KT / 2 : 0, NF = NV + (QK ? KT * KS : 0), F = SH_AHEAD;
    const sh_lds st = lds + slot * STG;
    // (before the other group's vector instructions, which would keep the products, few as
    // they are, from being issued)
    __builtin_amdgcn_s_setprio(1);
    tr_u32x4 f[F];
    auto read = [&](int i) {
      if (i < NV) {
        const int nt = i % NT, c = i / NT;
        const sh_lds p = st + TILE + (vat ^ (uint32_t)(nt << 5)) + c * 32 * D * 2;
        const tr_u32x2 x = sh_transposed(p), y = sh_transposed(p + 16 * D * 2);
        f[i % F] = tr_u32x4{x[0], x[1], y[0], y[1]};
      } else {
        const int kt = (i - NV) % KT, ks = (i - NV) / KT;
        f[i % F] = *reinterpret_cast<__attribute__((address_space(3))) tr_u32x4*>(
            st + (kat ^ (uint32_t)(ks << 6)) + kt * 16 * D * 2);
      }
    };
#pragma unroll
    for (int i = 0; i < F; i++) read(i);
#pragma unroll
    for (int i = 0; i < NF; i++) {
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        if (i < NV) {
          const int nt = i % NT, c = i / NT;
          o[rt][nt] = Y::mfma(f[i % F], pf[rt][c], o[rt][nt]);
        } else {
          const int kt = (i - NV) % KT, ks = (i - NV) / KT;
          s[rt][kt] = Y::mfma(f[i % F], qf[rt][ks],
                              ks ? s[rt][kt] : tr_f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        }
      }
      if (i + F < NF) read(i + F);
      if (PV && QK && i % (NF / (2 * PK)) == NF / (4 * PK)) ask(i / (NF / (2 * PK)));
    }
    // (the compiler would read each fragment right before its products)
    constexpr int MFMA = 0x8, READ = 0x100;
#pragma unroll
    for (int i = 0; i < F; i++) {
      if (i < NV)
        __builtin_amdgcn_sched_group_barrier(READ, 2, 0);
      else
        __builtin_amdgcn_sched_group_barrier(READ, 1, 0);
    }
#pragma unroll
    for (int i = 0; i < NF; i++) {
      __builtin_amdgcn_sched_group_barrier(MFMA, RT, 0);
      if (i + F < NF) {
        if (i + F < NV)
          __builtin_amdgcn_sched_group_barrier(READ, 2, 0);
        else
          __builtin_amdgcn_sched_group_barrier(READ, 1, 0);
      }
    }
    tie();
    __builtin_amdgcn_s_setprio(0);
  };
  // the weights of tile t
  auto weights = [&](int t) {
    float of[RT];  // the sums of this tile's
    if (!full(t)) {
#pragma unroll
      for (int kt = 0; kt < KT; kt++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const bool on = exists(p0 + t * SH_KEYS + 16 * kt + 4 * g + i);
#pragma unroll
          for (int rt = 0; rt < RT; rt++) s[rt][kt][i] = on ? s[rt][kt][i] : -__builtin_inff();
        }
    }
    // m is raised only where a lane's weights of a row pass 2^TH (or are NaN), which their
    // sum tells without the maximum of the scores: then the weights are made again.
    auto weigh = [&]() {
      bool pass = false;
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        float sum = 0.0f;
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
          tr_f32x4 p;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float x = s[rt][kt][i];
            p[i] = __builtin_amdgcn_exp2f(far ? __builtin_fmaf(x - mx[rt], A.c, Y::OFF)
                                              : __builtin_fmaf(x, A.c, nb[rt]));
            sum += p[i];
          }
          pf[rt][kt >> 1][2 * (kt & 1)] = Y::pack(p[0], p[1]);
          pf[rt][kt >> 1][2 * (kt & 1) + 1] = Y::pack(p[2], p[3]);
        }
        pass |= !(sum <= Y::MUCH);
        of[rt] = sum;
      }
      return __ballot(pass) != 0;
    };
    if (weigh()) {
      bool out = false;
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        float top = s[rt][0][0];
#pragma unroll
        for (int e = 1; e < 4 * KT; e++)
          top = __builtin_elementwise_maximum(top, s[rt][e >> 2][e & 3]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float mn = fmaxf(mx[rt], top);
        const float al = tr_lift(mx[rt], mn, A.c);
        mx[rt] = mn;
        l[rt] *= al;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) o[rt][nt] *= al;
        out |= !(fabsf(mn * A.c) <= TR_NEAR);
      }
      far = __ballot(out) != 0;
#pragma unroll
      for (int rt = 0; rt < RT; rt++) nb[rt] = Y::OFF - mx[rt] * A.c;
      weigh();
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) l[rt] += of[rt];
    tie();
  };
  // At the start of interval 2 t + 2: what lies in the place of a position of tile t that
  // does not exist may be anything, and 0 times it is not 0.
  auto blank = [&](int t, int slot) {  // slot: of stage t + 1
    if (full(t)) return;
    for (int i = tid; i < TILE / 16; i += 64 * SH_WAVES) {
      if (!exists(p0 + t * SH_KEYS + i / PR))
        *reinterpret_cast<tr_u32x4*>(sh + slot * STG + TILE + i * 16) = tr_u32x4{0u, 0u, 0u, 0u};
    }
    __syncthreads();
  };
  constexpr int L = 2 * PK;  // loads of a wave for a stage
  lm_wait<(NS - 1) * L>();
  sh_barrier();
  int slot = 0;
  auto after = [&](int i) { return i + 1 == NS ? 0 : i + 1; };
  constexpr std::true_type YES = {};
  constexpr std::false_type NO = {};
  // a step with both products; the stage t - 1 + NS is asked for
  auto step = [&](int t) {
    int64_t at[PK];
    pages_of(t + NS, at);
    if (!idle) {
      products(slot, YES, YES);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * PK; i++) ask(i);
    }
    go_on(t + NS, at);
  };
  if (w < SH_WAVES / 2) {
    if (!idle) products(0, NO, YES);
    sh_barrier();
    if (!idle) weights(0);
    lm_wait<(NS - 2) * L>();
    sh_barrier();
#pragma clang loop unroll(disable)
    for (int t = 1; t < n; t++) {
      slot = after(slot);
      blank(t - 1, slot);
      step(t);
      sh_barrier();
      if (!idle) weights(t);
      lm_wait<(NS - 2) * L>();
      sh_barrier();
    }
    slot = after(slot);
    blank(n - 1, slot);
    if (!idle) products(slot, YES, NO);
    sh_barrier();
    sh_barrier();  // (group 1 has as many)
  } else {
    sh_barrier();
    if (!idle) products(0, NO, YES);
    lm_wait<(NS - 2) * L>();
    sh_barrier();
    slot = after(slot);
    blank(0, slot);
    if (!idle) weights(0);
    sh_barrier();
#pragma clang loop unroll(disable)
    for (int t = 1; t < n; t++) {
      step(t);
      lm_wait<(NS - 2) * L>();
      sh_barrier();
      slot = after(slot);
      blank(t, slot);
      if (!idle) weights(t);
      sh_barrier();
    }
    if (!idle) products(slot, YES, NO);
    sh_barrier();
  }
  lm_wait<0>();
  if (idle) return;
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    float sum = l[rt];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    const int r = row0 + rt * 16 + m;
    if (r >= rows) continue;
    const int t = r / A.group, hq = h * A.group + (r - t * A.group);
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
      tr_part<D>(A, sp, (size_t)(J.node0 + t) * (A.n_kv * A.group) + hq, 16 * nt + 4 * g,
                 o[rt][nt], mx[rt], sum);
  }
}

}  // namespace
