// pz_tree.hip -- attention of drafted tokens over a paged cache and over each
// other along a tree (pz_tree_attention; its kernels: pz_treedev.h), and the accepted
// tokens' way into the pages (pz_cache_append).
#include <hip/hip_runtime.h>

#include "../../include/pz_sampler.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"
#include "pz_treedev.h"
#include "pz_treeplan.h"

namespace {

template <int TYPE, int D, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(D * (1 + RT) >= 512 ? 1 : 2, 8))) void
k_tree(const WholeArgs A) {
  __shared__ TrLds<D, RT, WAVES> lds;
  tr_narrow<TYPE, D, RT, WAVES>(A, blockIdx.x, threadIdx.x, lds);
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
k_tree_wide(const WholeArgs A) {
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
  TrJob J;
  if (!tr_job<WAVES * ROWS>(A, blockIdx.x, lane, A.nblk / WAVES, &J)) return;
  const int b = J.b, h = J.h, sp = J.sp, rows = J.rows, row0 = (J.blk * WAVES + w) * ROWS;
  const int node0 = J.node0;
  const int ctx = pz_pages_len(A.pages, A.len[b]), nn = tr_nodes(A, b);
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
      qf[rt][ks] = *reinterpret_cast<const tr_u32x4*>(A.q + (size_t)(node0 + t) * A.ld_q +
                                                      (size_t)hq * D + ks * 32 + 8 * g);
    sees[rt] = A.tree ? A.tree[node0 + t] : ~0ull >> (63 - t);
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
      const int first = (tl - nc) * TR_KEYS;
      uint32_t on = 0u, vr[8][NW];
#pragma unroll
      for (int e = 0; e < 8; e++)
        on |= first + 16 * (e >> 2) + 4 * g + (e & 3) < nn ? 1u << e : 0u;
      uint64_t of_tile[RT];
#pragma unroll
      for (int rt = 0; rt < RT; rt++) of_tile[rt] = sees[rt] >> first;
      scores(buf);
#pragma unroll
      for (int e = 0; e < 8; e++)
        fetch(sh + buf * STG + TILE + (16 * (e >> 2) + 4 * g + (e & 3)) * D * 2 + m * NT * 2, vr[e]);
      R.drop(on, [&](int rt, int key) { return of_tile[rt] >> key & 1ull; });
      R.blank(on, vr);
      R.weights();
      R.odd_values(vr, of_tile, vn + (size_t)first * A.ld_n, A.ld_n,
                   reinterpret_cast<float*>(sh + NS * STG + w * LDS_P));
      R.values(vr);
    }
    next();
  }
  lm_wait<0>();
  if (idle) return;
  const size_t unit = ((size_t)b * A.n_kv + h) * A.nblk + J.blk * WAVES + w;
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
    uint16_t* out = A.out + (size_t)(node0 + t) * A.ld_out + (size_t)hq * D + 4 * NT * g;
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

constexpr int TR_JOIN = 4;  // waves of a joining workgroup

// Adds up the splits of one unit (key head and row block): for each float4 of a
// lane's results WAVES waves, which take the splits in turn; TR_JOIN / WAVES of
// them in a workgroup.  (One wave where the splits are few enough to be under way
// together: 512 units of 4 splits of 32 rows 20
// -> 11 us.)
template <int TYPE, int D, int RT, int WAVES>
__global__ __launch_bounds__(64 * TR_JOIN) void k_tree_join(const WholeArgs A) {
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
int plan(pz_sampler* s, WholeArgs& A, int64_t units, int64_t tiles, int64_t want) {
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
int join(pz_sampler* s, const WholeArgs& A, int64_t units) {
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
int narrow(pz_sampler* s, WholeArgs& A, int64_t tiles, int64_t want) {
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
int wide(pz_sampler* s, WholeArgs& A, int64_t tiles, int64_t want) {
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
int run_rows(pz_sampler* s, WholeArgs& A) {
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
int run(pz_sampler* s, WholeArgs& A, int D) {
  if (D == 64) return run_rows<TYPE, 64>(s, A);
  if (D == 128) return run_rows<TYPE, 128>(s, A);
  return run_rows<TYPE, 256>(s, A);
}

// ---- append --------------------------------------------------------------------
// One workgroup per node: its row of keys and its row of values, 16 bytes a
// thread.
__global__ __launch_bounds__(256) void k_append(const WholeArgs A, int row, const int32_t* take,
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

WholeArgs args_of(const pz_kv_cache* c, const void* d_kn, const void* d_vn, long ld_n, int B,
                 int T) {
  WholeArgs A = {};
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

int pz_tree_workspace(pz_sampler* s) {
  if (!s->tree_dev && hipMalloc(&s->tree_dev, PZ_TREE_WS) != hipSuccess) {
    s->tree_dev = nullptr;
    (void)hipGetLastError();
    return fail(s, PZ_ENOMEM, "tree attention's workspace");
  }
  return PZ_OK;
}

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
  const int rc = pz_tree_workspace(s);
  if (rc != PZ_OK) return rc;
  WholeArgs A = args_of(cache, d_kn, d_vn, ld_n, B, T);
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
  const WholeArgs A = args_of(cache, d_kn, d_vn, ld_n, B, T);
  hipLaunchKernelGGL(k_append, dim3((unsigned)B * (unsigned)T), dim3(256), 0, s->stream, A,
                     cache->n_kv_heads * cache->head_dim, d_take, d_count);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}
