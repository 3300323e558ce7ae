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
  hipLaunchKernelGGL((k_tree<TYPE, D, RT, WAVES, WholeArgs>), dim3((unsigned)(groups * A.nblk)),
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
  hipLaunchKernelGGL((k_tree_wide<TYPE, D, RT, WholeArgs>), dim3((unsigned)(groups * nwg)),
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
