// pz_prefix.hip -- attention of sequences that share prefixes (pz_prefix_attention).
//
//   out[r] = sum_p softmax_p(scale q[r] . k[p]) v[p],  p over the positions of the
//   prefix of r's sequence, its own cached positions and the nodes that r's node sees.
//
// The softmax comes in parts that meet at the end, each with its maximum m, its sum l
// and its sum of values (pz_treedev.h): the prefix's, where the rows of all sequences
// that share it meet each key, in splits of the longest prefix, and each sequence's
// own.  k_prefix_join adds them up:
//   M = max m_i,  out = sum_i 2^(c (m_i - M)) o_i / sum_i 2^(c (m_i - M)) l_i.
// Both parts are one launch: where few rows share a prefix memory bounds both, and where
// many do the products bound the prefix's part, memory the others.  32 heads over 8 of 128,
// bf16, kernel and join in us:
//   1 prefix of 500 positions, 4 beams of up to 40 of their own: 8.4 + 3.9, the launches and
//     one tile's way through; 18 as two launches and a join
//   8 of up to 4096, 8 beams each (119 MB): 33 + 5.5, 3.6 TB/s in the first; twice the
//     splits 4 us more, half of them 7
//   1 of up to 32768, 256 sequences of up to 512 (104 GFLOP, 374 MB): 176 + 10
// The weights' rounding to 16 bits for their product with the values takes results to 2.1e-3 to
// 2.3e-3 of their norm from 64 bits in bf16 (1.65e-3 rounded once from 32 bits), to 2.8e-4 in
// fp16 (2.1e-4).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/pz_sampler.h"
#include "pz_prefixplan.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"
#include "pz_sharedattn.h"
#include "pz_treedev.h"

namespace {

// The prefix of the launch's sequence b: -1 where it has none (wave-uniform).
__device__ __forceinline__ int pf_prefix_of(const SharedArgs& P, int b, int lane) {
  if (!P.first) return (b + P.b0) / P.each;
  for (int i0 = 0; i0 < P.B; i0 += 64) {
    bool it = false;
    if (i0 + lane < P.B) {
      int lo;
      const int n = tr_sharers(P, i0 + lane, &lo);
      it = lo <= b && b - lo < n;
    }
    const uint64_t any = __ballot(it);
    if (any) return i0 + __ffsll((unsigned long long)any) - 1;
  }
  return -1;
}

// A wave for each head of a node: D / 4 lanes with four results each, 256 / D splits at
// a time.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void k_prefix_join(const OwnArgs A, const SharedArgs P) {
  constexpr int LANES = D / 4, AT = 64 / LANES;
  const int lane = threadIdx.x & 63;
  const int n_heads = A.n_kv * A.group;
  const size_t row = (size_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= A.R) return;
  const int node = (int)(row / (unsigned)n_heads), hq = (int)(row - (size_t)node * n_heads);
  const int b = node / A.T, t = node - b * A.T;
  if (t >= tr_nodes(A, b)) return;
  const int i = pf_prefix_of(P, b, lane);
  int ns = 0;  // splits of the prefix
  if (i >= 0) {
    const int chunk = tr_chunk(P, i, lane);
    ns = (tr_tiles(P, i) + chunk - 1) / chunk;
  }
  const int chunk = tr_chunk(A, b, lane), no = (tr_tiles(A, b) + chunk - 1) / chunk;
  const int at = lane / LANES, d = lane % LANES * 4;
  float mt = TR_LOW, lt = 0.0f;
  tr_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](float m, float l, tr_f32x4 v) {
    const float mn = fmaxf(mt, m), al = tr_lift(mt, mn, A.c), e = tr_lift(m, mn, A.c);
    mt = mn;
    lt = lt * al + l * e;
    o = o * al + v * e;
  };
  for (int k = at; k < ns + no; k += AT) {
    const size_t slot = (size_t)(k < ns ? P.slot + k : A.slot + k - ns) * A.R + row;
    add(A.ml[2 * slot], A.ml[2 * slot + 1],
        *reinterpret_cast<const tr_f32x4*>(A.part + slot * D + d));
  }
#pragma unroll
  for (int k = LANES; k < 64; k <<= 1) {
    const float m = __shfl_xor(mt, k, 64), l = __shfl_xor(lt, k, 64);
    tr_f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = __shfl_xor(o[e], k, 64);
    add(m, l, v);
  }
  // a sum of 0: nothing attended (zeros), or every score -infinity (NaN)
  float inv = tr_inverse(A, b, t, lt);
  if (lt == 0.0f && i >= 0) {
    const int ctx = pz_pages_len(P.pages, P.len[i]);
    for (int e = 0; (int64_t)e << P.pages.shift < ctx; e++)
      if ((uint32_t)P.blocks[(size_t)i * P.pages.max_blocks + e] < (uint32_t)P.pages.n_blocks)
        inv = __builtin_nanf("");
  }
  if (at == 0) tr_store4<TYPE>(A.out + (size_t)node * A.ld_out + (size_t)hq * D + d, o * inv);
}

// Splits of `wgs` workgroups' work of up to `tiles` tiles: a workgroup a CU, and
// TR_SHARE tiles for each at least.
int splits(const pz_sampler* s, int64_t wgs, int64_t tiles, int64_t room) {
  int64_t S = (s->n_cu + wgs - 1) / wgs;
  S = S < tiles / TR_SHARE ? S : tiles / TR_SHARE;
  S = S < room ? S : room;
  S = S < 64 ? S : 64;
  return (int)(S < 1 ? 1 : S);
}

template <class ARGS>
void share_out(ARGS& A, int64_t tiles, int S) {
  A.chunk = (int)((tiles + S - 1) / S);
  A.S = (int)((tiles + A.chunk - 1) / A.chunk);
}

// The prefixes' part and the sequences' own in one launch: the first `shared` workgroups
// and the others.
template <int TYPE, int D, int RTS, int RTO>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D * (1 + (RTS > RTO ? RTS : RTO)) >= 512 ? 1 : 2, 8))) void
k_prefix(const SharedArgs P, const OwnArgs A, uint32_t shared) {
  typedef TrLds<D, RTS, 4> S;
  typedef TrLds<D, RTO, 4> O;
  __shared__ __align__(16) char buf[sizeof(S) > sizeof(O) ? sizeof(S) : sizeof(O)];
  if (blockIdx.x < shared)
    tr_narrow<TYPE, D, RTS, 4>(P, blockIdx.x, threadIdx.x, *reinterpret_cast<S*>(buf));
  else
    tr_narrow<TYPE, D, RTO, 4>(A, blockIdx.x - shared, threadIdx.x, *reinterpret_cast<O*>(buf));
}

// Alike, where many rows share a prefix: there every wave of the other workgroups has a unit
// of its own, with no barrier.
template <int TYPE, int D, int RTO>
__global__ __launch_bounds__(64 * SH_WAVES) __attribute__((amdgpu_waves_per_eu(2, 2))) void
k_prefix_wide(const SharedArgs P, const OwnArgs A, uint32_t shared) {
  typedef ShLds<D> S;
  typedef TrLds<D, RTO, 1> O;
  __shared__ __align__(16)
      char buf[sizeof(S) > SH_WAVES * sizeof(O) ? sizeof(S) : SH_WAVES * sizeof(O)];
  if (blockIdx.x < shared) {
    sh_attend<TYPE, D>(P, blockIdx.x, *reinterpret_cast<S*>(buf));
  } else {
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    tr_narrow<TYPE, D, RTO, 1>(A, (blockIdx.x - shared) * SH_WAVES + w, threadIdx.x & 63,
                               reinterpret_cast<O*>(buf)[w]);
  }
}

template <int TYPE, int D>
int run_part(pz_sampler* s, OwnArgs A, SharedArgs P) {
  const int rows = A.T * A.group;
  const int64_t most = (int64_t)A.B * rows;  // rows of a key head
  // (two slots are there: the host takes sequences accordingly)
  const int64_t slots =
      (int64_t)(PZ_TREE_WS / ((size_t)(D + 2) * sizeof(float))) / (int64_t)A.R;

  // the prefixes': the rows of a key head of all who share one
  const int64_t tiles = ((int64_t)P.pages.max_blocks << P.pages.shift) / TR_KEYS + 1;
  const int64_t heads = (int64_t)A.B * A.n_kv;
  const int64_t k = P.B < A.B ? P.B : A.B;  // prefixes with a row, at most
  const PfKernel kernel = pf_kernel_for((most + k - 1) / k, k * P.n_kv, tiles, heads, s->n_cu, D,
                                        P.ld, P.pages.shift);
  const bool wide = kernel == PF_WIDE;
  static_assert(SH_ROWS * SH_WAVES == PF_ROWS, "");
  const int block = wide ? PF_ROWS : kernel == PF_SOME ? 32 : 16;
  // (k of them: at most (most - k) / block + k row blocks)
  const int64_t blocks = P.first ? (most - k) / block + k
                                 : P.B * ((std::min<int64_t>(P.each, P.nb) * rows + block - 1) / block);

  // each sequence's own keys: 16 or 32 rows of a key head at a time
  const int64_t own = ((int64_t)A.pages.max_blocks << A.pages.shift) / TR_KEYS + 1 +
                      (A.T + TR_KEYS - 1) / TR_KEYS;
  const int own_rows = rows <= 16 ? 16 : 32;
  A.nblk = (rows + own_rows - 1) / own_rows;
  const int64_t units = heads * A.nblk;
  const int64_t own_wgs = wide ? (units + SH_WAVES - 1) / SH_WAVES : units;
  share_out(A, own, splits(s, own_wgs, own, slots - 1));
  const int64_t wgs = blocks * P.n_kv;
  int S;
  if (wide) {
    // (32 own keys take a CU 0.25 us; of the table's length half is there as a rule)
    S = pf_wide_splits(s->n_cu, wgs, tiles, units * own / 8,
                       std::min<int64_t>({64, slots - A.S, tiles / TR_SHARE}));
  } else {
    S = splits(s, wgs, tiles, slots - A.S);
  }
  share_out(P, tiles, S);
  P.run = (int)((blocks + k - 1) / k);
  const int64_t runs = (blocks + P.run - 1) / P.run;
  const int64_t shared = (runs * P.n_kv * P.S + 7) / 8 * 8 * P.run;
  int64_t others = (heads * A.S + 7) / 8 * 8 * A.nblk;
  if (wide) others = (others + SH_WAVES - 1) / SH_WAVES;
  if (!pz_launch_fits(shared + others, 512))
    return fail(s, PZ_ERANGE, "B=%d sequences of T=%d nodes", A.B, A.T);
  P.nblk = (int)blocks;
  P.slot = 0;
  A.slot = P.S;
  P.part = A.part = static_cast<float*>(s->tree_dev);
  P.ml = A.ml = A.part + (size_t)(P.S + A.S) * A.R * D;

  const dim3 grid((unsigned)(shared + others));
  const uint32_t first = (uint32_t)shared;
  const hipStream_t st = s->stream;
  if constexpr (D < 256) {
    if (wide && own_rows == 16)
      hipLaunchKernelGGL((k_prefix_wide<TYPE, D, 1>), grid, dim3(64 * SH_WAVES), 0, st, P, A, first);
    else if (wide)
      hipLaunchKernelGGL((k_prefix_wide<TYPE, D, 2>), grid, dim3(64 * SH_WAVES), 0, st, P, A, first);
  }
  if (kernel == PF_SOME && own_rows == 16)
    hipLaunchKernelGGL((k_prefix<TYPE, D, 2, 1>), grid, dim3(256), 0, st, P, A, first);
  else if (kernel == PF_SOME)
    hipLaunchKernelGGL((k_prefix<TYPE, D, 2, 2>), grid, dim3(256), 0, st, P, A, first);
  else if (kernel == PF_FEW)  // (a sequence's rows are its prefix's, too: 16 at most)
    hipLaunchKernelGGL((k_prefix<TYPE, D, 1, 1>), grid, dim3(256), 0, st, P, A, first);
  PZ_HIP(s, hipGetLastError());
  hipLaunchKernelGGL((k_prefix_join<TYPE, D>), dim3((unsigned)((A.R + 3) / 4)), dim3(256), 0, st,
                     A, P);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}

template <int TYPE>
int run_type(pz_sampler* s, const OwnArgs& A, const SharedArgs& P, int D) {
  if (D == 64) return run_part<TYPE, 64>(s, A, P);
  if (D == 128) return run_part<TYPE, 128>(s, A, P);
  return run_part<TYPE, 256>(s, A, P);
}

}  // namespace

extern "C" int pz_prefix_attention(pz_sampler* s, const pz_kv_cache* cache,
                                   const pz_kv_prefix* prefix, const void* d_kn, const void* d_vn,
                                   long ld_n, int B, int T, const int32_t* d_n_nodes,
                                   const uint64_t* d_tree, int n_heads, float scale,
                                   const void* d_q, long ld_q, void* d_out, long ld_out) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no = pz_refuse_prefix(cache, prefix, d_kn, d_vn, ld_n, B, T, n_heads, scale,
                                        d_q, ld_q, d_out, ld_out);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (B == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  const int rc = pz_tree_workspace(s);
  if (rc != PZ_OK) return rc;
  const int D = cache->head_dim;
  const int shift = __builtin_ctz((unsigned)cache->block_size);
  const size_t per = (size_t)T * n_heads;  // results of a sequence in a slot
  // as many sequences at a time as two slots hold
  int64_t step = (int64_t)(PZ_TREE_WS / (2 * (size_t)(D + 2) * sizeof(float)) / per);
  step = step < B ? step : B;
  for (int b0 = 0; b0 < B; b0 += (int)step) {
    const int nb = B - b0 < step ? B - b0 : (int)step;
    const size_t node0 = (size_t)b0 * T;
    OwnArgs A = {};
    A.k = static_cast<const uint16_t*>(cache->d_k);
    A.v = static_cast<const uint16_t*>(cache->d_v);
    A.ld = cache->ld;
    A.T = T;
    A.n_kv = cache->n_kv_heads;
    A.group = n_heads / cache->n_kv_heads;
    A.c = scale * TR_LOG2E;
    A.q = static_cast<const uint16_t*>(d_q) + node0 * ld_q;
    A.ld_q = ld_q;
    A.out = static_cast<uint16_t*>(d_out) + node0 * ld_out;
    A.ld_out = ld_out;
    A.R = (size_t)nb * per;
    SharedArgs P = {};
    static_cast<PartArgs&>(P) = A;
    P.first = prefix->d_first;
    P.each = B / prefix->n_prefixes;
    // (without ranges only the prefixes that these sequences have)
    const int p0 = P.first ? 0 : b0 / P.each;
    P.B = P.first ? prefix->n_prefixes : (b0 + nb - 1) / P.each + 1 - p0;
    P.pages = {cache->n_blocks, shift, prefix->max_blocks};
    P.blocks = prefix->d_blocks + (size_t)p0 * prefix->max_blocks;
    P.len = prefix->d_len + p0;
    P.b0 = b0 - p0 * P.each;
    P.nb = nb;
    A.B = nb;
    A.pages = {cache->n_blocks, shift, cache->max_blocks};
    A.blocks = cache->d_blocks + (size_t)b0 * cache->max_blocks;
    A.len = cache->d_len + b0;
    A.kn = static_cast<const uint16_t*>(d_kn) + node0 * ld_n;
    A.vn = static_cast<const uint16_t*>(d_vn) + node0 * ld_n;
    A.ld_n = ld_n;
    A.n_nodes = d_n_nodes ? d_n_nodes + b0 : nullptr;
    A.tree = d_tree ? d_tree + node0 : nullptr;
    const int rc = cache->type == PZ_BF16 ? run_type<PZ_BF16>(s, A, P, D)
                                          : run_type<PZ_F16>(s, A, P, D);
    if (rc != PZ_OK) return rc;
  }
  return PZ_OK;
}
