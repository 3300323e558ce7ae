// pz_beam.hip -- beam search: the best continuations of each group of beams
// (pz_beam_select) and the reordering of the chosen beams' caches (pz_beam_reorder).
//
// Selection.  score[w, i] = d_scores[w] + (x[w, i] - lse_w), lse_w = log sum_j exp(x[w, j]).
// Beams of a group lie close together, so that lse decides between their candidates: it is
// held in 64 bits.  Exponentials are off by at most 2^-43 (pz_beamexp.h), the factors that
// join a row's segments alike, lse by 2^-42 and a few 2^-53 of its value.  (A 64-bit fma takes
// a wave as long as a 32-bit one here.)  Within a beam the score rises with the logit, so that
// a row's K best are the K largest logits:
//
//   * k_beam_row: a workgroup a segment of a row, which it reads once, to registers:
//     maximum, sum of exponentials, and its K best as keys (order key of the logit, then
//     the id counted down: larger is better).  The threads' maxima meet in groups, the K-th
//     largest of which is a bound that K elements reach; the few at or above it meet in
//     LDS, where each counts those that are better.
//   * k_beam_join: a workgroup a group; the same over its beams' candidates.
//
// Where many more than K reach the bound (masks of low logits that are finite, of which all tie;
// beams whose scores lie far apart) the join takes a better one from those that have met, and
// either kernel takes the K best one by one where that is less work (be_counted).  1 x 4 beams
// of 128256 ids, 8 best: 11 us, 16 where a thousandth of the ids is above the mask; 16 beams, 128
// best: 46, and 85 where their scores are 6 apart (365 and 9700 before).
//
// Bound by the read of the logits with the vector instructions (13 an id) close behind: 256
// rows of 151936 ids (10% ended, 140 MB) 35-39 us, 4.0-3.6 TB/s, and 6 to join; 47 us with a
// series of 12 terms in place of the table.  Few rows take segments of 2048 ids, so that they
// fill the CUs (8 rows of 128256 ids: 12 us); of 8192 otherwise (64 rows 26 us, 38 in 2048).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/pz_sampler.h"
#include "pz_beamexp.h"
#include "pz_device.h"
#include "pz_pages.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"

namespace {

constexpr int BE_CAP = 2048;   // elements of a segment that meet in LDS
constexpr int BE_JCAP = 1024;  // candidates of a group that do
constexpr int BE_LONG = 256 * 32, BE_SHORT = 256 * 8;  // ids of a segment
constexpr int BE_LISTS = PZ_BEAM_MAX_WIDTH * (PZ_MOST_IDS / BE_LONG + 1);  // of a group, and one a beam

struct BeamStat {
  double sum;  // of exp(x - m); not finite where a logit is NaN or +infinity
  float m;     // the segment's maximum, -infinity without a finite logit
};

struct BeamArgs {
  const float* x;
  long ld;
  int W, V, S, K;  // beams, ids, segments of a row
  float per_list, per_segment;  // 1 / (W S), 1 / S
  int row_most, join_most;      // that are counted against each other (be_counted)
  const float* score;
  const uint8_t* done;
  int32_t pad;
  uint64_t* cand;   // [row][S][K]
  BeamStat* stat;   // [row][S]
  int32_t* parent;
  int32_t* ids;
  float* score_out;
  uint8_t* done_out;
  const int32_t* eos;
  int n_eos;
};

// (The logits' exponentials: pz_beamexp.h.)
constexpr float BE_PLAIN = 500.0f;  // largest |m| whose exponentials are taken as they are
constexpr float BE_LEAST = -650.0f;  // smaller logits count as this beside such an m (10^-65 of it)
typedef __attribute__((address_space(3))) const be_u32x2* be_table;
__device__ __forceinline__ be_u32x2 be_bits(uint64_t v) { return __builtin_bit_cast(be_u32x2, v); }

__device__ __forceinline__ double be_wave_sum(double v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

__device__ __forceinline__ uint64_t be_key(float x, int id) {
  return (uint64_t)pz_key(x) << 32 | (0xffffffffu - (uint32_t)id);
}
constexpr uint32_t BE_NONE = 0x007fffffu;  // the order key of -infinity

// max(v, v of the lane that DPP control CTRL names), CTRL one that gives every lane one.
template <int CTRL>
__device__ __forceinline__ float be_max_dpp(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf,
                                                             true)));
}
template <int CTRL>
__device__ __forceinline__ double be_max_dpp(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t l = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true),
                 h = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xf, 0xf, true);
  return fmax(v, __builtin_bit_cast(double, (uint64_t)h << 32 | l));
}

// A bound that at least K of the block's elements reach, -infinity where there are fewer:
// the K-th largest of the maxima of groups of threads (64, 16, 4 or 2 each, while there are
// 2 K of these at least, else 1; at least K).  mine: the thread's largest (-infinity
// without one); *most: the block's.  lds: BLOCK + 1 numbers.  One barrier, two with more
// than 64 groups, of which each wave then looks at 64 (all of them in every wave: one beam
// of 128256 ids, the 128 best: 92 us, 45 so).
template <int BLOCK, class F>
__device__ __forceinline__ F be_bound(F mine, int K, F* lds, F* most) {
  const int tid = threadIdx.x, lane = tid & 63;
  int shift = 0;  // of a group's threads
  if (BLOCK / 2 >= 2 * K) {
    mine = be_max_dpp<0xb1>(mine);  // the neighbour
    shift = 1;
    if (BLOCK / 4 >= 2 * K) {
      mine = be_max_dpp<0x4e>(mine);  // the other pair of a quad
      shift = 2;
    }
    if (BLOCK / 16 >= 2 * K) {
      mine = be_max_dpp<0x141>(mine);  // the eight mirrored, then the row's sixteen
      mine = be_max_dpp<0x140>(mine);
      shift = 4;
    }
    if (BLOCK / 64 >= 2 * K) {
      F v = __shfl_xor(mine, 16, 64);
      mine = v > mine ? v : mine;
      v = __shfl_xor(mine, 32, 64);
      mine = v > mine ? v : mine;
      shift = 6;
    }
  }
  const int groups = BLOCK >> shift;
  if ((tid & ((1 << shift) - 1)) == 0) lds[tid >> shift] = mine;
  if (tid == 0) lds[BLOCK] = -__builtin_inff();
  pz_lds_barrier();
  const int at = (groups > 64 ? tid & ~63 : 0) + lane;
  const bool on = at < groups;
  const F v = lds[on ? at : 0];
  F top = -__builtin_inff(), bound = -__builtin_inff();
  int more = 0, least = 0;  // groups above it, groups that it does not pass
  // (a multiple of four, aligned; no short cuts, which would be branches and a wait for each)
  typedef F four __attribute__((ext_vector_type(4)));
#pragma unroll 4
  for (int j = 0; j < groups; j += 4) {
    const four o = *reinterpret_cast<const four*>(lds + j);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      more += o[e] > v;
      least += o[e] >= v;
      top = o[e] > top ? o[e] : top;
    }
  }
  const bool is = on & (more < K) & (least >= K);  // (equal ones together)
  const uint64_t kth = __ballot(is);
  if (groups > 64) {
    if (is) lds[BLOCK] = v;
    pz_lds_barrier();
    bound = lds[BLOCK];
  } else if (kth) {
    bound = __shfl(v, __ffsll((unsigned long long)kth) - 1, 64);
  }
  *most = top;
  return bound;
}

template <int BLOCK, int NV>
__global__ __launch_bounds__(BLOCK) __attribute__((amdgpu_waves_per_eu(6, 8))) void k_beam_row(const BeamArgs A) {
  constexpr int WAVES = BLOCK / 64, N = 4 * NV;
  __shared__ uint64_t list[BE_CAP + 8];
  __shared__ double part[WAVES];
  __shared__ be_u32x2 roots[32];
  __shared__ __align__(16) float tops[BLOCK + 1];
  __shared__ int n_list;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int row = blockIdx.x / A.S, seg = blockIdx.x - row * A.S;
  // (what offers nothing is not read; the join sees the same)
  if (A.done && A.done[row]) return;
  if (!(fabsf(A.score[row]) < __builtin_inff())) return;
  const float* x = A.x + (size_t)row * A.ld;
  const int base = seg * (BLOCK * N);
  float v[N];
  if (base + BLOCK * N <= A.V) {
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const pz_f4u q = *reinterpret_cast<const pz_f4u*>(x + base + (j * BLOCK + tid) * 4);
#pragma unroll
      for (int e = 0; e < 4; e++) v[4 * j + e] = q[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int i = base + (j * BLOCK + tid) * 4 + e;
        v[4 * j + e] = i < A.V ? x[i] : -__builtin_inff();
      }
  }
  if (tid < 32) roots[tid] = be_bits(be_roots[tid]);
  if (tid == 0) n_list = 0;
  pz_lds_barrier();
  auto id_of = [&](int e) { return base + ((e >> 2) * BLOCK + tid) * 4 + (e & 3); };
  // (the exponentials as they are, which need no maximum: they are made while the later
  // loads are on their way)
  float mine = -__builtin_inff();
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < NV; j++) {
    // (four at a time: the compiler's mixture of all of them takes three times the registers)
    asm volatile("" : "+v"(v[4 * j]), "+v"(v[4 * j + 1]), "+v"(v[4 * j + 2]), "+v"(v[4 * j + 3]),
                 "+v"(sum));
#pragma unroll
    for (int e = 4 * j; e < 4 * j + 4; e++) {
      mine = fmaxf(mine, v[e]);  // (past a NaN, which the other maximum keeps)
      sum = be_add_exp(sum, (double)__builtin_elementwise_maximum(v[e], BE_LEAST), (be_table)roots);
    }
  }
  // (a NaN is in the sum of a row that has a finite maximum; without one it counts as infinite)
  if (mine == -__builtin_inff() && sum != sum) mine = __builtin_inff();
  float m;
  const float T = be_bound<BLOCK>(mine, A.K, tops, &m);
  uint64_t* out = A.cand + (size_t)blockIdx.x * A.K;
  if (!(fabsf(m) < __builtin_inff())) {  // no finite logit, or an infinite one
    for (int i = tid; i < A.K; i += BLOCK) out[i] = 0u;
    if (tid == 0) A.stat[blockIdx.x] = {m > 0.0f ? (double)m : 0.0, m};
    return;
  }
  const float least = fmaxf(T, -3.40282346638528859812e38f);  // (-infinity is never chosen)
#pragma unroll
  for (int e = 0; e < N; e++)
    if (__ballot(v[e] >= least))
      if (v[e] >= least) {
        const int i = atomicAdd(&n_list, 1);
        if (i < BE_CAP) list[i] = be_key(v[e], id_of(e));
      }
  const bool plain = fabsf(m) <= BE_PLAIN;
  if (!plain) {
    sum = 0.0;
#pragma unroll
    for (int e = 0; e < N; e++) {
      asm volatile("" : "+v"(v[e]), "+v"(sum));
      sum += be_exp(v[e], m, (be_table)roots);
    }
  }
  sum = be_wave_sum(sum);
  if (lane == 0) part[w] = sum;
  pz_lds_barrier();
  const int n = n_list;
  if (tid == 0) {
    double s = part[0];
#pragma unroll
    for (int i = 1; i < WAVES; i++) s += part[i];
    if (plain) s *= exp(-(double)m);
    A.stat[blockIdx.x] = {s, m};
  }
  for (int i = n + tid; i < A.K; i += BLOCK) out[i] = 0u;
  if (n <= A.row_most) {
    for (int i = tid; i < n; i += BLOCK) {
      const uint64_t k = list[i];
      int better = 0;
      for (int j = 0; j < n; j += 8)  // (eight on their way at a time)
#pragma unroll
        for (int c = 0; c < 8; c++) better += (list[j + c] > k) & (j + c < n);
      if (better < A.K) out[better] = k;
    }
    return;
  }
  // one by one
  uint64_t last = ~0ull;
  for (int k = 0; k < A.K; k++) {
    uint64_t best = 0u;
#pragma unroll
    for (int e = 0; e < N; e++) {
      const uint64_t c = pz_key(v[e]) > BE_NONE ? be_key(v[e], id_of(e)) : 0u;
      best = c < last && c > best ? c : best;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
      const uint64_t c = __shfl_xor(best, o, 64);
      best = c > best ? c : best;
    }
    pz_lds_barrier();
    if (lane == 0) list[w] = best;
    pz_lds_barrier();
    best = list[0];
#pragma unroll
    for (int i = 1; i < WAVES; i++) best = list[i] > best ? list[i] : best;
    if (tid == 0) out[k] = best;
    last = best;
  }
}

// A candidate of a group: larger scores first, then lower beams, then larger keys.
struct BeamCand {
  double score;
  uint64_t key;
  int beam;
};
__device__ __forceinline__ bool be_better(const BeamCand& a, const BeamCand& b) {
  // (no short cuts: they would be branches, and a wait for each member)
  return (a.score > b.score) |
         ((a.score == b.score) & ((a.beam < b.beam) | ((a.beam == b.beam) & (a.key > b.key))));
}

constexpr int BE_JOIN = 1024;  // threads
constexpr int BE_HELD = 4;     // candidates that a thread keeps
constexpr int BE_JLDS = std::max<int>(BE_JCAP * sizeof(BeamCand) + (BE_JOIN + 1) * sizeof(double),
                                      BE_JOIN / 64 * sizeof(BeamCand) + BE_LISTS);
static_assert(BE_JCAP * sizeof(BeamCand) % 32 == 0, "four of tops together");

// e / d for e, d < 2^24 and per = 1 / d as a float.
__device__ __forceinline__ int be_div(int e, int d, float per) {
  int q = (int)((float)e * per);
  q -= q * d > e;
  return q + (e - q * d >= d);
}

__global__ __launch_bounds__(BE_JOIN) void k_beam_join(const BeamArgs A) {
  constexpr int WAVES = BE_JOIN / 64;
  // list and tops; or, where candidates are taken one by one, how many of each list are
  __shared__ __align__(32) char mem[BE_JLDS];
  BeamCand* const list = reinterpret_cast<BeamCand*>(mem);
  double* const tops = reinterpret_cast<double*>(mem + BE_JCAP * sizeof(BeamCand));
  uint8_t* const taken = reinterpret_cast<uint8_t*>(mem + WAVES * sizeof(BeamCand));
  __shared__ be_u32x2 roots[32];
  __shared__ double lse[PZ_BEAM_MAX_WIDTH], sum[PZ_BEAM_MAX_WIDTH];
  __shared__ int state[PZ_BEAM_MAX_WIDTH];  // 0: offers nothing, 1: its row, 2: itself
  __shared__ int n_list;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row0 = (int64_t)blockIdx.x * A.W;
  const int lists = A.W * A.S, total = lists * A.K;
  const uint64_t* cand = A.cand + row0 * A.S * A.K;
  // Candidate e: one of every beam that has ended, then the lists' first ones, their second
  // ones, ...  A thread keeps BE_HELD of them.  Each wave's are of all lists alike, however
  // many lists there are, so that be_bound's groups are of equal chances (8 groups of 8
  // beams, 16 of 16 segments: 100 us with a wave's candidates in a row).
  auto nth = [&](int i) { return i * BE_JOIN + lane * WAVES + ((w + lane + i) & (WAVES - 1)); };
  auto load = [&](int e, int* beam) {
    const int f = e < A.W ? 0 : e - A.W, rank = be_div(f, lists, A.per_list), l = f - rank * lists;
    *beam = e < A.W ? e : be_div(l, A.S, A.per_segment);
    return e >= A.W && f < total ? cand[l * A.K + rank] : 0u;
  };
  // (on their way beside the beams' sums; what beams that offer nothing left is not used)
  uint64_t key[BE_HELD];
  int beam[BE_HELD];
#pragma unroll
  for (int i = 0; i < BE_HELD; i++) {
    key[i] = 0u;
    beam[i] = 0;
    if (i * BE_JOIN < total + A.W) key[i] = load(nth(i), &beam[i]);
  }
  if (tid < 32) roots[tid] = be_bits(be_roots[tid]);
  if (tid == 0) n_list = 0;
  pz_lds_barrier();
  for (int b = w; b < A.W; b += WAVES) {
    const int64_t row = row0 + b;
    const BeamStat* s = A.stat + row * A.S;
    BeamStat one = {0.0, -__builtin_inff()};
    if (lane < A.S) one = s[lane];  // (with the next two, whether it counts or not)
    const float sc = A.score[row];
    const bool ended = A.done && A.done[row];
    int st = !(fabsf(sc) < __builtin_inff()) ? 0 : ended ? 2 : 1;
    double l = 0.0;
    if (st == 1) {
      float m = one.m;
      bool bad = !(one.sum < __builtin_inf());
      for (int i = 64 + lane; i < A.S; i += 64) {
        bad |= !(s[i].sum < __builtin_inf());
        m = fmaxf(m, s[i].m);
      }
      m = pz_wave_max(m);
      if (__ballot(bad) || m == -__builtin_inff()) {
        st = 0;
      } else {
        if (one.m > -__builtin_inff()) l = one.sum * be_exp(one.m, m, (be_table)roots);
        for (int i = 64 + lane; i < A.S; i += 64)
          if (s[i].m > -__builtin_inff()) l += s[i].sum * be_exp(s[i].m, m, (be_table)roots);
        l = (double)m + log(be_wave_sum(l));
      }
    }
    if (lane == 0) {
      state[b] = st;
      sum[b] = (double)sc;
      lse[b] = l;
    }
  }
  pz_lds_barrier();
  // the score of what a list of beam b holds (no key: none)
  auto score_of = [&](int b, uint64_t k) {
    return state[b] == 1 && k ? sum[b] + ((double)pz_unkey((uint32_t)(k >> 32)) - lse[b])
                              : -__builtin_inf();
  };
  auto take = [&](int e, uint64_t k, int b) -> BeamCand {
    if (e >= A.W) return {score_of(b, k), k, b};
    return {state[b] == 2 ? sum[b] : -__builtin_inf(), 0xffffffffu - (uint32_t)A.pad, b};
  };
  BeamCand held[BE_HELD];
  double mine = -__builtin_inf(), top;
#pragma unroll
  for (int i = 0; i < BE_HELD; i++) {
    held[i].score = -__builtin_inf();
    if (i * BE_JOIN < total + A.W) {
      held[i] = take(nth(i), key[i], beam[i]);
      mine = held[i].score > mine ? held[i].score : mine;
    }
  }
  // (a bound that K of those kept reach is one for all)
  double T = be_bound<BE_JOIN>(mine, A.K, tops, &top);
  auto meet = [&](const BeamCand& c) {
    if (c.score >= T && c.score > -__builtin_inf()) {
      const int at = atomicAdd(&n_list, 1);
      if (at < BE_JCAP) list[at] = c;
    }
  };
  // those of list l from `rank` on, while they reach the bound (the 32 best of 16 beams of
  // 151936 ids 70 us with all of them looked at, 40 so)
  auto open = [&](int l, int rank) {
    const int b = be_div(l, A.S, A.per_segment);
    for (; rank < A.K; rank++) {
      const uint64_t k = cand[l * A.K + rank];
      const BeamCand c = {score_of(b, k), k, b};
      if (!(c.score >= T)) break;
      meet(c);
    }
  };
  if (mine >= T)
#pragma unroll
    for (int i = 0; i < BE_HELD; i++)
      if (i * BE_JOIN < total + A.W) meet(held[i]);
  if (total + A.W > BE_HELD * BE_JOIN)  // the lists' others
    for (int l = tid; l < lists; l += BE_JOIN) {
      const int kept = BE_HELD * BE_JOIN - A.W;
      open(l, l < kept ? (kept - l - 1) / lists + 1 : 0);
    }
  pz_lds_barrier();
  int n = n_list;
  // More than there is room for (where some beams' scores are far above the others', the bound
  // is that of all lists' first ones): the K-th of those that have met is a better one, but
  // where they tie.
  static_assert(BE_JCAP == BE_JOIN, "one of them a thread");
  while (n > BE_JCAP) {
    const double better = be_bound<BE_JOIN>(list[tid].score, A.K, tops, &top);
    if (!(better > T)) break;
    T = better;
    if (tid == 0) n_list = 0;
    pz_lds_barrier();
    if (tid < A.W) meet(take(tid, 0u, tid));
    for (int l = tid; l < lists; l += BE_JOIN) open(l, 0);
    pz_lds_barrier();
    n = n_list;
  }
  const size_t o = (size_t)blockIdx.x * A.K;
  auto put = [&](int k, const BeamCand& c) {
    const int32_t id = (int32_t)(0xffffffffu - (uint32_t)c.key);
    A.parent[o + k] = c.beam;
    A.ids[o + k] = id;
    A.score_out[o + k] = (float)c.score;
    if (A.done_out) {
      uint8_t f = state[c.beam] == 2;
      for (int i = 0; i < A.n_eos; i++) f |= (uint8_t)(A.eos[i] == id);
      A.done_out[o + k] = f;
    }
  };
  for (int k = n + tid; k < A.K; k += BE_JOIN) {
    A.parent[o + k] = -1;
    A.ids[o + k] = -1;
    A.score_out[o + k] = -__builtin_inff();
    if (A.done_out) A.done_out[o + k] = 0;
  }
  if (n <= A.join_most) {
    // sixteen threads a candidate
    for (int i = tid >> 4; i < n; i += BE_JOIN / 16) {
      const BeamCand c = list[i];
      int better = 0;
      for (int j = tid & 15; j < n; j += 16) better += be_better(list[j], c);
#pragma unroll
      for (int s = 1; s < 16; s <<= 1) better += __shfl_xor(better, s, 64);
      if ((tid & 15) == 0 && better < A.K) put(better, c);
    }
    return;
  }
  // one by one: the best of the threads' best.  A thread has every BE_JOIN-th list (and those of
  // one candidate, the ended beams'), each of which is in order; who gave the best takes its
  // list's next.
  const int all = lists + A.W;
  pz_lds_barrier();
  for (int l = tid; l < all; l += BE_JOIN) taken[l] = 0;  // (a thread's own)
  BeamCand own;
  int from = 0;  // whose the best is
  auto look = [&]() {
    own = {-__builtin_inf(), 0u, 1 << 30};
    for (int l = tid; l < all; l += BE_JOIN) {
      const int rank = taken[l];
      if (rank == (l < lists ? A.K : 1)) continue;
      const BeamCand c = l < lists ? take(A.W, cand[l * A.K + rank], be_div(l, A.S, A.per_segment))
                                   : take(l - lists, 0u, l - lists);
      if (c.score > -__builtin_inf() && be_better(c, own)) own = c, from = l;
    }
  };
  look();
  for (int k = 0; k < A.K; k++) {
    BeamCand best = own;
#pragma unroll
    for (int s = 32; s; s >>= 1) {
      const BeamCand c = {__shfl_xor(best.score, s, 64), __shfl_xor(best.key, s, 64),
                          __shfl_xor(best.beam, s, 64)};
      if (be_better(c, best)) best = c;
    }
    __syncthreads();
    if (lane == 0) list[w] = best;
    __syncthreads();
    best = list[0];
    for (int i = 1; i < WAVES; i++)
      if (be_better(list[i], best)) best = list[i];
    if (tid == 0) put(k, best);
    if (best.beam == own.beam && best.key == own.key) {
      taken[from]++;
      look();
    }
  }
}

// Up to how many are counted against each other, each by those that are better, rather than
// taken one by one: n of a segment take ceil(n / 256) n 22 ns, one by one 0.5 us each of the K
// (2048 that tie, 8 best: 355 us and 4); of a group n^2 0.1 ns and 3 us each (1008, 16 best:
// 105 and 43).
struct BeamCounted {
  int row, join;
};
BeamCounted be_counted(int K) {
  const int few = std::min(23 * K, 256), many = (int)std::sqrt(256.0 * 23.0 * K);
  return {std::min(std::max(few, many), BE_CAP),
          std::min((int)std::sqrt(30720.0 * K), BE_JCAP)};
}

int be_workspace(pz_sampler* s) {
  if (!s->beam_dev && hipMalloc(&s->beam_dev, PZ_BEAM_WORKSPACE) != hipSuccess) {
    s->beam_dev = nullptr;
    (void)hipGetLastError();
    return fail(s, PZ_ENOMEM, "the beam search's workspace");
  }
  return PZ_OK;
}

// ---- reordering --------------------------------------------------------------
// Pages shared, kept, given out and free again without counts that live from call to
// call: which pages are in use is what the new tables name.
//   * k_beam_plan: a workgroup a group.  The parents' full pages and the page that the
//     first child keeps go to the new tables and are marked among the pool's (ascending:
//     a binary search; a bit each in LDS); then the unmarked ones are numbered and given
//     out in that order.
//   * k_beam_copy: the positions of the pages that other children share with the first.
//     A page that is copied from stays with a first child, so none is also written.
//   * k_beam_move, where tables and pool fit LDS: both in one launch.  A workgroup for the
//     tables of each group, and one for each beam and buffer, which finds out by itself what
//     it copies (8 x 8 beams, 8 layers: 12.7 us in two launches, 7.5 so).
struct ReorderArgs {
  const int32_t* blocks;
  const int32_t* len;
  PzPages pages;
  int W;
  const int32_t* parent;
  const int32_t* pool;
  int n_pool, ahead;
  int32_t* blocks_out;
  int32_t* len_out;
  int32_t* missing;
  int4* copy;  // [beam] page from, page to (-1: none), positions
};

constexpr int BE_PLAN = 512;  // threads

// Where `page` is in the pool, -1 if it is not.  Its n pages ascend, each once, so that their
// distance from the ends is at least what their numbers differ by: a pool of neighbours needs
// no search (64 beams, tables of 1024 pages: 419 us with one, 104 so; 8 of 2048 97, 37).
__device__ __forceinline__ int be_find(const int32_t* pool, int n, int32_t page) {
  if (n == 0) return -1;
  const int64_t below = (int64_t)page - pool[0], above = (int64_t)pool[n - 1] - page;
  if (below < 0 || above < 0) return -1;
  int lo = above < n ? n - 1 - (int)above : 0, hi = below < n ? (int)below : n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (pool[mid] < page)
      lo = mid + 1;
    else
      hi = mid;
  }
  return pool[lo] == page ? lo : -1;
}

__global__ __launch_bounds__(BE_PLAN) void k_beam_plan(const ReorderArgs A) {
  extern __shared__ uint32_t used[];  // a bit a page of the pool
  __shared__ int par[PZ_BEAM_MAX_WIDTH], lens[PZ_BEAM_MAX_WIDTH];
  __shared__ int keep[PZ_BEAM_MAX_WIDTH], want[PZ_BEAM_MAX_WIDTH];  // columns kept, columns filled
  __shared__ int eldest[PZ_BEAM_MAX_WIDTH];
  __shared__ int from[PZ_BEAM_MAX_WIDTH + 1];  // new pages of the beams before
  __shared__ int scan[BE_PLAN / 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const size_t beam0 = (size_t)blockIdx.x * A.W;
  const int per = A.pages.max_blocks, shift = A.pages.shift, size = 1 << shift;
  const int words = (A.n_pool + 31) / 32;
  const int32_t* pool = A.pool + (size_t)blockIdx.x * A.n_pool;
  for (int i = tid; i < words; i += BE_PLAN) used[i] = 0u;
  if (tid < A.W) {
    const int p = A.parent[beam0 + tid];
    const bool ok = p >= 0 && p < A.W;
    par[tid] = ok ? p : -1;
    lens[tid] = ok ? pz_pages_len(A.pages, A.len[beam0 + p]) : 0;
  }
  __syncthreads();
  if (tid < A.W) {
    const int p = par[tid], L = lens[tid];
    bool first = true;
    for (int i = 0; i < tid; i++) first = first && par[i] != p;
    const int64_t to = (((int64_t)L + A.ahead + size - 1) >> shift);
    eldest[tid] = first;
    keep[tid] = (L >> shift) + (first && (L & (size - 1)));
    want[tid] = p < 0 ? 0 : (int)(to < per ? to : per);
    A.len_out[beam0 + tid] = L;
    A.copy[beam0 + tid] = int4{-1, -1, 0, 0};
  }
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    for (int b = 0; b < A.W; b++) {
      from[b] = n;
      n += want[b] - keep[b];
    }
    from[A.W] = n;
  }
  for (int i = tid; i < A.W * per; i += BE_PLAN) {
    const int b = i / per, col = i - b * per;
    if (col >= keep[b]) {
      if (col >= want[b]) A.blocks_out[beam0 * per + i] = -1;
      continue;
    }
    const int32_t page = A.blocks[(beam0 + par[b]) * per + col];
    A.blocks_out[beam0 * per + i] = page;
    if (!eldest[b]) continue;  // (its first sibling marks the same)
    const int at = be_find(pool, A.n_pool, page);
    if (at >= 0) atomicOr(&used[at >> 5], 1u << (at & 31));
  }
  __syncthreads();
  const int all = from[A.W];
  // new page `n` of the group
  auto give = [&](int n, int32_t page) {
    int lo = 0, hi = A.W - 1;  // the last beam that starts at n or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (from[mid] <= n)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int col = keep[lo] + n - from[lo];
    A.blocks_out[(beam0 + lo) * per + col] = page;
    const int rem = lens[lo] & (size - 1);
    if (rem && !eldest[lo] && col == lens[lo] >> shift && page >= 0)
      A.copy[beam0 + lo] = int4{A.blocks[(beam0 + par[lo]) * per + col], page, rem, 0};
  };
  int given = 0;
  for (int i0 = 0; i0 < words && given < all; i0 += BE_PLAN) {
    const int i = i0 + tid;
    uint32_t free = 0u;
    if (i < words) {
      free = ~used[i];
      if (i == words - 1 && (A.n_pool & 31)) free &= (1u << (A.n_pool & 31)) - 1u;
    }
    const int mine = __popc(free);
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      sum += lane >= o ? v : 0;
    }
    if (lane == 63) scan[w] = sum;
    __syncthreads();
    int at = given + sum - mine, n = 0;
    for (int k = 0; k < BE_PLAN / 64; k++) {
      if (k < w) at += scan[k];
      n += scan[k];
    }
    for (; free && at < all; at++) {
      const int bit = __ffs(free) - 1;
      free &= free - 1u;
      give(at, pool[i * 32 + bit]);
    }
    given += n;
    __syncthreads();
  }
  for (int n = given + tid; n < all; n += BE_PLAN) give(n, -1);
  if (tid == 0 && A.missing) A.missing[blockIdx.x] = all > given ? all - given : 0;
}

constexpr int BE_LAYERS = 64;  // of a launch
struct CopyArgs {
  uint16_t* buf[BE_LAYERS][2];  // keys, values
  long ld;
  int row;  // elements of a position
  PzPages pages;
  const int4* copy;
};

typedef uint32_t be_u32x4 __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(256) void k_beam_copy(const CopyArgs A) {
  const int4 c = A.copy[blockIdx.x];
  if (c.y < 0) return;
  int64_t src, dst;
  if (!pz_pages_slot(A.pages, c.x, 0, &src) || !pz_pages_slot(A.pages, c.y, 0, &dst)) return;
  uint16_t* buf = A.buf[blockIdx.y >> 1][blockIdx.y & 1];
  // (16-byte pieces)
  for (PzPieces i(A.row / 8, blockIdx.z * 256 + threadIdx.x, gridDim.z * 256); i.p < c.z; i.next()) {
    const size_t at = (size_t)i.p * A.ld + (size_t)i.j * 8;
    *reinterpret_cast<be_u32x4*>(buf + dst * A.ld + at) =
        *reinterpret_cast<const be_u32x4*>(buf + src * A.ld + at);
  }
}

constexpr int BE_MOVE = 256;          // threads
constexpr int BE_MOVE_TABLE = 4096;   // most entries of a group's tables
constexpr int BE_MOVE_POOL = 32 * BE_MOVE;  // most pages of its pool
constexpr int64_t BE_MOVES = 1 << 20;  // most workgroups (each of which looks at its group)

__global__ __launch_bounds__(BE_MOVE) void k_beam_move(const ReorderArgs R, const CopyArgs C,
                                                       int buffers, int parts) {
  extern __shared__ int32_t lds[];
  __shared__ int par[PZ_BEAM_MAX_WIDTH], len[PZ_BEAM_MAX_WIDTH], old_len[PZ_BEAM_MAX_WIDTH];
  __shared__ int keep[PZ_BEAM_MAX_WIDTH], want[PZ_BEAM_MAX_WIDTH], eldest[PZ_BEAM_MAX_WIDTH];
  __shared__ int from[PZ_BEAM_MAX_WIDTH + 1];
  __shared__ int scan[BE_MOVE / 64], target;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  // workgroup 0 of a group: its tables; then one a beam, buffer and part of its positions
  const int each = 1 + R.W * buffers * parts, group = blockIdx.x / each,
            job = blockIdx.x - group * each - 1;
  const bool tables = job < 0;
  const int mine = tables ? 0 : job / (buffers * parts);
  const size_t beam0 = (size_t)group * R.W;
  const int per = R.pages.max_blocks, shift = R.pages.shift, size = 1 << shift;
  const int words = (R.n_pool + 31) / 32;
  int32_t* const tab = lds;               // [W, per]
  int32_t* const pool = tab + R.W * per;  // [n_pool]
  uint32_t* const used = reinterpret_cast<uint32_t*>(pool + R.n_pool);  // [words]
  auto fetch = [&]() {
    for (int i = tid; i < R.W * per; i += BE_MOVE) tab[i] = R.blocks[beam0 * per + i];
    for (int i = tid; i < R.n_pool; i += BE_MOVE) pool[i] = R.pool[(size_t)group * R.n_pool + i];
    for (int i = tid; i < words; i += BE_MOVE) used[i] = 0u;
  };
  if (tables) fetch();
  if (tid < R.W) {
    const int p = R.parent[beam0 + tid];
    par[tid] = p >= 0 && p < R.W ? p : -1;
    old_len[tid] = pz_pages_len(R.pages, R.len[beam0 + tid]);
  }
  __syncthreads();
  if (w == 0) {
    int n = 0;
    if (lane < R.W) {
      const int p = par[lane], L = p < 0 ? 0 : old_len[p];
      bool first = true;
      for (int i = 0; i < lane; i++) first = first & (par[i] != p);
      const int64_t to = ((int64_t)L + R.ahead + size - 1) >> shift;
      len[lane] = L;
      eldest[lane] = first;
      keep[lane] = (L >> shift) + (first && (L & (size - 1)));
      want[lane] = p < 0 ? 0 : (int)(to < per ? to : per);
      n = want[lane] - keep[lane];
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      sum += lane >= o ? v : 0;
    }
    if (lane < R.W) from[lane] = sum - n;
    if (lane == 63) from[R.W] = sum;
    if (lane == 0) target = -1;
  }
  __syncthreads();
  const int rem = len[mine] & (size - 1);
  if (!tables) {
    if (!rem || eldest[mine]) return;  // (as most do, before they read more)
    fetch();
    __syncthreads();
  }
  for (int i = tid; i < R.W * per; i += BE_MOVE) {
    const int b = i / per, col = i - b * per;
    if (col >= keep[b]) {
      if (tables && col >= want[b]) R.blocks_out[beam0 * per + i] = -1;
      continue;
    }
    const int32_t page = tab[par[b] * per + col];
    if (tables) R.blocks_out[beam0 * per + i] = page;
    if (!eldest[b]) continue;  // (its first sibling marks the same)
    const int at = be_find(pool, R.n_pool, page);
    if (at >= 0) atomicOr(&used[at >> 5], 1u << (at & 31));
  }
  __syncthreads();
  // the free pages' numbers: a word a thread
  uint32_t free = 0u;
  if (tid < words) {
    free = ~used[tid];
    if (tid == words - 1 && (R.n_pool & 31)) free &= (1u << (R.n_pool & 31)) - 1u;
  }
  const int count = __popc(free);
  int sum = count;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(sum, o, 64);
    sum += lane >= o ? v : 0;
  }
  if (lane == 63) scan[w] = sum;
  __syncthreads();
  int at = sum - count, given = 0;
  for (int k = 0; k < BE_MOVE / 64; k++) {
    if (k < w) at += scan[k];
    given += scan[k];
  }
  if (tables) {
    const int all = from[R.W];
    auto give = [&](int n, int32_t page) {
      int lo = 0, hi = R.W - 1;  // the last beam that starts at n or before
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (from[mid] <= n)
          lo = mid;
        else
          hi = mid - 1;
      }
      R.blocks_out[(beam0 + lo) * per + keep[lo] + n - from[lo]] = page;
    };
    for (; free && at < all; at++) {
      const int bit = __ffs(free) - 1;
      free &= free - 1u;
      give(at, pool[tid * 32 + bit]);
    }
    for (int n = given + tid; n < all; n += BE_MOVE) give(n, -1);
    if (tid == 0 && R.missing) R.missing[group] = all > given ? all - given : 0;
    if (tid < R.W) R.len_out[beam0 + tid] = len[tid];
    return;
  }
  // the first new page of this beam, if there is one
  const int n = from[mine];
  if (at <= n && n < at + count) {
    for (int i = at; i < n; i++) free &= free - 1u;
    target = pool[tid * 32 + __ffs(free) - 1];
  }
  __syncthreads();
  int64_t src, dst;
  if (!pz_pages_slot(C.pages, tab[par[mine] * per + (len[mine] >> shift)], 0, &src) ||
      !pz_pages_slot(C.pages, target, 0, &dst))
    return;
  const int rest = job - mine * (buffers * parts), which = rest / parts, part = rest - which * parts;
  uint16_t* buf = C.buf[which >> 1][which & 1];
  // (16-byte pieces)
  for (PzPieces i(C.row / 8, part * BE_MOVE + tid, parts * BE_MOVE); i.p < rem; i.next()) {
    const size_t o = (size_t)i.p * C.ld + (size_t)i.j * 8;
    *reinterpret_cast<be_u32x4*>(buf + dst * C.ld + o) =
        *reinterpret_cast<const be_u32x4*>(buf + src * C.ld + o);
  }
}

}  // namespace

extern "C" int pz_beam_select(pz_sampler* s, const float* d_logits, long ld, int n_groups, int W,
                              int V, const float* d_scores, const uint8_t* d_done, int32_t pad_id,
                              int K, int32_t* d_parent, int32_t* d_ids, float* d_scores_out,
                              uint8_t* d_done_out) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no = pz_refuse_select(d_logits, ld, n_groups, W, V, d_scores, K, d_parent,
                                        d_ids, d_scores_out);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (n_groups == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  const int rc = be_workspace(s);
  if (rc != PZ_OK) return rc;
  const int64_t rows = (int64_t)n_groups * W;
  const bool few = rows * ((V + BE_LONG - 1) / BE_LONG) < 2 * (int64_t)s->n_cu;
  const int S = few ? (V + BE_SHORT - 1) / BE_SHORT : (V + BE_LONG - 1) / BE_LONG;
  const BeamCounted counted = be_counted(K);
  const size_t per = (size_t)W * S * (sizeof(BeamStat) + (size_t)K * sizeof(uint64_t));
  int64_t step = (int64_t)(PZ_BEAM_WORKSPACE / per);
  const int64_t most = UINT32_MAX / 512 / ((int64_t)W * S);  // groups that a launch takes
  step = step < most ? step : most;
  step = step < n_groups ? step : n_groups;
  for (int64_t g = 0; g < n_groups; g += step) {
    const int n = (int)(n_groups - g < step ? n_groups - g : step);
    BeamStat* stat = static_cast<BeamStat*>(s->beam_dev);
    const BeamArgs A = {d_logits + g * W * ld,
                        ld,
                        W,
                        V,
                        S,
                        K,
                        1.0f / (float)(W * S),
                        1.0f / (float)S,
                        counted.row,
                        counted.join,
                        d_scores + g * W,
                        d_done ? d_done + g * W : nullptr,
                        pad_id,
                        reinterpret_cast<uint64_t*>(stat + (size_t)n * W * S),
                        stat,
                        d_parent + g * K,
                        d_ids + g * K,
                        d_scores_out + g * K,
                        d_done_out ? d_done_out + g * K : nullptr,
                        s->d_eos,
                        s->n_eos};
    const dim3 grid((unsigned)(n * W * S));
    if (few)
      hipLaunchKernelGGL((k_beam_row<256, 2>), grid, dim3(256), 0, s->stream, A);
    else
      hipLaunchKernelGGL((k_beam_row<256, 8>), grid, dim3(256), 0, s->stream, A);
    PZ_HIP(s, hipGetLastError());
    hipLaunchKernelGGL(k_beam_join, dim3((unsigned)n), dim3(BE_JOIN), 0, s->stream, A);
    PZ_HIP(s, hipGetLastError());
  }
  return PZ_OK;
}

extern "C" int pz_beam_reorder(pz_sampler* s, const pz_kv_cache* layers, int n_layers,
                               int n_groups, int W, const int32_t* d_parent,
                               const int32_t* d_pool, int n_pool, int ahead,
                               int32_t* d_blocks_out, int32_t* d_len_out, int32_t* d_missing) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no = pz_refuse_reorder(layers, n_layers, n_groups, W, d_parent, d_pool, n_pool,
                                         ahead, d_blocks_out, d_len_out);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (n_groups == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  const int rc = be_workspace(s);
  if (rc != PZ_OK) return rc;
  const pz_kv_cache& c = layers[0];
  const PzPages pages = {c.n_blocks, __builtin_ctz((unsigned)c.block_size), c.max_blocks};
  int4* copy = static_cast<int4*>(s->beam_dev);
  const ReorderArgs R = {c.d_blocks,   c.d_len,   pages,     W,    d_parent, d_pool, n_pool, ahead,
                         d_blocks_out, d_len_out, d_missing, copy};
  // workgroups of a page: 16 positions each
  const int parts = c.block_size < 16 * 64 ? (c.block_size + 15) / 16 : 64;
  auto layers_of = [&](int l) {
    const int n = n_layers - l < BE_LAYERS ? n_layers - l : BE_LAYERS;
    CopyArgs A = {};
    for (int i = 0; i < n; i++) {
      A.buf[i][0] = static_cast<uint16_t*>(layers[l + i].d_k);
      A.buf[i][1] = static_cast<uint16_t*>(layers[l + i].d_v);
    }
    A.ld = c.ld;
    A.row = c.n_kv_heads * c.head_dim;
    A.pages = pages;
    A.copy = copy;
    return A;
  };
  const int64_t moves = n_groups * (1 + (int64_t)W * 2 * n_layers * parts);
  if (n_layers <= BE_LAYERS && (int64_t)W * c.max_blocks <= BE_MOVE_TABLE &&
      n_pool <= BE_MOVE_POOL && moves <= BE_MOVES) {
    const size_t lds = ((size_t)W * c.max_blocks + n_pool + (n_pool + 31) / 32) * 4;
    hipLaunchKernelGGL(k_beam_move, dim3((unsigned)moves), dim3(BE_MOVE), lds, s->stream, R,
                       layers_of(0), 2 * n_layers, parts);
    PZ_HIP(s, hipGetLastError());
    return PZ_OK;
  }
  hipLaunchKernelGGL(k_beam_plan, dim3((unsigned)n_groups), dim3(BE_PLAN),
                     ((size_t)n_pool + 31) / 32 * 4, s->stream, R);
  PZ_HIP(s, hipGetLastError());
  for (int l = 0; l < n_layers; l += BE_LAYERS) {
    const unsigned n = (unsigned)(n_layers - l < BE_LAYERS ? n_layers - l : BE_LAYERS);
    // (most beams copy nothing: workgroups for each part of a page only while they are few)
    const int64_t z = std::min<int64_t>(parts, BE_MOVES / ((int64_t)n_groups * W * 2 * n) + 1);
    hipLaunchKernelGGL(k_beam_copy, dim3((unsigned)(n_groups * W), 2u * n, (unsigned)z), dim3(256),
                       0, s->stream, layers_of(l));
    PZ_HIP(s, hipGetLastError());
  }
  return PZ_OK;
}
