// pz_beam.hip -- beam search: the best continuations of each group of beams
// (pz_beam_select) and the reordering of the chosen beams' caches (pz_beam_reorder).
//
// Selection.  score[w, i] = d_scores[w] + (x[w, i] - lse_w), lse_w = log sum_j exp(x[w, j]).
// Beams of a group lie close together, so that lse decides between their candidates: it is
// held in 64 bits.  Its exponentials come from the series of exp on [-ln 2 / 2, ln 2 / 2],
// whose terms past x^11 are below 2^-47; a 64-bit fma takes a wave as long as a 32-bit one
// here, and a row's read hides them.  Within a beam the score rises with the logit, so that
// a row's K best are the K largest logits:
//
//   * k_beam_row: a workgroup a segment of a row, which it reads once, to registers:
//     maximum, sum of exponentials, and its K best as keys (order key of the logit, then
//     the id counted down: larger is better).  Of the threads' maxima the K-th largest,
//     found by its leading digits, is a bound that K elements reach; the few above it meet
//     in LDS, where each counts those that are better.
//   * k_beam_join: a workgroup a group; the same over its beams' candidates.
//
// Where more elements tie at the bound than LDS has room for, the K best are taken one by one.
#include <hip/hip_runtime.h>

#include "../../include/pz_sampler.h"
#include "pz_device.h"
#include "pz_pages.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"

namespace {

constexpr int BE_CAP = 2048;   // elements of a segment that meet in LDS
constexpr int BE_JCAP = 1024;  // candidates of a group that do
constexpr int BE_SLACK = 64;   // how many more than K a bound may let through

struct BeamStat {
  double sum;  // of exp(x - m)
  float m;     // the segment's maximum, -infinity without a finite logit
  int bad;     // a NaN or +infinity
};

struct BeamArgs {
  const float* x;
  long ld;
  int W, V, S, K;  // beams, ids, segments of a row
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

// exp(d), d <= 0.
__device__ __forceinline__ double be_exp(double d) {
  d = d > -1000.0 ? d : -1000.0;  // (0 from -746 on)
  const double t = d * 1.44269504088896340736, k = rint(t);
  const double r = (t - k) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = __builtin_fma(r, p, 1.0 / 3628800.0);
  p = __builtin_fma(r, p, 1.0 / 362880.0);
  p = __builtin_fma(r, p, 1.0 / 40320.0);
  p = __builtin_fma(r, p, 1.0 / 5040.0);
  p = __builtin_fma(r, p, 1.0 / 720.0);
  p = __builtin_fma(r, p, 1.0 / 120.0);
  p = __builtin_fma(r, p, 1.0 / 24.0);
  p = __builtin_fma(r, p, 1.0 / 6.0);
  p = __builtin_fma(r, p, 0.5);
  p = __builtin_fma(r, p, 1.0);
  p = __builtin_fma(r, p, 1.0);
  return __builtin_ldexp(p, (int)k);
}

__device__ __forceinline__ double be_wave_sum(double v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

__device__ __forceinline__ uint64_t be_key(float x, int id) {
  return (uint64_t)pz_key(x) << 32 | (0xffffffffu - (uint32_t)id);
}
constexpr uint32_t BE_NONE = 0x007fffffu;  // the order key of -infinity

// The bound T of at most 32 leading bits that at least K of the keys reach (0 where there
// are fewer), found digit by digit until it lets no more than K + BE_SLACK of them through.
// each(f) calls f(key) for this thread's keys; keys of 0 are none.  hist: LDS [256].
template <int BLOCK, class EACH>
__device__ __forceinline__ uint32_t be_bound(int K, uint32_t* hist, EACH each) {
  const int lane = threadIdx.x & 63;
  uint32_t T = 0u;
  int need = K;  // of the keys that share T's digits so far
  for (int sh = 24; sh >= 0; sh -= 8) {
    for (int i = threadIdx.x; i < 256; i += BLOCK) hist[i] = 0u;
    __syncthreads();
    each([&](uint32_t key) {
      if (key && (sh == 24 || key >> (sh + 8) == T >> (sh + 8)))
        atomicAdd(&hist[key >> sh & 255u], 1u);
    });
    __syncthreads();
    // (every wave for itself) lane l's four digits, and how many keys lie above
    uint32_t n[4], own = 0u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      n[i] = hist[4 * lane + i];
      own += n[i];
    }
    uint32_t sum = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_down(sum, o, 64);
      sum += lane + o < 64 ? v : 0u;
    }
    const uint64_t enough = __ballot((int)sum >= need);
    __syncthreads();  // (hist is cleared next)
    if (!enough) return 0u;  // (only at the first digit)
    const int at = 63 - __clzll((unsigned long long)enough);
    int above = (int)(sum - own), digit = 3;
#pragma unroll
    for (int i = 3; i > 0; i--)
      if (digit == i && above + (int)n[i] < need) {
        above += (int)n[i];
        digit = i - 1;
      }
    const uint32_t in = digit == 3 ? n[3] : digit == 2 ? n[2] : digit == 1 ? n[1] : n[0];
    const int d = __builtin_amdgcn_readlane(4 * lane + digit, at);
    need -= __builtin_amdgcn_readlane(above, at);
    T |= (uint32_t)d << sh;
    if (__builtin_amdgcn_readlane((int)in, at) - need <= BE_SLACK) break;
  }
  return T;
}

template <int BLOCK, int NV>
__global__ __launch_bounds__(BLOCK) void k_beam_row(const BeamArgs A) {
  constexpr int WAVES = BLOCK / 64, N = 4 * NV;
  __shared__ uint64_t list[BE_CAP];
  __shared__ uint32_t hist[256];
  __shared__ double part[WAVES];
  __shared__ float top[WAVES];
  __shared__ int flag[WAVES];
  __shared__ int n_list;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int row = blockIdx.x / A.S, seg = blockIdx.x - row * A.S;
  // (what offers nothing is not read; the join sees the same)
  if (A.done && A.done[row]) return;
  if (!(fabsf(A.score[row]) < __builtin_inff())) return;
  const float* x = A.x + (size_t)row * A.ld;
  const int base = seg * (BLOCK * N);
  float v[N];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int i = base + (j * BLOCK + tid) * 4;
    if (i + 3 < A.V) {
      const pz_f4u q = *reinterpret_cast<const pz_f4u*>(x + i);
#pragma unroll
      for (int e = 0; e < 4; e++) v[4 * j + e] = q[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[4 * j + e] = i + e < A.V ? x[i + e] : -__builtin_inff();
    }
  }
  auto id_of = [&](int e) { return base + ((e >> 2) * BLOCK + tid) * 4 + (e & 3); };
  if (tid == 0) n_list = 0;
  float mine = -__builtin_inff();
  bool bad = false;
#pragma unroll
  for (int e = 0; e < N; e++) {
    mine = fmaxf(mine, v[e]);
    bad |= !(v[e] < __builtin_inff());
  }
  const float wm = pz_wave_max(mine);
  const bool wb = __ballot(bad) != 0;
  if (lane == 0) {
    top[w] = wm;
    flag[w] = wb;
  }
  __syncthreads();
  float m = top[0];
  int any = flag[0];
#pragma unroll
  for (int i = 1; i < WAVES; i++) {
    m = fmaxf(m, top[i]);
    any |= flag[i];
  }
  uint64_t* out = A.cand + (size_t)blockIdx.x * A.K;
  if (any || m == -__builtin_inff()) {
    for (int i = tid; i < A.K; i += BLOCK) out[i] = 0u;
    if (tid == 0) A.stat[blockIdx.x] = {0.0, m, any};
    return;
  }
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < N; e++) sum += be_exp((double)v[e] - (double)m);
  sum = be_wave_sum(sum);
  if (lane == 0) part[w] = sum;
  // the K best
  const uint32_t tk = mine == -__builtin_inff() ? 0u : pz_key(mine);
  const uint32_t T = be_bound<BLOCK>(A.K, hist, [&](auto f) { f(tk); });
  if (tk >= T)
#pragma unroll
    for (int e = 0; e < N; e++) {
      const uint32_t k = pz_key(v[e]);
      if (k >= T && k > BE_NONE) {
        const int at = atomicAdd(&n_list, 1);
        if (at < BE_CAP) list[at] = be_key(v[e], id_of(e));
      }
    }
  __syncthreads();
  const int n = n_list;
  if (tid == 0) {
    double s = part[0];
#pragma unroll
    for (int i = 1; i < WAVES; i++) s += part[i];
    A.stat[blockIdx.x] = {s, m, 0};
  }
  for (int i = n + tid; i < A.K; i += BLOCK) out[i] = 0u;
  if (n <= BE_CAP) {
    for (int i = tid; i < n; i += BLOCK) {
      const uint64_t k = list[i];
      int better = 0;
      for (int j = 0; j < n; j++) better += list[j] > k;
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
    __syncthreads();
    if (lane == 0) list[w] = best;
    __syncthreads();
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
  if (a.score != b.score) return a.score > b.score;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}

constexpr int BE_JOIN = 1024;  // threads

__global__ __launch_bounds__(BE_JOIN) void k_beam_join(const BeamArgs A) {
  constexpr int WAVES = BE_JOIN / 64;
  __shared__ BeamCand list[BE_JCAP];
  __shared__ uint32_t hist[256];
  __shared__ double lse[PZ_BEAM_MAX_WIDTH], sum[PZ_BEAM_MAX_WIDTH];
  __shared__ int state[PZ_BEAM_MAX_WIDTH];  // 0: offers nothing, 1: its row, 2: itself
  __shared__ int n_list;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row0 = (int64_t)blockIdx.x * A.W;
  if (tid == 0) n_list = 0;
  for (int b = w; b < A.W; b += WAVES) {
    const int64_t row = row0 + b;
    const float sc = A.score[row];
    int st = !(fabsf(sc) < __builtin_inff()) ? 0 : A.done && A.done[row] ? 2 : 1;
    double l = 0.0;
    if (st == 1) {
      const BeamStat* s = A.stat + row * A.S;
      float m = -__builtin_inff();
      bool bad = false;
      for (int i = lane; i < A.S; i += 64) {
        bad |= s[i].bad != 0;
        m = fmaxf(m, s[i].m);
      }
      m = pz_wave_max(m);
      if (__ballot(bad) || m == -__builtin_inff()) {
        st = 0;
      } else {
        for (int i = lane; i < A.S; i += 64)
          if (s[i].m > -__builtin_inff()) l += s[i].sum * be_exp((double)s[i].m - (double)m);
        l = (double)m + log(be_wave_sum(l));
      }
    }
    if (lane == 0) {
      state[b] = st;
      sum[b] = (double)sc;
      lse[b] = l;
    }
  }
  __syncthreads();
  const int per = A.S * A.K, total = A.W * per;
  const uint64_t* cand = A.cand + row0 * per;
  // candidate e: of beam e / per, then one of every beam that has ended
  auto get = [&](int e, BeamCand* c) {
    if (e < total) {
      c->beam = e / per;
      if (state[c->beam] != 1) return false;
      c->key = cand[e];
      if (!c->key) return false;
      c->score = sum[c->beam] + ((double)pz_unkey((uint32_t)(c->key >> 32)) - lse[c->beam]);
      return true;
    }
    c->beam = e - total;
    c->key = 0xffffffffu - (uint32_t)A.pad;
    c->score = sum[c->beam];
    return state[c->beam] == 2;
  };
  // (the nearest float rises with the score; none is infinite after a finite score but
  // where that is near the largest float, and then -infinity's key is a key like others)
  const uint32_t T = be_bound<BE_JOIN>(A.K, hist, [&](auto f) {
    for (int e = tid; e < total + A.W; e += BE_JOIN) {
      BeamCand c;
      if (get(e, &c)) f(pz_key((float)c.score));
    }
  });
  for (int e = tid; e < total + A.W; e += BE_JOIN) {
    BeamCand c;
    if (get(e, &c) && pz_key((float)c.score) >= T) {
      const int at = atomicAdd(&n_list, 1);
      if (at < BE_JCAP) list[at] = c;
    }
  }
  __syncthreads();
  const int n = n_list;
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
  if (n <= BE_JCAP) {
    if (tid < n) {
      const BeamCand c = list[tid];
      int better = 0;
      for (int j = 0; j < n; j++) better += be_better(list[j], c);
      if (better < A.K) put(better, c);
    }
    return;
  }
  // one by one
  BeamCand last = {__builtin_inf(), ~0ull, -1};
  for (int k = 0; k < A.K; k++) {
    BeamCand best = {-__builtin_inf(), 0u, 1 << 30};
    for (int e = tid; e < total + A.W; e += BE_JOIN) {
      BeamCand c;
      if (get(e, &c) && be_better(last, c) && be_better(c, best)) best = c;
    }
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
    last = best;
  }
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
    int lo = 0, hi = A.n_pool;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (pool[mid] < page)
        lo = mid + 1;
      else
        hi = mid;
    }
    if (lo < A.n_pool && pool[lo] == page) atomicOr(&used[lo >> 5], 1u << (lo & 31));
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
  const int per = A.row / 8, n = c.z * per;  // 16-byte pieces
  for (int i = blockIdx.z * 256 + threadIdx.x; i < n; i += gridDim.z * 256) {
    const int p = i / per;
    const size_t at = (size_t)p * A.ld + (size_t)(i - p * per) * 8;
    *reinterpret_cast<be_u32x4*>(buf + dst * A.ld + at) =
        *reinterpret_cast<const be_u32x4*>(buf + src * A.ld + at);
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
  constexpr int LONG = 512 * 16, SHORT = 256 * 8;
  const bool few = rows * ((V + LONG - 1) / LONG) < 2 * (int64_t)s->n_cu;
  const int S = few ? (V + SHORT - 1) / SHORT : (V + LONG - 1) / LONG;
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
    if (few)
      hipLaunchKernelGGL((k_beam_row<256, 2>), dim3((unsigned)n * W * S), dim3(256), 0, s->stream,
                         A);
    else
      hipLaunchKernelGGL((k_beam_row<512, 4>), dim3((unsigned)n * W * S), dim3(512), 0, s->stream,
                         A);
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
  hipLaunchKernelGGL(k_beam_plan, dim3((unsigned)n_groups), dim3(BE_PLAN),
                     ((size_t)n_pool + 31) / 32 * 4, s->stream, R);
  PZ_HIP(s, hipGetLastError());
  // workgroups of a page: 16 positions each
  const int parts = c.block_size < 16 * 64 ? (c.block_size + 15) / 16 : 64;
  for (int l = 0; l < n_layers; l += BE_LAYERS) {
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
    hipLaunchKernelGGL(k_beam_copy, dim3((unsigned)(n_groups * W), 2u * n, (unsigned)parts),
                       dim3(256), 0, s->stream, A);
    PZ_HIP(s, hipGetLastError());
  }
  return PZ_OK;
}
