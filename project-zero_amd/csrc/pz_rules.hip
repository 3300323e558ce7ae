// pz_rules.hip -- logit rules (pz_rules_batch): penalties over a history of
// any length, biases and grammar masks, between the LM head and the sampler.
//
// Per row: a table in LDS of the ids that the history or the bias list names,
// with their counts and their first bias entry, then
//   y = in[i]; c > 0: y = (y > 0 ? y / rep : y * rep) - (c * freq + pres)
//   (the samplers' own penalties, pz_penalize); y += bias, entry by entry;
//   masked ids: -infinity.
// Integer atomics only, so the order in which ids arrive changes nothing; the
// bias entries of one id are added in the list's order.
//
//   * A row is cut into slices of W ids, one workgroup each; a workgroup reads
//     the whole history and keeps the ids of its slice.  In place and without
//     masks only the named ids are touched: one slice, a hash table of twice
//     the entries.  Lists too long for that take a table indexed by the id
//     itself (DENSE); there ids with several bias entries are added up in LDS by
//     one more pass over the list.
//   * With masks, or out of place, the slice's ids also stream through: 4 NQ
//     ids a thread, all loads of them issued before the table is made, the
//     slice's mask words in LDS, one 16-byte store where anything changes.  In
//     place, nothing of an all-allowed group is read or written.
//   * d_allowed has a workgroup of its own per row, beside the slices.
#include <hip/hip_runtime.h>

#include "../../include/pz_sampler.h"
#include "pz_device.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"

namespace {

constexpr int RU_NONE = 0x7fffffff;         // no bias entry
constexpr uint32_t RU_TWICE = 0x80000000u;  // in a count (DENSE): the id has more bias entries
constexpr int RU_WALK = 12;                 // (!DENSE) entries of one id that its thread walks through itself

struct RulesArgs {
  const float* in;
  long ld_in;
  float* out;
  long ld_out;
  int V, W, S, cap;  // ids, ids of a slice, slices of a row, slots of a table
  int count;         // 1: a workgroup more per row counts what its mask allows
  pz_logit_rules r;
};

typedef int32_t ru_i4u __attribute__((ext_vector_type(4), aligned(4)));

// Mask words of row b (nullptr: none).
__device__ __forceinline__ const uint32_t* ru_mask(const pz_logit_rules& r, int b) {
  if (r.n_masks <= 0) return nullptr;
  const int m = r.d_mask_row ? r.d_mask_row[b] : b;
  return m >= 0 && m < r.n_masks ? r.d_mask + (size_t)m * r.ld_mask : nullptr;
}

// The table: per slot the count and a bias entry (DENSE: the first, and a mark
// in the count where there are more; else the last to arrive, the others
// chained to it), and with !DENSE the id (-1: empty).
template <bool DENSE>
struct RuTable {
  uint32_t* cnt;
  int32_t* first;
  int32_t* key;
  int32_t* used;  // (!DENSE) the slots taken, in no order, and how many
  int* n_used;
  int base, lim, cap;
  __device__ __forceinline__ int slot(int id) const {
    if (DENSE) return id - base;
    const uint32_t mask = (uint32_t)cap - 1u;
    uint32_t s = pz_hash((uint32_t)id) & mask;
    // at most half of the slots are ever taken, so an empty one ends this
    while (true) {
      const int prev = atomicCAS(&key[s], -1, id);
      if (prev == -1) used[atomicAdd(n_used, 1)] = (int)s;
      if (prev == -1 || prev == id) return (int)s;
      s = (s + 1) & mask;
    }
  }
};

// The number of ids that a mask allows, by one workgroup.
template <int BLOCK>
__device__ __forceinline__ int ru_count(const uint32_t* mask, int V) {
  __shared__ int n_on;
  if (threadIdx.x == 0) n_on = 0;
  __syncthreads();
  int n = 0;
  const int words = (V + 31) >> 5;
#pragma unroll 4
  for (int w = threadIdx.x; w < words; w += BLOCK) {
    const uint32_t tail = w == words - 1 && (V & 31) ? (1u << (V & 31)) - 1u : ~0u;
    n += __popc(mask[w] & tail);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
  if ((threadIdx.x & 63) == 0) atomicAdd(&n_on, n);
  __syncthreads();
  return n_on;
}

// NQ 0: only the named ids that the mask allows.
template <bool DENSE, int NQ, int BLOCK>
__global__ __launch_bounds__(BLOCK) void k_rules(const RulesArgs A) {
  constexpr int U = 4;  // slots of a thread whose logits are on their way together
  extern __shared__ __align__(16) char lds[];
  __shared__ uint32_t on_sh[NQ ? NQ * BLOCK / 8 : 1];
  __shared__ int n_used;
  __shared__ int n_many;  // (DENSE) whether an id has more bias entries than one
  const pz_logit_rules& r = A.r;
  const int tid = threadIdx.x, lane = tid & 63;
  const int per = A.S + A.count;
  const int b = blockIdx.x / per, sl = blockIdx.x - b * per;
  const int V = A.V;
  // (the first of the history while the mask and the parameters arrive)
  const int32_t* h = r.d_hist + (size_t)b * r.H;
  ru_i4u h0;
  if (4 * tid + 3 < r.H) h0 = *reinterpret_cast<const ru_i4u*>(h + 4 * tid);
  const uint32_t* mask = ru_mask(r, b);
  if (sl == A.S) {
    const int n = mask ? ru_count<BLOCK>(mask, V) : V;
    if (tid == 0) r.d_allowed[b] = n;
    return;
  }
  RuTable<DENSE> T;
  T.base = sl * A.W;
  T.lim = V - T.base < A.W ? V : T.base + A.W;
  T.cap = A.cap;
  T.cnt = reinterpret_cast<uint32_t*>(lds);
  T.first = reinterpret_cast<int32_t*>(lds) + T.cap;
  T.key = reinterpret_cast<int32_t*>(lds) + 2 * T.cap;
  T.used = T.key + T.cap;  // (at most half of the slots)
  T.n_used = &n_used;
  // (!DENSE) the entry that named an entry's id before it
  int32_t* next = T.used + T.cap / 2;
  const float* in = A.in + (size_t)b * A.ld_in;
  float* out = A.out + (size_t)b * A.ld_out;
  const bool inplace = A.in == A.out;
  pz_f4u q[NQ ? NQ : 1];
  if constexpr (NQ > 0) {
    if (!inplace) {
#pragma unroll
      for (int k = 0; k < NQ; k++) {
        const int i = T.base + 4 * (k * BLOCK + tid);
        if (i + 3 < T.lim) {
          q[k] = *reinterpret_cast<const pz_f4u*>(in + i);
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) q[k][e] = i + e < T.lim ? in[i + e] : 0.0f;
        }
      }
    }
    if (mask)
#pragma unroll
      for (int w = tid; w < NQ * BLOCK / 8; w += BLOCK)
        on_sh[w] = T.base + 32 * w < T.lim ? mask[(T.base >> 5) + w] : 0u;
  }
  float rep = r.rep_penalty, pres = r.presence_penalty, freq = r.frequency_penalty;
  if (r.d_penalties) {
    rep = r.d_penalties[3 * (size_t)b];
    pres = r.d_penalties[3 * (size_t)b + 1];
    freq = r.d_penalties[3 * (size_t)b + 2];
  }
  int H = r.H;
  if (H > 0 && r.d_hist_len) {
    const int n = r.d_hist_len[b];
    H = n < 0 ? 0 : (n < H ? n : H);
  }
  if (rep == 1.0f && pres == 0.0f && freq == 0.0f) H = 0;
  const bool lists = H > 0 || r.n_bias > 0;
  const int32_t* bid = r.d_bias_ids + (size_t)b * r.n_bias;
  const float* bias = r.d_bias + (size_t)b * r.n_bias;

  if (lists) {
    for (int i = tid; i < T.cap; i += BLOCK) {
      T.cnt[i] = 0u;
      T.first[i] = RU_NONE;
      if (!DENSE) T.key[i] = -1;
    }
    if (tid == 0) n_used = n_many = 0;
    __syncthreads();
    auto seen = [&](int id) {
      if (id >= T.base && id < T.lim) atomicAdd(&T.cnt[T.slot(id)], 1u);
    };
    const int H4 = H & ~3;
    if (4 * tid < H4)
#pragma unroll
      for (int e = 0; e < 4; e++) seen(h0[e]);
    int j = 4 * (BLOCK + tid);
    for (; j < H4 - 12 * BLOCK; j += 16 * BLOCK) {  // (four loads on their way)
      ru_i4u h4[4];
#pragma unroll
      for (int k = 0; k < 4; k++)
        h4[k] = *reinterpret_cast<const ru_i4u*>(h + j + 4 * k * BLOCK);
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) seen(h4[k][e]);
    }
    for (; j < H4; j += 4 * BLOCK) {
      const ru_i4u h4 = *reinterpret_cast<const ru_i4u*>(h + j);
#pragma unroll
      for (int e = 0; e < 4; e++) seen(h4[e]);
    }
    for (j = H4 + tid; j < H; j += BLOCK) seen(h[j]);
    for (int e = tid; e < r.n_bias; e += BLOCK) {
      const int id = bid[e];
      if (id < T.base || id >= T.lim) continue;
      const int at = T.slot(id);
      if (!DENSE) next[e] = atomicExch(&T.first[at], e);
      else if (atomicMin(&T.first[at], e) != RU_NONE) atomicOr(&T.cnt[at], RU_TWICE);
    }
  }
  if constexpr (NQ > 0) {
    if (mask && !lists) __syncthreads();
    // (with lists, the barrier after the tables were cleared)
    const float ninf = -__builtin_inff();
    uint32_t on[NQ];
#pragma unroll
    for (int k = 0; k < NQ; k++) {
      const int t = k * BLOCK + tid, i = T.base + 4 * t;
      on[k] = mask ? on_sh[t >> 3] >> (4 * (t & 7)) & 0xfu : 0xfu;
      if (inplace && on[k] != 0xfu && on[k] != 0u && i + 3 < T.lim)
        q[k] = *reinterpret_cast<const pz_f4u*>(in + i);
    }
#pragma unroll
    for (int k = 0; k < NQ; k++) {
      const int i = T.base + 4 * (k * BLOCK + tid);
      if (inplace && on[k] == 0xfu) continue;
      if (i + 3 < T.lim) {
#pragma unroll
        for (int e = 0; e < 4; e++) q[k][e] = on[k] >> e & 1u ? q[k][e] : ninf;
        *reinterpret_cast<pz_f4u*>(out + i) = q[k];
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const bool keep = on[k] >> e & 1u;
          if (i + e < T.lim && !(inplace && keep)) out[i + e] = keep ? q[k][e] : ninf;
        }
      }
    }
  }
  if (!lists) return;
  __syncthreads();  // the table is complete, and so is the slice's stream
  const int slots = DENSE ? T.cap : n_used;
  for (int i0 = 0; i0 < slots; i0 += U * BLOCK) {
    uint32_t c[U];
    int f[U], id[U];
    float x[U], bv[U];
    bool act[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = i0 + u * BLOCK + tid;
      c[u] = 0u;
      f[u] = RU_NONE;
      id[u] = 0;
      if (at < slots) {
        const int i = DENSE ? at : T.used[at];
        c[u] = T.cnt[i];
        f[u] = T.first[i];
        id[u] = DENSE ? T.base + i : T.key[i];
      }
      act[u] = c[u] != 0u || f[u] != RU_NONE;
      if (act[u] && mask)
        act[u] = (NQ ? on_sh[(id[u] - T.base) >> 5] : mask[id[u] >> 5]) >> (id[u] & 31) & 1u;
      x[u] = bv[u] = 0.0f;
      if (act[u]) x[u] = in[id[u]];
      if (act[u] && f[u] != RU_NONE) bv[u] = bias[f[u]];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t times = c[u] & ~RU_TWICE;
      if (act[u] && times) {
        x[u] = x[u] > 0.0f ? x[u] / rep : x[u] * rep;
        float t = (float)times * freq;
        t = t + pres;
        x[u] = x[u] - t;
      }
      if (DENSE && act[u] && (c[u] & RU_TWICE)) {
        // (its entries: below)
        T.first[i0 + u * BLOCK + tid] = __float_as_int(x[u]);
        n_many = 1;
        act[u] = false;
      }
      bool many = false;
      if (act[u] && f[u] != RU_NONE) {
        int n = 1;
        if (!DENSE)
          for (int e = next[f[u]]; e != RU_NONE && n <= RU_WALK; e = next[e]) n++;
        many = n > RU_WALK;
        if (n == 1) {
          x[u] = x[u] + bv[u];
        } else if (!many) {
          // a short chain, in no order: its entries in the list's order
          for (int last = -1, k = 0; k < n; k++) {
            int lo = RU_NONE;
            for (int e = f[u]; e != RU_NONE; e = next[e]) lo = e > last && e < lo ? e : lo;
            x[u] = x[u] + bias[lo];
            last = lo;
          }
        }
      }
      // an id with many entries: the wave looks through the list, of at most 4096
      if constexpr (!DENSE) {
        for (uint64_t todo = __ballot(many); todo; todo &= todo - 1) {
          const int L = __builtin_ctzll(todo);
          const int its = __builtin_amdgcn_readlane(id[u], L);
          float v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x[u]), L));
          for (int e0 = 0; e0 < r.n_bias; e0 += 64) {
            const int e = e0 + lane;
            const bool is = e < r.n_bias && bid[e] == its;
            const int more = is ? __float_as_int(bias[e]) : 0;
            for (uint64_t hit = __ballot(is); hit; hit &= hit - 1)
              v = v + __int_as_float(__builtin_amdgcn_readlane(more, __builtin_ctzll(hit)));
          }
          if (lane == L) x[u] = v;
        }
      }
      if (act[u]) out[id[u]] = x[u];
    }
  }
  if constexpr (DENSE) {
    // Ids with more than one entry: each wave reads the list once, in order, and
    // adds what belongs to its share of them, where their logits stand in LDS.  (The
    // list once for every id: 2^18 entries over 100000 ids 154 ms, 1.05 so; 2^16 over
    // 1000 22.8 and 1.07.)
    __syncthreads();
    if (!n_many) return;
    const int w = tid >> 6;
    for (int e0 = 0; e0 < r.n_bias; e0 += 64) {
      const int e = e0 + lane, id = e < r.n_bias ? bid[e] : -1;
      const bool here = id >= T.base && id < T.lim;
      const int at = here ? id - T.base : 0;
      const bool mine = here && (at & (BLOCK / 64 - 1)) == w && (T.cnt[at] & RU_TWICE);
      const int add = mine ? __float_as_int(bias[e]) : 0;
      for (uint64_t todo = __ballot(mine); todo; todo &= todo - 1) {
        const int L = __builtin_ctzll(todo);
        const int to = __builtin_amdgcn_readlane(at, L);
        const float v = __int_as_float(__builtin_amdgcn_readlane(add, L));
        if (lane == 0) T.first[to] = __float_as_int(__int_as_float(T.first[to]) + v);
      }
    }
    __syncthreads();
    for (int i = tid; i < T.lim - T.base; i += BLOCK) {
      const int id = T.base + i;
      if ((T.cnt[i] & RU_TWICE) && (!mask || (mask[id >> 5] >> (id & 31) & 1u)))
        out[id] = __int_as_float(T.first[i]);
    }
  }
}

int next_pow2(long v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

template <bool DENSE, int NQ, int BLOCK>
int launch(pz_sampler* s, RulesArgs& A, int B, size_t slot_bytes) {
  if (NQ > 0) A.W = 4 * BLOCK * NQ;
  A.S = (A.V + A.W - 1) / A.W;
  if (DENSE) A.cap = A.W;
  const int64_t grid = (int64_t)B * (A.S + A.count);
  if (!pz_launch_fits(grid, BLOCK)) return fail(s, PZ_ERANGE, "B=%d rows of V=%d", B, A.V);
  const size_t lds = (size_t)A.cap * slot_bytes + (DENSE ? 0 : (size_t)A.r.n_bias * 4);
  // (the counting workgroups and the mask words have LDS of their own)
  auto k = k_rules<DENSE, NQ, BLOCK>;
  if (lds > 65536 - 4096)
    PZ_HIP(s, hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)lds));
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(BLOCK), lds, s->stream, A);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}

}  // namespace

extern "C" int pz_rules_batch(pz_sampler* s, const float* d_in, long ld_in, float* d_out,
                              long ld_out, int B, int V, const pz_logit_rules* rules) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no = pz_refuse_rules(d_in, ld_in, d_out, ld_out, B, V, rules);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (B == 0) return PZ_OK;
  RulesArgs A;
  A.in = d_in;
  A.ld_in = ld_in;
  A.out = d_out;
  A.ld_out = ld_out;
  A.V = V;
  A.r = *rules;
  const bool stream = d_in != d_out || A.r.n_masks > 0;
  const long entries = (long)A.r.H + A.r.n_bias;
  A.count = A.r.d_allowed ? 1 : 0;
  if (!stream && entries == 0 && !A.count) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  // few rows: smaller slices, so that every CU has some
  const bool few = (int64_t)B * ((V + 8191) / 8192) < 2 * s->n_cu;
  if (stream) {
    // Lists of up to 1024 entries are applied by the slices that stream; longer
    // ones by a launch after them, because their tables leave room for fewer
    // workgroups of the stream (256 rows of 151936 out of place with masks: 69
    // us at H = 512, 104 at 1984 where a launch of its own makes it 81; 64 of
    // 128256 in place at H = 2048 22.8 and 17.9).
    RulesArgs L = A;
    if (entries > 1024) L.r.H = L.r.n_bias = L.cap = 0;
    else L.cap = entries == 0 ? 0 : next_pow2(2 * entries);
    const int rc = few ? launch<false, 2, 256>(s, L, B, 14) : launch<false, 8, 256>(s, L, B, 14);
    if (rc != PZ_OK || entries <= 1024) return rc;
    A.count = 0;
  }
  // A hash table takes 14 bytes a slot at two slots an entry and 4 bytes a bias:
  // up to 4096 entries fit, and one workgroup reads a row's history, not one
  // per slice (256 rows of 128256, H = 2049: 7 us, 72 with a table per slice).
  if (entries > 4096) {
    A.W = few ? 2048 : 8192;
    return launch<true, 0, 512>(s, A, B, 8);
  }
  A.W = (V + 31) / 32 * 32;
  A.cap = entries == 0 ? 0 : next_pow2(2 * entries);
  // (H = 2048: 256 threads 10.7 us for one row, 13.0 for 256; 1024 5.1 and 7.1)
  return entries <= 256 ? launch<false, 0, 256>(s, A, B, 14) : launch<false, 0, 1024>(s, A, B, 14);
}
