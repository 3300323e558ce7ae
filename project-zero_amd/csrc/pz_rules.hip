// pz_rules.hip -- logit rules (pz_rules_batch): penalties over a history of
// any length, biases and grammar masks, between the LM head and the sampler.
//
// Per row: a table in LDS of the ids that the history or the bias list names,
// with their counts and their first bias entry, then
//   y = in[i]; c > 0: y = (y > 0 ? y / rep : y * rep) - (c * freq + pres)
//   (the samplers' own penalties, pz_penalize); y += bias, entry by entry;
//   masked ids: -infinity.
// Integer atomics only, so the order in which ids arrive changes nothing; two
// bias entries of one id are added by one thread in the list's order.
//
//   * A row is cut into slices of W ids, one workgroup each; a workgroup reads
//     the whole history and keeps the ids of its slice.  In place and without
//     masks only the named ids are touched: one slice, a hash table of twice
//     the entries.  Lists too long for that take a table indexed by the id
//     itself (DENSE), 8192 ids a slice.
//   * With masks, or out of place, the slice's ids also stream through: four
//     ids a thread, a mask nibble, one 16-byte store where anything changes.
//     In place, nothing of an all-allowed group is read or written.
#include <hip/hip_runtime.h>

#include "../../include/pz_sampler.h"
#include "pz_device.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"

namespace {

constexpr int RU_NONE = 0x7fffffff;  // no bias entry

struct RulesArgs {
  const float* in;
  long ld_in;
  float* out;
  long ld_out;
  int V, W, S, cap;  // ids, ids of a slice, slices of a row, hash entries
  pz_logit_rules r;
};

typedef int32_t ru_i4u __attribute__((ext_vector_type(4), aligned(4)));

// Mask words of row b (nullptr: none).
__device__ __forceinline__ const uint32_t* ru_mask(const pz_logit_rules& r, int b) {
  if (r.n_masks <= 0) return nullptr;
  const int m = r.d_mask_row ? r.d_mask_row[b] : b;
  return m >= 0 && m < r.n_masks ? r.d_mask + (size_t)m * r.ld_mask : nullptr;
}

// The table: per slot the count and the first bias entry, and with !DENSE the
// id (-1: empty).
template <bool DENSE>
struct RuTable {
  uint32_t* cnt;
  int32_t* first;
  int32_t* key;
  int base, lim, cap;
  __device__ __forceinline__ int slot(int id) const {
    if (DENSE) return id - base;
    const uint32_t mask = (uint32_t)cap - 1u;
    uint32_t s = pz_hash((uint32_t)id) & mask;
    // at most half of the slots are ever taken, so an empty one ends this
    while (true) {
      const int prev = atomicCAS(&key[s], -1, id);
      if (prev == -1 || prev == id) return (int)s;
      s = (s + 1) & mask;
    }
  }
};

template <bool DENSE, bool STREAM, int BLOCK>
__global__ __launch_bounds__(BLOCK) void k_rules(const RulesArgs A) {
  extern __shared__ __align__(16) char lds[];
  __shared__ int dup, n_on;
  const pz_logit_rules& r = A.r;
  const int tid = threadIdx.x;
  const int b = blockIdx.x / A.S, sl = blockIdx.x - b * A.S;
  const int V = A.V;
  RuTable<DENSE> T;
  T.base = sl * A.W;
  T.lim = V - T.base < A.W ? V : T.base + A.W;
  T.cap = DENSE ? A.W : A.cap;
  T.cnt = reinterpret_cast<uint32_t*>(lds);
  T.first = reinterpret_cast<int32_t*>(lds) + T.cap;
  T.key = reinterpret_cast<int32_t*>(lds) + 2 * T.cap;
  const float* in = A.in + (size_t)b * A.ld_in;
  float* out = A.out + (size_t)b * A.ld_out;
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
  const uint32_t* mask = ru_mask(r, b);
  const bool lists = H > 0 || r.n_bias > 0;

  if (lists) {
    for (int i = tid; i < T.cap; i += BLOCK) {
      T.cnt[i] = 0u;
      T.first[i] = RU_NONE;
      if (!DENSE) T.key[i] = -1;
    }
    if (tid == 0) dup = 0;
    __syncthreads();
    const int32_t* h = r.d_hist + (size_t)b * r.H;
    auto seen = [&](int id) {
      if (id >= T.base && id < T.lim) atomicAdd(&T.cnt[T.slot(id)], 1u);
    };
    const int H4 = H & ~3;
    for (int j = 4 * tid; j < H4; j += 4 * BLOCK) {
      const ru_i4u q = *reinterpret_cast<const ru_i4u*>(h + j);
#pragma unroll
      for (int e = 0; e < 4; e++) seen(q[e]);
    }
    for (int j = H4 + tid; j < H; j += BLOCK) seen(h[j]);
    const int32_t* bid = r.d_bias_ids + (size_t)b * r.n_bias;
    for (int e = tid; e < r.n_bias; e += BLOCK) {
      const int id = bid[e];
      if (id >= T.base && id < T.lim && atomicMin(&T.first[T.slot(id)], e) != RU_NONE) dup = 1;
    }
  }
  if (STREAM) {
    const bool inplace = A.in == A.out;
    const float ninf = -__builtin_inff();
    if (!inplace || mask)
      for (int i = T.base + 4 * tid; i < T.lim; i += 4 * BLOCK) {
        const uint32_t on = mask ? mask[i >> 5] >> (i & 31) & 0xfu : 0xfu;
        if (inplace && on == 0xfu) continue;
        if (i + 3 < T.lim) {
          pz_f4u q;
          if (!inplace) q = *reinterpret_cast<const pz_f4u*>(in + i);
          if (!inplace || on == 0u) {
#pragma unroll
            for (int e = 0; e < 4; e++) q[e] = on >> e & 1u ? q[e] : ninf;
            *reinterpret_cast<pz_f4u*>(out + i) = q;
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (!(on >> e & 1u)) out[i + e] = ninf;
          }
        } else {
          for (int e = 0; i + e < T.lim; e++) {
            if (!(on >> e & 1u)) out[i + e] = ninf;
            else if (!inplace) out[i + e] = in[i + e];
          }
        }
      }
  }
  if (lists) {
    __syncthreads();  // the table is complete, and so is the slice's stream
    const int32_t* bid = r.d_bias_ids + (size_t)b * r.n_bias;
    const float* bias = r.d_bias + (size_t)b * r.n_bias;
    const bool twice = dup != 0;
    for (int i = tid; i < T.cap; i += BLOCK) {
      const uint32_t c = T.cnt[i];
      const int f = T.first[i];
      if (c == 0u && f == RU_NONE) continue;
      const int id = DENSE ? T.base + i : T.key[i];
      if (mask && !(mask[id >> 5] >> (id & 31) & 1u)) continue;
      float x = in[id];
      if (c) {
        x = x > 0.0f ? x / rep : x * rep;
        float t = (float)c * freq;
        t = t + pres;
        x = x - t;
      }
      if (f != RU_NONE) {
        x = x + bias[f];
        if (twice)
          for (int e = f + 1; e < r.n_bias; e++)
            if (bid[e] == id) x = x + bias[e];
      }
      out[id] = x;
    }
  }
  if (r.d_allowed && sl == 0) {
    // (the row's first workgroup counts all of it)
    if (!mask) {
      if (tid == 0) r.d_allowed[b] = V;
      return;
    }
    if (tid == 0) n_on = 0;
    __syncthreads();
    int n = 0;
    const int words = (V + 31) >> 5;
    for (int w = tid; w < words; w += BLOCK) {
      const uint32_t tail = w == words - 1 && (V & 31) ? (1u << (V & 31)) - 1u : ~0u;
      n += __popc(mask[w] & tail);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
    if ((tid & 63) == 0) atomicAdd(&n_on, n);
    __syncthreads();
    if (tid == 0) r.d_allowed[b] = n_on;
  }
}

int next_pow2(long v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

constexpr int RU_HASH_MOST = 2048;  // list entries a hash table is made for
constexpr int RU_DENSE = 8192;      // ids of a slice with a table of its own

template <bool DENSE, bool STREAM, int BLOCK>
int launch(pz_sampler* s, const RulesArgs& A, int B, size_t lds) {
  auto k = k_rules<DENSE, STREAM, BLOCK>;
  if (lds > 65536)
    PZ_HIP(s, hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)lds));
  hipLaunchKernelGGL(k, dim3((unsigned)B * (unsigned)A.S), dim3(BLOCK), lds, s->stream, A);
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
  if (!stream && entries == 0 && !A.r.d_allowed) return PZ_OK;
  const bool dense = entries > RU_HASH_MOST;
  A.W = dense || stream ? RU_DENSE : (V + 31) / 32 * 32;
  A.S = (V + A.W - 1) / A.W;
  if ((long)B * A.S > INT32_MAX) return fail(s, PZ_ERANGE, "B=%d rows of V=%d", B, V);
  A.cap = dense ? 0 : next_pow2(2 * entries);
  const size_t lds = entries == 0 ? 0 : dense ? (size_t)A.W * 8 : (size_t)A.cap * 12;
  PZ_HIP(s, hipSetDevice(s->device));
  if (dense) return stream ? launch<true, true, 1024>(s, A, B, lds)
                           : launch<true, false, 1024>(s, A, B, lds);
  return stream ? launch<false, true, 256>(s, A, B, lds) : launch<false, false, 256>(s, A, B, lds);
}
