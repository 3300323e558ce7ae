// pz_rope.hip -- RMS norm of each head of queries and keys and its rotation to the
// token's position (pz_qk_norm_rope).
//
//   y = x w / sqrt(mean(x^2) + eps);  (a, b) -> (a cos - b sin, b cos + a sin) amplitude
//
// The angle pos * freq is wanted modulo a turn.  In 64 bits, in quarter turns, t = pos * (freq
// 2 / pi) is off by at most 3 2^-53 of itself (below 2^-24 up to 2^27 radians); its distance to
// the nearest whole number (at most a half: at most pi / 4), which is exact below 2^51 quarters,
// is left for fp32, where the series of sine and cosine stop after x^9 and x^10 (terms of 2e-9
// and 1e-10 are left out at pi / 4).
//
// k_qk_rope: a head is LG lanes, each of which owns two 16-byte vectors: of the same
// place in the two halves (ROPE_HALVES; past the rotated part, the next two), or
// neighbours (ROPE_PAIRS), so that both elements of a pair are in one lane.  Halves that
// are no whole vectors (ROPE_ODD) are neighbours, too, and an element's other one comes
// from LDS.  A wave takes 64 / LG heads at once and `turns` times that many of one token,
// whose angles it makes once; the next heads are on their way meanwhile.  Bound by memory:
// 16384 tokens of 32 + 8 heads of 128 in bf16 (336 MB in and out) 74 us, 4.5 TB/s; 109 us
// with the norms' weights read for every head and with quotients and angles' quarters by
// conversions.  5000 tokens with 102 of 128 elements rotated in halves: 96 us in k_qk_rope_any, 37 so.
// k_qk_rope_any: one element pair a lane, a wave a head, whatever the sizes, strides and
// alignment.
#include <hip/hip_runtime.h>

#include "../../include/pz_sampler.h"
#include "pz_device.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"

namespace {

struct RopeArgs {
  const void* in[2];  // queries, keys
  void* out[2];
  long ld_in[2], ld_out[2];
  const float* norm[2];
  int heads[2];
  int D, rot;
  const float* freq;
  const int32_t* pos;
  float per_D, eps, amplitude;  // 1 / D
  int n, turns, waves;  // tokens, heads' groups of a wave, waves of a token
};

template <int TYPE>
struct RopeType;
template <>
struct RopeType<PZ_F32> {
  typedef float T;
  static constexpr int E = 4;  // elements of 16 bytes
  __device__ __forceinline__ static float widen(float v) { return v; }
  __device__ __forceinline__ static float narrow(float v) { return v; }
};
template <>
struct RopeType<PZ_BF16> {
  typedef __bf16 T;
  static constexpr int E = 8;
  __device__ __forceinline__ static float widen(__bf16 v) { return (float)v; }
  __device__ __forceinline__ static __bf16 narrow(float v) { return (__bf16)v; }
};
template <>
struct RopeType<PZ_F16> {
  typedef _Float16 T;
  static constexpr int E = 8;
  __device__ __forceinline__ static float widen(_Float16 v) { return (float)v; }
  __device__ __forceinline__ static _Float16 narrow(float v) { return (_Float16)v; }
};

// cos and sin of the angle of t quarter turns, |t| < 2^51.
__device__ __forceinline__ void rope_turn(double t, float& c, float& s) {
  constexpr double ROUND = 6755399441055744.0;  // 1.5 2^52: the sum's last bits are t's nearest
  const double q = t + ROUND;
  const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, q);
  const float x = (float)(t - (q - ROUND)) * 1.57079632679489661923f, z = x * x;
  // sin x = x - x^3/3! + ..., cos x = 1 - x^2/2! + ...
  float p = __builtin_fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
  p = __builtin_fmaf(z, p, 1.0f / 120.0f);
  p = __builtin_fmaf(z, p, -1.0f / 6.0f);
  const float sn = __builtin_fmaf(x * z, p, x);
  float r = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  r = __builtin_fmaf(z, r, -1.0f / 720.0f);
  r = __builtin_fmaf(z, r, 1.0f / 24.0f);
  r = __builtin_fmaf(z, r, -0.5f);
  const float cs = __builtin_fmaf(z, r, 1.0f);
  // quarters 0 .. 3: (cs, sn), (-sn, cs), (-cs, -sn), (sn, -cs)
  const uint32_t a = __float_as_uint(k & 1u ? sn : cs), b = __float_as_uint(k & 1u ? cs : sn);
  c = __uint_as_float(a ^ ((k + 1u) << 30 & 0x80000000u));
  s = __uint_as_float(b ^ (k << 30 & 0x80000000u));
}
// 1 / sqrt(v).  (The instruction takes no subnormal numbers.)
__device__ __forceinline__ float rope_rsqrt(float v) {
  const bool small = v < 0x1p-100f;
  const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p100f : v);
  return small ? r * 0x1p50f : r;
}
constexpr double ROPE_QUARTERS = 0.63661977236758134308;  // 2 / pi

enum RopeForm { ROPE_HALVES, ROPE_PAIRS, ROPE_ODD };

template <int TYPE, RopeForm FORM, int LG>
__global__ __launch_bounds__(256) void k_qk_rope(const RopeArgs A) {
  typedef RopeType<TYPE> Y;
  typedef typename Y::T T;
  constexpr int E = Y::E, HPW = 64 / LG;
  // angles of a lane: of its pairs, or (ROPE_ODD) of its elements
  constexpr int N = FORM == ROPE_ODD ? 2 * E : E;
  __shared__ float heads[FORM == ROPE_ODD ? 4 : 1][FORM == ROPE_ODD ? 64 * (2 * E + 1) : 1];
  typedef T vec __attribute__((ext_vector_type(E)));
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = (int)(wave / A.waves), part = (int)(wave - (int64_t)r * A.waves);
  if (r >= A.n) return;
  const int j = lane % LG, nv = A.D / E, rv = A.rot / 2 / E;
  int v0 = 2 * j, v1 = 2 * j + 1;
  if (FORM == ROPE_HALVES && j < rv) {
    v0 = j;
    v1 = rv + j;
  }
  const bool on0 = v0 < nv, on1 = v1 < nv;
  // groups of HPW heads, first the queries', then the keys'
  const int of_q = (A.heads[0] + HPW - 1) / HPW, all = of_q + (A.heads[1] + HPW - 1) / HPW;
  const int g0 = part * A.turns, g1 = g0 + A.turns < all ? g0 + A.turns : all;
  vec a, b;  // those of the next group
  auto load = [&](int gi) {
    const int key = gi >= of_q, h = (key ? gi - of_q : gi) * HPW + lane / LG;
    const T* in = static_cast<const T*>(A.in[key]) + (size_t)r * A.ld_in[key] + (size_t)h * A.D;
    const bool on = h < A.heads[key];
    a = b = vec{};
    if (on && on0) a = *reinterpret_cast<const vec*>(in + v0 * E);
    if (on && on1) b = *reinterpret_cast<const vec*>(in + v1 * E);
  };
  load(g0);
  // pair e of the lane: elements e of both vectors (halves), 2 e and 2 e + 1 (pairs)
  float c[N] = {}, s[N] = {};
  uint32_t turned = 0u;
  if (A.rot) {
    const double pos = (double)A.pos[r];
    const int half = A.rot / 2;
#pragma unroll
    for (int e = 0; e < N; e++) {
      const int i = j * N + e, pair = FORM == ROPE_ODD && i >= half ? i - half : i;
      if (pair < half) {
        rope_turn(pos * ((double)A.freq[pair] * ROPE_QUARTERS), c[e], s[e]);
        c[e] *= A.amplitude;
        s[e] *= FORM == ROPE_ODD && i < half ? -A.amplitude : A.amplitude;
        turned |= 1u << e;
      }
    }
  }
  const bool whole = A.rot == A.D;  // (then nothing is left as it is)
  int has = -1;                     // whose norm weights are in wx, wy
  float wx[E], wy[E];
  for (int gi = g0; gi < g1; gi++) {
    const int key = gi >= of_q, h = (key ? gi - of_q : gi) * HPW + lane / LG;
    T* out = static_cast<T*>(A.out[key]) + (size_t)r * A.ld_out[key] + (size_t)h * A.D;
    const float* w = A.norm[key];
    if (w && has != key) {
      has = key;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        pz_f4u p = {}, q = {};
        if (on0) p = *reinterpret_cast<const pz_f4u*>(w + v0 * E + e);
        if (on1) q = *reinterpret_cast<const pz_f4u*>(w + v1 * E + e);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          wx[e + i] = p[i];
          wy[e + i] = q[i];
        }
      }
    }
    float x[E], y[E];
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      x[e] = Y::widen(a[e]);
      y[e] = Y::widen(b[e]);
    }
    if (gi + 1 < g1) load(gi + 1);
    if (w) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        sum = __builtin_fmaf(x[e], x[e], sum);
        sum = __builtin_fmaf(y[e], y[e], sum);
      }
#pragma unroll
      for (int o = 1; o < LG; o <<= 1) sum += __shfl_xor(sum, o, 64);
      const float f = rope_rsqrt(__builtin_fmaf(sum, A.per_D, A.eps));
#pragma unroll
      for (int e = 0; e < E; e++) {
        x[e] = x[e] * f * wx[e];
        y[e] = y[e] * f * wy[e];
      }
    }
    if constexpr (FORM == ROPE_ODD) {
      // (a wave's own LDS; the lanes' elements one place apart, so that what the lanes read
      // and write together lies in different banks: 40 us without)
      float* const all_of = heads[threadIdx.x >> 6] + lane / LG * (LG * (2 * E + 1));
      auto place = [](int i) { return (unsigned)i + (unsigned)i / (2 * E); };
#pragma unroll
      for (int e = 0; e < E; e++) {
        all_of[j * (2 * E + 1) + e] = x[e];
        all_of[j * (2 * E + 1) + E + e] = y[e];
      }
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < N; e++) {
        const int i = j * N + e, half = A.rot / 2;
        float& p = e < E ? x[e] : y[e - E];
        if (turned >> e & 1u)
          p = __builtin_fmaf(p, c[e], all_of[place(i < half ? i + half : i - half)] * s[e]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      __builtin_amdgcn_wave_barrier();
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) {
        float& p = FORM == ROPE_HALVES ? x[e] : (e < E / 2 ? x[2 * e] : y[2 * e - E]);
        float& q = FORM == ROPE_HALVES ? y[e] : (e < E / 2 ? x[2 * e + 1] : y[2 * e + 1 - E]);
        const float pt = __builtin_fmaf(p, c[e], -(q * s[e])),
                    qt = __builtin_fmaf(q, c[e], p * s[e]);
        const bool on = whole || (turned >> e & 1u);
        p = on ? pt : p;
        q = on ? qt : q;
      }
    }
    vec ra, rb;
#pragma unroll
    for (int e = 0; e < E; e++) {
      ra[e] = Y::narrow(x[e]);
      rb[e] = Y::narrow(y[e]);
    }
    const bool on = h < A.heads[key];
    if (on && on0) *reinterpret_cast<vec*>(out + v0 * E) = ra;
    if (on && on1) *reinterpret_cast<vec*>(out + v1 * E) = rb;
  }
}

template <int TYPE>
__global__ __launch_bounds__(64) void k_qk_rope_any(const RopeArgs A, int layout) {
  typedef RopeType<TYPE> Y;
  typedef typename Y::T T;
  const int lane = threadIdx.x, total = A.heads[0] + A.heads[1];
  const int r = (int)(blockIdx.x / (unsigned)total), at = (int)(blockIdx.x - (unsigned)r * total);
  const bool key = at >= A.heads[0];
  const int h = key ? at - A.heads[0] : at;
  const T* in = static_cast<const T*>(A.in[key]) + (size_t)r * A.ld_in[key] + (size_t)h * A.D;
  T* out = static_cast<T*>(A.out[key]) + (size_t)r * A.ld_out[key] + (size_t)h * A.D;
  const float* w = A.norm[key];
  float f = 1.0f;
  if (w) {
    float sum = 0.0f;
    for (int d = lane; d < A.D; d += 64) {
      const float v = Y::widen(in[d]);
      sum = __builtin_fmaf(v, v, sum);
    }
    // (every lane's loads are done before any lane's stores: in place is fine)
    f = rope_rsqrt(__builtin_fmaf(pz_wave_sum(sum), A.per_D, A.eps));
  }
  auto load = [&](int d) {
    const float v = Y::widen(in[d]);
    return w ? v * f * w[d] : v;
  };
  const double pos = A.rot ? (double)A.pos[r] : 0.0;
  const int half = A.rot / 2;
  for (int i = lane; i < half; i += 64) {
    const int p = layout == PZ_ROPE_HALVES ? i : 2 * i,
              q = layout == PZ_ROPE_HALVES ? i + half : 2 * i + 1;
    float c, s;
    rope_turn(pos * ((double)A.freq[i] * ROPE_QUARTERS), c, s);
    c *= A.amplitude;
    s *= A.amplitude;
    const float x = load(p), y = load(q);
    out[p] = Y::narrow(__builtin_fmaf(x, c, -(y * s)));
    out[q] = Y::narrow(__builtin_fmaf(y, c, x * s));
  }
  for (int d = A.rot + lane; d < A.D; d += 64) out[d] = Y::narrow(load(d));
}

template <int TYPE, RopeForm FORM, int LG>
int launch(pz_sampler* s, RopeArgs& A) {
  constexpr int HPW = 64 / LG;
  const int groups = (A.heads[0] + HPW - 1) / HPW + (A.heads[1] + HPW - 1) / HPW;
  // 16 waves a CU, and then more heads for each (2000 tokens of 32 + 8 heads 11.3 us, with
  // 32 waves 12.4, with 64 14.6)
  const int64_t room = (int64_t)s->n_cu * 16, all = (int64_t)A.n * groups;
  const int64_t turns = (all + room - 1) / room;
  A.turns = (int)(turns < groups ? turns : groups);
  A.waves = (groups + A.turns - 1) / A.turns;
  const int64_t wgs = ((int64_t)A.n * A.waves + 3) / 4;
  hipLaunchKernelGGL((k_qk_rope<TYPE, FORM, LG>), dim3((unsigned)wgs), dim3(256), 0, s->stream, A);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}

template <int TYPE, RopeForm FORM>
int lanes(pz_sampler* s, RopeArgs& A) {
  const int want = (A.D / RopeType<TYPE>::E + 1) / 2;
  if (want <= 4) return launch<TYPE, FORM, 4>(s, A);
  if (want <= 8) return launch<TYPE, FORM, 8>(s, A);
  if (want <= 16) return launch<TYPE, FORM, 16>(s, A);
  if (want <= 32) return launch<TYPE, FORM, 32>(s, A);
  return launch<TYPE, FORM, 64>(s, A);
}

template <int TYPE>
int run(pz_sampler* s, RopeArgs& A, int layout) {
  constexpr int E = RopeType<TYPE>::E;
  bool quick = A.D % E == 0 && A.D / E <= 128 && pz_rope_in_fours(A.n, A.heads[0] + A.heads[1]);
  for (int i = 0; i < 2; i++)
    quick = quick && (!A.heads[i] || (pz_aligned16(A.in[i]) && pz_aligned16(A.out[i]) &&
                                      A.ld_in[i] % E == 0 && A.ld_out[i] % E == 0));
  if (quick && layout == PZ_ROPE_PAIRS) return lanes<TYPE, ROPE_PAIRS>(s, A);
  if (quick && A.rot / 2 % E == 0) return lanes<TYPE, ROPE_HALVES>(s, A);
  if (quick) return lanes<TYPE, ROPE_ODD>(s, A);
  hipLaunchKernelGGL((k_qk_rope_any<TYPE>), dim3((unsigned)A.n * (A.heads[0] + A.heads[1])),
                     dim3(64), 0, s->stream, A, layout);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}

}  // namespace

extern "C" int pz_qk_norm_rope(pz_sampler* s, const pz_qk_rope* rope, const void* d_q, long ld_q,
                               const void* d_k, long ld_k, void* d_q_out, long ld_q_out,
                               void* d_k_out, long ld_k_out, int n, const int32_t* d_pos) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no =
      pz_refuse_rope(rope, d_q, ld_q, d_k, ld_k, d_q_out, ld_q_out, d_k_out, ld_k_out, n, d_pos);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (n == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  RopeArgs A = {{d_q, d_k},
                {d_q_out, d_k_out},
                {ld_q, ld_k},
                {ld_q_out, ld_k_out},
                {rope->d_q_norm, rope->d_k_norm},
                {rope->n_heads, rope->n_kv_heads},
                rope->head_dim,
                rope->rot_dim,
                rope->d_freq,
                d_pos,
                1.0f / (float)rope->head_dim,
                rope->eps,
                rope->amplitude,
                n,
                1,
                1};
  if (rope->type == PZ_F32) return run<PZ_F32>(s, A, rope->layout);
  if (rope->type == PZ_BF16) return run<PZ_BF16>(s, A, rope->layout);
  return run<PZ_F16>(s, A, rope->layout);
}
