// pz_rope.hip -- RMS norm of each head of queries and keys and its rotation to the
// token's position (pz_qk_norm_rope).
//
//   y = x w / sqrt(mean(x^2) + eps);  (a, b) -> (a cos - b sin, b cos + a sin) amplitude
//
// The angle pos * freq is wanted modulo a turn, to fp32's precision, for positions of
// any size: in 64 bits, in quarter turns, t = pos * (freq 2 / pi), whose distance to
// the nearest whole number (at most a half: at most pi / 4) is left for fp32, where
// the series of sine and cosine stop after x^9 and x^10 (terms of 2e-9 and 1e-10 are
// left out at pi / 4).
//
// k_qk_rope: a head is LG lanes, each of which owns two 16-byte vectors: of the same
// place in the two halves (PZ_ROPE_HALVES; past the rotated part, the next two), or
// neighbours (PZ_ROPE_PAIRS), so that both elements of a pair are in one lane.  A wave
// takes 64 / LG heads at once and `turns` times that many of one token, whose angles it
// makes once.  k_qk_rope_any: one element pair a lane, a wave a head, whatever the sizes,
// strides and alignment.
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
  float eps, amplitude;
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

// cos and sin of the angle of t quarter turns.
__device__ __forceinline__ void rope_turn(double t, float& c, float& s) {
  const double q = rint(t);
  const float x = (float)(t - q) * 1.57079632679489661923f, z = x * x;
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
  // the quarter: its last two bits (|t| < 2^53, so that they are there)
  const int k = (int)((long long)q & 3);
  const float a = k & 1 ? sn : cs, b = k & 1 ? cs : sn;
  c = k == 1 || k == 2 ? -a : a;
  s = k & 2 ? -b : b;
}
constexpr double ROPE_QUARTERS = 0.63661977236758134308;  // 2 / pi

template <int TYPE, int LAYOUT, int LG>
__global__ __launch_bounds__(256) void k_qk_rope(const RopeArgs A) {
  typedef RopeType<TYPE> Y;
  typedef typename Y::T T;
  constexpr int E = Y::E, HPW = 64 / LG;
  typedef T vec __attribute__((ext_vector_type(E)));
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = (int)(wave / A.waves), part = (int)(wave - (int64_t)r * A.waves);
  if (r >= A.n) return;
  const int j = lane % LG, nv = A.D / E, rv = A.rot / 2 / E;
  int v0 = 2 * j, v1 = 2 * j + 1;
  if (LAYOUT == PZ_ROPE_HALVES && j < rv) {
    v0 = j;
    v1 = rv + j;
  }
  const bool on0 = v0 < nv, on1 = v1 < nv;
  // pair e of the lane: elements e of both vectors (halves), 2 e and 2 e + 1 (pairs)
  float c[E] = {}, s[E] = {};
  uint32_t turned = 0u;
  if (A.rot) {
    const double pos = (double)A.pos[r];
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int i = j * E + e;
      if (i < A.rot / 2) {
        rope_turn(pos * ((double)A.freq[i] * ROPE_QUARTERS), c[e], s[e]);
        c[e] *= A.amplitude;
        s[e] *= A.amplitude;
        turned |= 1u << e;
      }
    }
  }
  const int total = A.heads[0] + A.heads[1];
  for (int i = 0; i < A.turns; i++) {
    const int at = (part * A.turns + i) * HPW + lane / LG;
    const bool key = at >= A.heads[0], there = at < total;
    const int h = key ? at - A.heads[0] : at;
    const T* in = static_cast<const T*>(A.in[key]) + (size_t)r * A.ld_in[key] + (size_t)h * A.D;
    T* out = static_cast<T*>(A.out[key]) + (size_t)r * A.ld_out[key] + (size_t)h * A.D;
    vec a = {}, b = {};
    if (there && on0) a = *reinterpret_cast<const vec*>(in + v0 * E);
    if (there && on1) b = *reinterpret_cast<const vec*>(in + v1 * E);
    float x[E], y[E];
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      x[e] = Y::widen(a[e]);
      y[e] = Y::widen(b[e]);
      sum = __builtin_fmaf(x[e], x[e], sum);
      sum = __builtin_fmaf(y[e], y[e], sum);
    }
    if (A.norm[0] || A.norm[1]) {
#pragma unroll
      for (int o = 1; o < LG; o <<= 1) sum += __shfl_xor(sum, o, 64);
      const float* w = A.norm[key];
      if (w) {
        const float f = 1.0f / sqrtf(sum / (float)A.D + A.eps);
#pragma unroll
        for (int e = 0; e < E; e++) {
          x[e] = x[e] * f * (on0 ? w[v0 * E + e] : 0.0f);
          y[e] = y[e] * f * (on1 ? w[v1 * E + e] : 0.0f);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
      float& p = LAYOUT == PZ_ROPE_HALVES ? x[e] : (e < E / 2 ? x[2 * e] : y[2 * e - E]);
      float& q = LAYOUT == PZ_ROPE_HALVES ? y[e] : (e < E / 2 ? x[2 * e + 1] : y[2 * e + 1 - E]);
      const float pt = __builtin_fmaf(p, c[e], -(q * s[e])), qt = __builtin_fmaf(q, c[e], p * s[e]);
      const bool on = turned >> e & 1u;
      p = on ? pt : p;
      q = on ? qt : q;
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
      a[e] = Y::narrow(x[e]);
      b[e] = Y::narrow(y[e]);
    }
    if (there && on0) *reinterpret_cast<vec*>(out + v0 * E) = a;
    if (there && on1) *reinterpret_cast<vec*>(out + v1 * E) = b;
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
    f = 1.0f / sqrtf(pz_wave_sum(sum) / (float)A.D + A.eps);
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

template <int TYPE, int LAYOUT, int LG>
int launch(pz_sampler* s, RopeArgs& A) {
  constexpr int HPW = 64 / LG;
  const int groups = (A.heads[0] + A.heads[1] + HPW - 1) / HPW;
  // as many waves as the device holds at once, and then more heads for each
  const int64_t room = (int64_t)s->n_cu * 32, all = (int64_t)A.n * groups;
  const int64_t turns = (all + room - 1) / room;
  A.turns = (int)(turns < groups ? turns : groups);
  A.waves = (groups + A.turns - 1) / A.turns;
  const int64_t wgs = ((int64_t)A.n * A.waves + 3) / 4;
  hipLaunchKernelGGL((k_qk_rope<TYPE, LAYOUT, LG>), dim3((unsigned)wgs), dim3(256), 0, s->stream,
                     A);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}

template <int TYPE, int LAYOUT>
int lanes(pz_sampler* s, RopeArgs& A) {
  const int want = (A.D / RopeType<TYPE>::E + 1) / 2;
  if (want <= 4) return launch<TYPE, LAYOUT, 4>(s, A);
  if (want <= 8) return launch<TYPE, LAYOUT, 8>(s, A);
  if (want <= 16) return launch<TYPE, LAYOUT, 16>(s, A);
  if (want <= 32) return launch<TYPE, LAYOUT, 32>(s, A);
  return launch<TYPE, LAYOUT, 64>(s, A);
}

template <int TYPE>
int run(pz_sampler* s, RopeArgs& A, int layout) {
  constexpr int E = RopeType<TYPE>::E;
  bool quick = A.D % E == 0 && A.D / E <= 128 && (layout == PZ_ROPE_PAIRS || A.rot / 2 % E == 0);
  for (int i = 0; i < 2; i++)
    quick = quick && (!A.heads[i] || (pz_aligned16(A.in[i]) && pz_aligned16(A.out[i]) &&
                                      A.ld_in[i] % E == 0 && A.ld_out[i] % E == 0));
  if (quick)
    return layout == PZ_ROPE_HALVES ? lanes<TYPE, PZ_ROPE_HALVES>(s, A)
                                    : lanes<TYPE, PZ_ROPE_PAIRS>(s, A);
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
                rope->eps,
                rope->amplitude,
                n,
                1,
                1};
  if (rope->type == PZ_F32) return run<PZ_F32>(s, A, rope->layout);
  if (rope->type == PZ_BF16) return run<PZ_BF16>(s, A, rope->layout);
  return run<PZ_F16>(s, A, rope->layout);
}
