// pz_lmhead_i8.hip -- the LM head in 8-bit integers (pz_lm_head_i8,
// pz_lm_head_argmax_i8) and the quantisation of its operands
// (pz_quant_rows_i8).
//
//   scale = max|x| / 127, q = rne(x / scale)                       (rows)
//   logits[b, i] = (fl32(sum_j w[i, j] q[b, j]) * sw[i]) * sx[b]   (product)
//
// The sum is exact in int32 (16384 n < 2^31), so the order in which k is added
// up is free and every tile shape gives the same logits.
#include <hip/hip_runtime.h>

#include "../../include/pz_sampler.h"
#include "pz_device.h"
#include "pz_lmdev.h"
#include "pz_lmtile.h"
#include "pz_refuse.h"
#include "pz_sampler_impl.h"

namespace {

// ---- quantisation --------------------------------------------------------------
// One workgroup per row: the row's |x| maximum over the bit patterns (an
// infinity or NaN has the largest), then x / scale, correctly rounded.  Rows of
// up to 4 QB NV elements stay in registers between the two; longer ones are
// read again (from the caches).
constexpr int QB = 256;
typedef uint16_t q_u16x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t q_u32u __attribute__((aligned(1)));

template <int TYPE>
__device__ __forceinline__ float q_widen(uint16_t h) {
  return TYPE == PZ_BF16 ? __uint_as_float((uint32_t)h << 16)
                         : (float)__builtin_bit_cast(_Float16, h);
}

// x[j .. j + 3] of a row (zeros past n).
template <int TYPE>
__device__ __forceinline__ void q_load4(const void* row, int j, int n, float (&v)[4]) {
  if (j + 3 < n) {
    if (TYPE == PZ_F32) {
      const pz_f4u q = *reinterpret_cast<const pz_f4u*>(static_cast<const float*>(row) + j);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = q[e];
    } else {
      const q_u16x4 q =
          *reinterpret_cast<const q_u16x4*>(static_cast<const uint16_t*>(row) + j);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = q_widen<TYPE>(q[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      v[e] = 0.0f;
      if (j + e < n)
        v[e] = TYPE == PZ_F32 ? static_cast<const float*>(row)[j + e]
                              : q_widen<TYPE>(static_cast<const uint16_t*>(row)[j + e]);
    }
  }
}

template <int TYPE, int NV>
__global__ __launch_bounds__(QB) void k_quant(const void* __restrict__ X, long ldx, int n,
                                              int8_t* __restrict__ Q, long ldq,
                                              float* __restrict__ scale) {
  __shared__ uint32_t part[QB / 64];
  const int tid = threadIdx.x;
  const size_t row = blockIdx.x;
  const void* x = static_cast<const char*>(X) + row * ldx * (TYPE == PZ_F32 ? 4 : 2);
  int8_t* q = Q + row * ldq;
  float v[NV ? NV : 1][4];
  uint32_t top = 0u;
  auto most = [&](const float(&y)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t a = __float_as_uint(y[e]) & 0x7fffffffu;
      top = a > top ? a : top;
    }
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; i++) q_load4<TYPE>(x, 4 * (i * QB + tid), n, v[i]);
#pragma unroll
    for (int i = 0; i < NV; i++) most(v[i]);
  } else {
    for (int j = 4 * tid; j < n; j += 4 * QB) {
      q_load4<TYPE>(x, j, n, v[0]);
      most(v[0]);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t o = __shfl_xor(top, off, 64);
    top = o > top ? o : top;
  }
  if ((tid & 63) == 0) part[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < QB / 64; i++) top = part[i] > top ? part[i] : top;
  const bool fin = top < 0x7f800000u;
  const float sc = fin ? __uint_as_float(top) / 127.0f : __builtin_nanf("");
  if (tid == 0) scale[row] = sc;
  const bool zero = !fin || sc == 0.0f;
  auto put = [&](int j, const float(&y)[4]) {
    uint32_t w = 0u;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      // (the clamp: a scale rounded down among the subnormals)
      const float r = zero ? 0.0f : fminf(fmaxf(rintf(y[e] / sc), -127.0f), 127.0f);
      w |= ((uint32_t)(int)r & 0xffu) << (8 * e);
    }
    if (j + 3 < n) {
      *reinterpret_cast<q_u32u*>(q + j) = w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (j + e < n) q[j + e] = (int8_t)(w >> (8 * e));
    }
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; i++) put(4 * (i * QB + tid), v[i]);
  } else {
    for (int j = 4 * tid; j < n; j += 4 * QB) {
      q_load4<TYPE>(x, j, n, v[0]);
      put(j, v[0]);
    }
  }
}

template <int TYPE>
int quant(pz_sampler* s, const void* d_x, long ldx, int rows, int n, int8_t* d_q, long ldq,
          float* d_scale) {
  auto k = n <= 4 * QB       ? k_quant<TYPE, 1>
           : n <= 4 * QB * 2 ? k_quant<TYPE, 2>
           : n <= 4 * QB * 4 ? k_quant<TYPE, 4>
           : n <= 4 * QB * 8 ? k_quant<TYPE, 8>
                             : k_quant<TYPE, 0>;
  hipLaunchKernelGGL(k, dim3(rows), dim3(QB), 0, s->stream, d_x, ldx, n, d_q, ldq, d_scale);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}

// ---- product -------------------------------------------------------------------
// v_mfma_i32_16x16x64_i8: A = 16 rows of W x 64 k, B = 64 k x 16 batch rows, D =
// 16 rows x 16 batch rows (lane l: batch row l % 16, rows 4 (l / 16) .. +3); of
// A and B lane l holds row l % 16 and the 16 bytes of k from 16 (l / 16) on.
//
//   * A workgroup owns WR TR x 16 rows of W and WC TC x 16 batch rows; wave
//     (wr, wc) TR x TC tiles of it.  k advances 128 at a time -- whole cache
//     lines of W -- through a ring of NS stages in LDS: one load instruction
//     brings 8 rows x 128 bytes, straight to LDS, NS - 1 stages ahead, one
//     barrier per stage.  The 16-byte pieces of a row are rotated by XOR with
//     the row so that the fragment reads do not meet in the banks.
//   * !FAST: rows off 16 bytes (n or ldx not a multiple of 16) go through
//     registers, the pieces that cross a row's end byte by byte.
typedef int i8_i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t i8_u32x4u __attribute__((ext_vector_type(4), aligned(1)));

// 16 bytes at p, of which the first `valid` belong to the row (zeros past
// them).
__device__ __forceinline__ lm_u32x4 i8_load16(const int8_t* p, int valid) {
  lm_u32x4 q = {0u, 0u, 0u, 0u};
  if (valid >= 16) {
    q = *reinterpret_cast<const i8_u32x4u*>(p);
  } else {
#pragma unroll
    for (int e = 0; e < 16; e++)
      if (e < valid) q[e >> 2] |= (uint32_t)(uint8_t)p[e] << (8 * (e & 3));
  }
  return q;
}

template <int WR, int WC, int TR, int TC, int NS, int MODE, bool FAST, bool NT>
__global__ __launch_bounds__(64 * WR * WC) void k_lmhead_i8(
    const int8_t* __restrict__ W, const float* __restrict__ sw, int V, int n,
    const int8_t* __restrict__ X, const float* __restrict__ sx, long ldx, int nb, int ncb, int nrt,
    float* __restrict__ logits, long ld, unsigned long long* __restrict__ keys, int kstride,
    uint8_t* __restrict__ nan0) {
  constexpr int NW = WR * WC;
  constexpr int RF = WR * TR, CF = WC * TC;
  constexpr int WI = RF * 2, XI = CF * 2;  // 1 KiB loads of a stage
  constexpr int WPW = WI / NW, XPW = (XI + NW - 1) / NW, PER = WPW + XPW;
  constexpr int STG = (WI + XI) * 1024;
  static_assert(WI % NW == 0 && NS >= 2, "");
  static_assert(NS * STG >= NW * CF * 16 * 8, "the epilogue's keys reuse the ring");
  __shared__ __align__(16) int8_t sh[NS * STG];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int wr = w % WR, wc = w / WR;
  // the batch blocks of a row tile on one XCD, one after the other
  const int slot = blockIdx.x >> 3;
  const int rt = (slot / ncb) * 8 + (blockIdx.x & 7), cb = slot % ncb;
  if (rt >= nrt) return;
  const int row0 = rt * RF * 16, b0 = cb * CF * 16;
  i8_i32x4 acc[TR][TC];
#pragma unroll
  for (int t = 0; t < TR; t++)
#pragma unroll
    for (int j = 0; j < TC; j++) acc[t][j] = i8_i32x4{0, 0, 0, 0};
  const int nst = (n + 127) >> 7;
  const int lrow = lane >> 3, piece = (lane & 7) ^ lrow;  // of this lane's loads
  // rows past V and batch rows past nb: the last one (results unused)
  auto wrow = [&](int i) {
    const int r = (w * WPW + i) * 8 + lrow, last = V - 1 - row0;
    return r < last ? r : last;
  };
  auto xload_of = [&](int i) {
    const int q = w * XPW + i;
    return XI % NW && q >= XI ? XI - 1 : q;  // (the same bytes to the same place again)
  };
  auto xrow = [&](int i) {
    const int r = xload_of(i) * 8 + lrow, last = nb - 1 - b0;
    return r < last ? r : last;
  };
  const int8_t* wbase = W + (size_t)row0 * n;
  const int8_t* xbase = X + (size_t)b0 * ldx;
  auto mma = [&](const int8_t* st, int c) {
    // (FAST: pieces past n hold the row's last piece again: zeros in B)
    const bool tail = FAST && c == nst - 1 && (n & 127);
#pragma unroll
    for (int s = 0; s < 2; s++) {
      i8_i32x4 a[TR], b[TC];
      const int at = ((s * 4 + g) ^ (m & 7)) * 16;
#pragma unroll
      for (int j = 0; j < TC; j++)
        b[j] = *reinterpret_cast<const i8_i32x4*>(st + WI * 1024 + ((wc * TC + j) * 16 + m) * 128 +
                                                  at);
      if (tail)
#pragma unroll
        for (int j = 0; j < TC; j++)
          if (c * 128 + s * 64 + 16 * g >= n) b[j] = i8_i32x4{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < TR; t++)
        a[t] = *reinterpret_cast<const i8_i32x4*>(st + ((wr * TR + t) * 16 + m) * 128 + at);
#pragma unroll
      for (int j = 0; j < TC; j++)
#pragma unroll
        for (int t = 0; t < TR; t++)
          acc[t][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[t], b[j], acc[t][j], 0, 0, 0);
    }
  };
  if constexpr (FAST) {
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)sh;
    uint32_t woff[WPW], xoff[XPW];
#pragma unroll
    for (int i = 0; i < WPW; i++) woff[i] = (uint32_t)wrow(i) * (uint32_t)n + 16u * piece;
#pragma unroll
    for (int i = 0; i < XPW; i++) xoff[i] = (uint32_t)xrow(i) * (uint32_t)ldx + 16u * piece;
    const int klast = (nst - 1) * 128 + 16 * piece;
    const uint32_t adj = klast < n ? 0u : (uint32_t)(klast - (n - 16));
    auto issue = [&](int c, int buf) {
      const uint32_t l0 = lds0 + (uint32_t)buf * STG;
      const uint32_t back = c == nst - 1 ? adj : 0u;
#pragma unroll
      for (int i = 0; i < WPW; i++)
        lm_lds_load16<NT>(wbase + (size_t)c * 128, woff[i] - back, l0 + (w * WPW + i) * 1024);
#pragma unroll
      for (int i = 0; i < XPW; i++)
        lm_lds_load16<false>(xbase + (size_t)c * 128, xoff[i] - back,
                             l0 + (WI + xload_of(i)) * 1024);
    };
#pragma unroll
    for (int i = 0; i < NS - 1; i++) issue(i < nst ? i : nst - 1, i);
    int buf = 0, nbuf = NS - 1;
#pragma clang loop unroll(disable)
    for (int c = 0; c < nst; c++) {
      // stage c has arrived (the NS - 2 after it may be on their way), in every
      // wave; and every wave is done reading the slot that is filled next
      lm_wait<(NS - 2) * PER>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      issue(c + NS - 1 < nst ? c + NS - 1 : nst - 1, nbuf);  // (past the end: reloaded, unused)
      mma(sh + buf * STG, c);
      asm volatile("" ::: "memory");
      buf = buf + 1 == NS ? 0 : buf + 1;
      nbuf = nbuf + 1 == NS ? 0 : nbuf + 1;
    }
    lm_wait<0>();
  } else {
    lm_u32x4 q[PER];
    auto fetch = [&](int c) {
      const int k = c * 128 + 16 * piece;
#pragma unroll
      for (int i = 0; i < WPW; i++) q[i] = i8_load16(wbase + (size_t)wrow(i) * n + k, n - k);
#pragma unroll
      for (int i = 0; i < XPW; i++) q[WPW + i] = i8_load16(xbase + (size_t)xrow(i) * ldx + k, n - k);
    };
    fetch(0);
#pragma clang loop unroll(disable)
    for (int c = 0; c < nst; c++) {
      int8_t* st = sh + (c & 1) * STG;
#pragma unroll
      for (int i = 0; i < WPW; i++)
        *reinterpret_cast<lm_u32x4*>(st + (w * WPW + i) * 1024 + lane * 16) = q[i];
#pragma unroll
      for (int i = 0; i < XPW; i++)
        *reinterpret_cast<lm_u32x4*>(st + (WI + xload_of(i)) * 1024 + lane * 16) = q[WPW + i];
      __syncthreads();
      if (c + 1 < nst) fetch(c + 1);
      mma(st, c);
      // (the slot written next was last read before this stage's barrier)
    }
  }
  // epilogue: lane l holds batch row l % 16 of each tile, rows 4 (l / 16) + i
  float fx[TC];
#pragma unroll
  for (int j = 0; j < TC; j++) {
    const int b = b0 + (wc * TC + j) * 16 + m;
    fx[j] = b < nb ? sx[b] : 0.0f;
  }
  unsigned long long best[TC];
#pragma unroll
  for (int j = 0; j < TC; j++) best[j] = 0ull;
  const bool vec = MODE == 0 && (ld & 3) == 0 && ((uintptr_t)logits & 15) == 0;
#pragma unroll
  for (int t = 0; t < TR; t++) {
    const int row = row0 + (wr * TR + t) * 16 + 4 * g;
    float fw[4];
#pragma unroll
    for (int i = 0; i < 4; i++) fw[i] = row + i < V ? sw[row + i] : 0.0f;
#pragma unroll
    for (int j = 0; j < TC; j++) {
      const int b = b0 + (wc * TC + j) * 16 + m;
      if (b >= nb) continue;
      lm_f32x4 y;
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = ((float)acc[t][j][i] * fw[i]) * fx[j];
      if (MODE == 0) {
        float* o = logits + (size_t)b * ld + row;
        if (vec && row + 3 < V) {
          *reinterpret_cast<lm_f32x4*>(o) = y;
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (row + i < V) o[i] = y[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (row + i < V) {
            if (row + i == 0) nan0[b] = y[i] != y[i] ? 1 : 0;
            if (!(y[i] != y[i])) {
              const unsigned long long kk = argmax_key(y[i], row + i);
              best[j] = kk > best[j] ? kk : best[j];
            }
          }
      }
    }
  }
  if (MODE == 1) {
    __syncthreads();  // the ring is free
    unsigned long long* best_sh = reinterpret_cast<unsigned long long*>(sh);  // [WR][CF * 16]
#pragma unroll
    for (int j = 0; j < TC; j++) {
      // the maximum over the four lane groups, then over the row waves
#pragma unroll
      for (int off = 16; off < 64; off <<= 1) {
        const unsigned long long o = __shfl_xor(best[j], off, 64);
        best[j] = o > best[j] ? o : best[j];
      }
      if (g == 0) best_sh[wr * CF * 16 + (wc * TC + j) * 16 + m] = best[j];
    }
    __syncthreads();
    for (int bl = tid; bl < CF * 16; bl += 64 * NW) {
      const int b = b0 + bl;
      if (b >= nb) break;
      unsigned long long mx = best_sh[bl];
#pragma unroll
      for (int i = 1; i < WR; i++) {
        const unsigned long long o = best_sh[i * CF * 16 + bl];
        mx = o > mx ? o : mx;
      }
      if (mx) atomicMax(&keys[(size_t)(blockIdx.x % LMM_SLOTS) * kstride + b], mx);
    }
  }
}

struct I8Call {
  const int8_t* w;
  const float* sw;
  int V, n;
  const int8_t* x;
  const float* sx;
  long ldx;
  int B;
  float* out;
  long ld;
};

template <int WR, int WC, int TR, int TC, int NS, int MODE, bool FAST>
int launch(pz_sampler* s, const I8Call& c) {
  constexpr int rows = WR * TR * 16, cols = WC * TC * 16;
  const int ncb = (c.B + cols - 1) / cols, nrt = (c.V + rows - 1) / rows;
  const unsigned grid = (unsigned)((nrt + 7) / 8 * 8) * ncb;
  // weights past the Infinity Cache are not kept (lm_once counts bf16 weights)
  auto k = FAST && lm_once(c.V, (c.n + 1) / 2)
               ? k_lmhead_i8<WR, WC, TR, TC, NS, MODE, FAST, FAST>
               : k_lmhead_i8<WR, WC, TR, TC, NS, MODE, FAST, false>;
  hipLaunchKernelGGL(k, dim3(grid), dim3(64 * WR * WC), 0, s->stream, c.w, c.sw, c.V, c.n, c.x,
                     c.sx, c.ldx, c.B, ncb, nrt, c.out, c.ld, s->d_lmh_keys, s->max_batch,
                     s->d_lmh_nan);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}

template <int MODE>
int run(pz_sampler* s, const I8Call& c) {
  const bool fast = c.n % 16 == 0 && c.ldx % 16 == 0 && pz_aligned16(c.w) && pz_aligned16(c.x) &&
                    (int64_t)c.ldx * 256 <= UINT32_MAX;
  if (!fast) {
    if (c.B <= 16) return launch<4, 1, 1, 1, 2, MODE, false>(s, c);
    return launch<4, 1, 1, 4, 2, MODE, false>(s, c);
  }
  if (c.B <= 16) return launch<8, 1, 2, 1, 4, MODE, true>(s, c);
  if (c.B <= 32) return launch<8, 1, 2, 2, 4, MODE, true>(s, c);
  if (c.B <= 64) return launch<4, 2, 4, 2, 3, MODE, true>(s, c);
  if (c.B <= 128) return launch<4, 2, 4, 4, 3, MODE, true>(s, c);
  return launch<2, 4, 8, 4, 2, MODE, true>(s, c);
}

}  // namespace

extern "C" int pz_quant_rows_i8(pz_sampler* s, const void* d_x, int x_type, long ldx, int rows,
                                int n, int8_t* d_q, long ldq, float* d_scale) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no = pz_refuse_quant(d_x, x_type, ldx, rows, n, d_q, ldq, d_scale);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (rows == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  if (x_type == PZ_F32) return quant<PZ_F32>(s, d_x, ldx, rows, n, d_q, ldq, d_scale);
  if (x_type == PZ_BF16) return quant<PZ_BF16>(s, d_x, ldx, rows, n, d_q, ldq, d_scale);
  return quant<PZ_F16>(s, d_x, ldx, rows, n, d_q, ldq, d_scale);
}

extern "C" int pz_lm_head_i8(pz_sampler* s, const int8_t* d_w, const float* d_sw, int V, int n,
                             const int8_t* d_x, const float* d_sx, int B, long ldx,
                             float* d_logits, long ld) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no = pz_refuse_i8(d_w, d_sw, V, n, d_x, d_sx, B, ldx, s->max_batch);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (!d_logits || ld < V) return fail(s, PZ_EINVAL, "bad logits buffer");
  if (B == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  return run<0>(s, {d_w, d_sw, V, n, d_x, d_sx, ldx, B, d_logits, ld});
}

extern "C" int pz_lm_head_argmax_i8(pz_sampler* s, const int8_t* d_w, const float* d_sw, int V,
                                    int n, const int8_t* d_x, const float* d_sx, int B, long ldx,
                                    int32_t* d_ids) {
  if (!s) return PZ_EINVAL;
  const PzRefusal no = pz_refuse_i8(d_w, d_sw, V, n, d_x, d_sx, B, ldx, s->max_batch);
  if (no.code) return fail(s, no.code, "%s", no.why);
  if (!d_ids) return fail(s, PZ_EINVAL, "null ids");
  if (B == 0) return PZ_OK;
  PZ_HIP(s, hipSetDevice(s->device));
  const int rc = run<1>(s, {d_w, d_sw, V, n, d_x, d_sx, ldx, B, nullptr, 0});
  return rc != PZ_OK ? rc : pz_lm_finish(s, B, d_ids);
}
