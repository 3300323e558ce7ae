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
// up to 16384 elements stay in registers between the two; longer ones are
// read again (from the caches).
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

template <int TYPE, int NV, int QB>
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
  // (long rows: more threads; 1 row of 20000 13.1 -> 5.8 us, 1024 29.2 -> 25.8; but
  // 8192 rows of 2560 21.6, 31.6 with 1024 threads)
  const bool wide = n > 8192;
  auto k = n <= 1024   ? k_quant<TYPE, 1, 256>
           : n <= 2048 ? k_quant<TYPE, 2, 256>
           : n <= 4096 ? k_quant<TYPE, 4, 256>
           : !wide     ? k_quant<TYPE, 8, 256>
           : n <= 16384 ? k_quant<TYPE, 4, 1024>
                        : k_quant<TYPE, 0, 1024>;
  hipLaunchKernelGGL(k, dim3(rows), dim3(wide ? 1024 : 256), 0, s->stream, d_x, ldx, n, d_q, ldq,
                     d_scale);
  PZ_HIP(s, hipGetLastError());
  return PZ_OK;
}

// ---- product -------------------------------------------------------------------
// v_mfma_i32_16x16x64_i8: A = 16 rows of W x 64 k, B = 64 k x 16 batch rows, D =
// 16 rows x 16 batch rows (lane l: batch row l % 16, rows 4 (l / 16) .. +3); of
// A and B lane l holds row l % 16 and the 16 bytes of k from 16 (l / 16) on.
//
//   * A workgroup owns WR TR x 16 rows of W and WC TC x 16 batch rows; wave (wr, wc, wk)
//     TR x TC tiles of it over every WKth stage of k.  k advances 128 a stage --
//     whole cache lines of W -- through a ring in LDS for each wk, NS stages of W
//     and NX of X: one load instruction brings 8 rows x 128 bytes, straight to
//     LDS, one barrier per stage.  The 16-byte pieces of a row are rotated so
//     that the fragment reads do not meet in the banks.  The fragments of one
//     product are read while the one before runs.
//   * WK > 1 for few rows of W, whose waves would be too few to cover the loads'
//     latency: 128 batch rows at 1292 x 6832 51 us with 256-row tiles, 16 so.
//   * The shape: pz_lmtile.h (i8_tile_for).  128256 x 2560: batch 1 50 us (6.6
//     TB/s), 16 58, 32 61, 64 67, 128 87, 256 111-118; bound by one read of W to
//     64 batch rows, then by LDS (a stage of a 256 x 256 tile: 192 KiB of fragments
//     and 64 KiB of loads are 0.99 us of it, its products 0.97; 2.2 us in all) and
//     the logits' 131 MB, which a workgroup writes between its tiles (89 us without
//     them, 67 without loads either).  32 x 32 x 32 products take as long (109 us fused
//     at 256; 16 x 16 x 64 104) and write the logits in 32-byte pieces.
//   * Workgroups start k at different stages, so that rows a multiple of 4 KiB
//     apart do not all meet in the same memory channels.
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

template <int WR, int WC, int WK, int TR, int TC, int NS, int NX, int MODE, bool FAST, bool NT>
__global__ __launch_bounds__(64 * WR * WC * WK) void k_lmhead_i8(
    const int8_t* __restrict__ W, const float* __restrict__ sw, int V, int n,
    const int8_t* __restrict__ X, const float* __restrict__ sx, long ldx, int nb, int ncb, int nrt,
    float* __restrict__ logits, long ld, unsigned long long* __restrict__ keys, int kstride,
    uint8_t* __restrict__ nan0) {
  constexpr int NW = WR * WC;  // waves that share a stage
  constexpr int ROWS = WR * TR * 16, COLS = WC * TC * 16;
  constexpr int KB = 128, KM = 64, KN = KB / KM;  // k of a stage, of a product; its products
  constexpr int WI = ROWS / 8, XI = COLS / 8;           // 1 KiB loads of a stage
  constexpr int WPW = (WI + NW - 1) / NW, XPW = (XI + NW - 1) / NW, PER = WPW + XPW;
  constexpr int WST = WI * 1024, XST = XI * 1024;  // bytes of a stage
  constexpr int RING = NS * WST + NX * XST;        // W's ring, then X's
  constexpr int SH = WK * RING;
  static_assert(NX >= 2 && NS >= NX, "");
  static_assert(SH >= WR * COLS * 8 && SH >= (WK - 1) * ROWS * COLS * 4,
                "the sums over WK and the epilogue's keys reuse the ring");
  __shared__ __align__(16) int8_t sh[SH];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int wk = w / NW, ws = w % NW, wr = ws % WR, wc = ws / WR;
  // the batch blocks of a row tile on one XCD, one after the other
  const int slot = blockIdx.x >> 3;
  const int rt = (slot / ncb) * 8 + (blockIdx.x & 7), cb = slot % ncb;
  if (rt >= nrt) return;
  const int row0 = rt * ROWS, b0 = cb * COLS;
  i8_i32x4 acc[TR][TC];
#pragma unroll
  for (int t = 0; t < TR; t++)
#pragma unroll
    for (int j = 0; j < TC; j++) acc[t][j] = i8_i32x4{0, 0, 0, 0};
  const int nst = (n + KB - 1) / KB;
  // This lane's part of load q: row q * 8 + lane / 8, the 16-byte piece that
  // belongs in place lane % 8 of that row: piece ^ (row / 2 % 8), so that the 16
  // rows that one cycle reads for a fragment lie in 16 places of 256 bytes.
  const int lrow = lane >> 3;
  auto piece = [&](int q) { return (lane & 7) ^ ((q & 1) << 2 | lrow >> 1); };
  // rows past V and batch rows past nb: the last one (results unused)
  auto wload_of = [&](int i) {
    const int q = ws * WPW + i;
    return WI % NW && q >= WI ? WI - 1 : q;  // (the same bytes to the same place again)
  };
  auto wrow = [&](int i) {
    const int r = wload_of(i) * 8 + lrow, last = V - 1 - row0;
    return r < last ? r : last;
  };
  auto xload_of = [&](int i) {
    const int q = ws * XPW + i;
    return XI % NW && q >= XI ? XI - 1 : q;
  };
  auto xrow = [&](int i) {
    const int r = xload_of(i) * 8 + lrow, last = nb - 1 - b0;
    return r < last ? r : last;
  };
  const int8_t* wbase = W + (size_t)row0 * n;
  const int8_t* xbase = X + (size_t)b0 * ldx;
  // fragments of k step s of a stage: i < TC those of X, then those of W
  struct Frags {
    i8_i32x4 a[TR], b[TC];
  };
  auto read = [&](Frags& f, const int8_t* wst, const int8_t* xst, int s, int i) {
    const int at = m * KB + ((s * 4 + g) ^ (m >> 1 & 7)) * 16;
    if (i < TC)
      f.b[i] = *reinterpret_cast<const i8_i32x4*>(xst + (wc * TC + i) * 16 * KB + at);
    else
      f.a[i - TC] = *reinterpret_cast<const i8_i32x4*>(wst + (wr * TR + i - TC) * 16 * KB + at);
  };
  if constexpr (FAST) {
    const uint32_t lds0 =
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)sh + wk * RING;
    uint32_t woff[WPW], xoff[XPW];
#pragma unroll
    for (int i = 0; i < WPW; i++) woff[i] = (uint32_t)wrow(i) * (uint32_t)n + 16u * piece(wload_of(i));
#pragma unroll
    for (int i = 0; i < XPW; i++) xoff[i] = (uint32_t)xrow(i) * (uint32_t)ldx + 16u * piece(xload_of(i));
    auto adj = [&](int c, int q) {  // from a piece past n back to the row's last
      const int k = (nst - 1) * KB + 16 * piece(q);
      return c < nst - 1 || k < n ? 0u : (uint32_t)(k - (n - 16));
    };
    auto issue_w = [&](int c, int buf, int i) {
      lm_lds_load16<NT>(wbase + (size_t)c * KB, woff[i] - adj(c, wload_of(i)),
                        lds0 + buf * WST + wload_of(i) * 1024);
    };
    auto issue_x = [&](int c, int buf, int i) {
      lm_lds_load16<false>(xbase + (size_t)c * KB, xoff[i] - adj(c, xload_of(i)),
                           lds0 + NS * WST + buf * XST + xload_of(i) * 1024);
    };
    // Order of the loads: X of stage c, W of stage c + NS - NX, for c = 0, 1, ..
    // with the first NS - NX of W before them.  So a wait for X of stage c leaves
    // its W done and the loads after it on their way.
    constexpr int DX = NX - 1, LEAD = NS - NX;
    const int c0 = slot % nst, turns = (nst + WK - 1) / WK;
    auto clip = [&](int c) {  // stage of turn c (past the last: any, unused)
      int k = c * WK + wk;
      k = (k < nst ? k : nst - 1) + c0;
      return k < nst ? k : k - nst;
    };
#pragma unroll
    for (int c = 0; c < LEAD; c++)
#pragma unroll
      for (int i = 0; i < WPW; i++) issue_w(clip(c), c, i);
#pragma unroll
    for (int c = 0; c < DX; c++) {
#pragma unroll
      for (int i = 0; i < XPW; i++) issue_x(clip(c), c, i);
#pragma unroll
      for (int i = 0; i < WPW; i++) issue_w(clip(c + LEAD), c + LEAD, i);
    }
    // The products of a k step while the next one's fragments are read, the
    // stages' loads between them: the last step of a stage runs behind the
    // barrier of the next, when its fragments are in registers and its slot is free.
    Frags f[2];
#pragma unroll
    for (int j = 0; j < TC; j++) f[1].b[j] = i8_i32x4{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < TR; t++) f[1].a[t] = i8_i32x4{0, 0, 0, 0};
    constexpr int NM = TR * TC, NR = TR + TC;
    auto mul = [&](const Frags& u, auto between) {
#pragma unroll
      for (int q = 0; q < NM; q++) {
        const int t = q % TR, j = q / TR;
        acc[t][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.a[t], u.b[j], acc[t][j], 0, 0, 0);
        between(q);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // (pieces past n hold the row's last piece again: zeros in B)
    auto past = [&](Frags& u, int k) {
#pragma unroll
      for (int j = 0; j < TC; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) u.b[j][e] = k + 16 * g < n ? u.b[j][e] : 0;
    };
    int wb = 0, xb = 0, nwb = NS - 1, nxb = NX - 1;
#pragma clang loop unroll(disable)
    for (int c = 0; c < turns; c++) {
      // stage c has arrived, in every wave; and every wave has read the slots
      // that are filled next
      lm_wait<(DX - 1) * PER + (LEAD ? WPW : 0)>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const int8_t* wst = sh + wk * RING + wb * WST;
      const int8_t* xst = sh + wk * RING + NS * WST + xb * XST;
      const int k0 = WK == 1 || c * WK + wk < nst ? clip(c) * KB : n;  // (n: nothing of it counts)
      const int cx = clip(c + DX), cw = clip(c + DX + LEAD);
#pragma unroll
      for (int s = 0; s < KN; s++) {
        Frags& to = f[s & 1];
        mul(f[(s + 1) & 1], [&](int q) {
#pragma unroll
          for (int i = 0; i < NR; i++)
            if (i * NM / NR == q) read(to, wst, xst, s, i);
          if (s == 0)
#pragma unroll
            for (int i = 0; i < PER; i++)
              if (i * NM / PER == q) {
                if (i < XPW) issue_x(cx, nxb, i);
                else issue_w(cw, nwb, i - XPW);
              }
        });
        past(to, k0 + s * KM);
      }
      asm volatile("" ::: "memory");
      wb = wb + 1 == NS ? 0 : wb + 1;
      xb = xb + 1 == NX ? 0 : xb + 1;
      nwb = nwb + 1 == NS ? 0 : nwb + 1;
      nxb = nxb + 1 == NX ? 0 : nxb + 1;
    }
    mul(f[1], [](int) {});
    lm_wait<0>();
  } else {

    static_assert(FAST || (NS == 2 && NX == 2), "");
    const int turns = (nst + WK - 1) / WK;
    int8_t* ring = sh + wk * RING;
    lm_u32x4 q[PER];
    auto fetch = [&](int c) {  // (zeros past n)
      const int k0 = (c * WK + wk) * KB;
#pragma unroll
      for (int i = 0; i < WPW; i++) {
        const int k = k0 + 16 * piece(wload_of(i));
        q[i] = i8_load16(wbase + (size_t)wrow(i) * n + k, n - k);
      }
#pragma unroll
      for (int i = 0; i < XPW; i++) {
        const int k = k0 + 16 * piece(xload_of(i));
        q[WPW + i] = i8_load16(xbase + (size_t)xrow(i) * ldx + k, n - k);
      }
    };
    fetch(0);
#pragma clang loop unroll(disable)
    for (int c = 0; c < turns; c++) {
      int8_t* wst = ring + (c & 1) * WST;
      int8_t* xst = ring + NS * WST + (c & 1) * XST;
#pragma unroll
      for (int i = 0; i < WPW; i++)
        *reinterpret_cast<lm_u32x4*>(wst + wload_of(i) * 1024 + lane * 16) = q[i];
#pragma unroll
      for (int i = 0; i < XPW; i++)
        *reinterpret_cast<lm_u32x4*>(xst + xload_of(i) * 1024 + lane * 16) = q[WPW + i];
      __syncthreads();
      if (c + 1 < turns) fetch(c + 1);
#pragma unroll
      for (int s = 0; s < KN; s++) {
        Frags f;
#pragma unroll
        for (int i = 0; i < TR + TC; i++) read(f, wst, xst, s, i);
#pragma unroll
        for (int j = 0; j < TC; j++)
#pragma unroll
          for (int t = 0; t < TR; t++)
            acc[t][j] =
                __builtin_amdgcn_mfma_i32_16x16x64_i8(f.a[t], f.b[j], acc[t][j], 0, 0, 0);
      }
      // (the slot written next was last read before this stage's barrier)
    }
  }
  if constexpr (WK > 1) {
    // the sums over the k of the other wave groups
    __syncthreads();
    i8_i32x4* part = reinterpret_cast<i8_i32x4*>(sh);
    if (wk > 0)
#pragma unroll
      for (int t = 0; t < TR; t++)
#pragma unroll
        for (int j = 0; j < TC; j++)
          part[(((wk - 1) * NW + ws) * TR * TC + t * TC + j) * 64 + lane] = acc[t][j];
    __syncthreads();
    if (wk > 0 && MODE == 0) return;
    if (wk == 0)
#pragma unroll
      for (int t = 0; t < TR; t++)
#pragma unroll
        for (int j = 0; j < TC; j++)
#pragma unroll
          for (int o = 0; o < WK - 1; o++)
            acc[t][j] += part[((o * NW + ws) * TR * TC + t * TC + j) * 64 + lane];
  }
  // epilogue: lane l holds batch row l % 16 of each tile, rows 4 (l / 16) + i
  float fx[TC];
#pragma unroll
  for (int j = 0; j < TC; j++) {
    const int b = b0 + (wc * TC + j) * 16 + m;
    fx[j] = b < nb ? sx[b] : 0.0f;
  }
  const bool vec = MODE == 0 && (ld & 3) == 0 && ((uintptr_t)logits & 15) == 0;
  // A tile's logits go out as whole rows of the batch, 256 bytes and more together:
  // the workgroup turns 16 batch rows of each wc at a time in LDS.  (256 x 2560 x
  // 128256 131 -> 123 us, to 50257 logits, whose rows are off 16 bytes, 74 -> 64; a
  // batch of 8 the same.  Written past the caches they take 114, but then what reads
  // them next loses more: with their maxima 148 -> 154.)
  constexpr int RS = ROWS + 4, CG = WC * 16;  // floats of a row there, rows
  constexpr bool TURN = MODE == 0 && WK == 1 && ROWS >= 64 && SH >= CG * RS * 4;
  if constexpr (TURN) {
    constexpr int NB = SH >= 2 * CG * RS * 4 ? 2 : 1, TH = 64 * NW;
    __syncthreads();  // the ring is free
#pragma unroll
    for (int j = 0; j < TC; j++) {
      float* turn = reinterpret_cast<float*>(sh) + (j % NB) * CG * RS;
      if (NB == 1 && j > 0) __syncthreads();
#pragma unroll
      for (int t = 0; t < TR; t++) {
        const int r = (wr * TR + t) * 16 + 4 * g;
        lm_f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; i++)
          y[i] = ((float)acc[t][j][i] * (row0 + r + i < V ? sw[row0 + r + i] : 0.0f)) * fx[j];
        *reinterpret_cast<lm_f32x4*>(turn + (wc * 16 + m) * RS + r) = y;
      }
      __syncthreads();
      auto batch = [&](int c) { return b0 + ((c >> 4) * TC + j) * 16 + (c & 15); };
      if (vec) {
#pragma unroll 4
        for (int i = tid; i < CG * ROWS / 4; i += TH) {
          const int c = i / (ROWS / 4), r = i % (ROWS / 4) * 4, row = row0 + r, b = batch(c);
          if (b >= nb) continue;
          const lm_f32x4 y = *reinterpret_cast<const lm_f32x4*>(turn + c * RS + r);
          float* o = logits + (size_t)b * ld + row;
          if (row + 3 < V) {
            *reinterpret_cast<lm_f32x4*>(o) = y;
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (row + e < V) o[e] = y[e];
          }
        }
      } else {
#pragma unroll 4
        for (int i = tid; i < CG * ROWS; i += TH) {
          const int c = i / ROWS, r = i % ROWS, row = row0 + r, b = batch(c);
          if (b >= nb || row >= V) continue;
          logits[(size_t)b * ld + row] = turn[c * RS + r];
        }
      }
    }
    return;
  }
  // (rows in descending order, so that >= leaves the first of equal ones, and
  // -infinity counts where there is nothing above it; NaN never does)
  float bv[TC];
  int bi[TC];
#pragma unroll
  for (int j = 0; j < TC; j++) {
    bv[j] = -__builtin_inff();
    bi[j] = -1;
  }
#pragma unroll
  for (int t = TR - 1; t >= 0; t--) {
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
          for (int i = 3; i >= 0; i--) {
            const bool up = row + i < V && y[i] >= bv[j];
            bv[j] = up ? y[i] : bv[j];
            bi[j] = up ? row + i : bi[j];
          }
          if (row == 0 && wk == 0) nan0[b] = y[0] != y[0] ? 1 : 0;
        }
      }
    }
  if (MODE == 1) {
    __syncthreads();  // the ring is free
    unsigned long long* best_sh = reinterpret_cast<unsigned long long*>(sh);  // [WR][COLS]
#pragma unroll
    for (int j = 0; j < TC; j++) {
      unsigned long long best = bi[j] < 0 ? 0ull : argmax_key(bv[j], bi[j]);
      // the maximum over the lane groups, then over the row waves
#pragma unroll
      for (int off = 16; off < 64; off <<= 1) {
        const unsigned long long o = __shfl_xor(best, off, 64);
        best = o > best ? o : best;
      }
      if (g == 0 && wk == 0) best_sh[wr * COLS + (wc * TC + j) * 16 + m] = best;
    }
    __syncthreads();
    for (int bl = tid; bl < COLS; bl += 64 * NW * WK) {
      const int b = b0 + bl;
      if (b >= nb) break;
      unsigned long long mx = best_sh[bl];
#pragma unroll
      for (int i = 1; i < WR; i++) {
        const unsigned long long o = best_sh[i * COLS + bl];
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

template <int WR, int WC, int WK, int TR, int TC, int NS, int NX, int MODE, bool FAST>
int launch(pz_sampler* s, const I8Call& c) {
  constexpr int rows = WR * TR * 16, cols = WC * TC * 16;
  const int ncb = (c.B + cols - 1) / cols, nrt = (c.V + rows - 1) / rows;
  const int64_t grid = i8_workgroups(c.V, c.B, rows, cols);
  if (!pz_launch_fits(grid, 64 * WR * WC * WK))
    return fail(s, PZ_ERANGE, "V=%d x B=%d are more tiles than a launch takes", c.V, c.B);
  // weights past the Infinity Cache are not kept (lm_once counts bf16 weights)
  auto k = FAST && lm_once(c.V, (c.n + 1) / 2)
               ? k_lmhead_i8<WR, WC, WK, TR, TC, NS, NX, MODE, FAST, FAST>
               : k_lmhead_i8<WR, WC, WK, TR, TC, NS, NX, MODE, FAST, false>;
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * WR * WC * WK), 0, s->stream, c.w, c.sw, c.V, c.n, c.x,
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
    switch (i8_odd_tile_for(c.V, c.B, s->n_cu)) {
      case 0: return launch<2, 1, 4, 1, 1, 2, 2, MODE, false>(s, c);
      case 1: return launch<2, 1, 2, 1, 1, 2, 2, MODE, false>(s, c);
      case 2: return launch<2, 2, 2, 1, 2, 2, 2, MODE, false>(s, c);
      case 3: return launch<2, 2, 1, 2, 2, 2, 2, MODE, false>(s, c);
      case 4: return launch<4, 1, 1, 2, 4, 2, 2, MODE, false>(s, c);
      case 5: return launch<2, 2, 2, 1, 4, 2, 2, MODE, false>(s, c);
      case 6: return launch<2, 2, 2, 2, 4, 2, 2, MODE, false>(s, c);
      default: return launch<4, 2, 1, 2, 4, 2, 2, MODE, false>(s, c);
    }
  }
  const int tile = i8_tile_for(c.V, c.B, s->n_cu);
  switch (tile) {
#define PZ_I8_CASE(I, ...) \
  case I: return launch<__VA_ARGS__, MODE, true>(s, c)
    // waves over rows of W, batch rows and k, their tiles, stages of W and X
    PZ_I8_CASE(0, 1, 1, 4, 1, 1, 4, 4);
    PZ_I8_CASE(1, 2, 1, 1, 1, 1, 4, 4);
    PZ_I8_CASE(2, 4, 1, 1, 1, 1, 4, 4);
    PZ_I8_CASE(3, 1, 1, 4, 1, 2, 3, 3);
    PZ_I8_CASE(4, 2, 1, 2, 1, 2, 4, 4);
    PZ_I8_CASE(5, 4, 1, 1, 2, 2, 3, 3);
    PZ_I8_CASE(6, 1, 2, 4, 1, 2, 4, 4);
    PZ_I8_CASE(7, 2, 2, 2, 1, 2, 4, 4);
    PZ_I8_CASE(8, 2, 2, 1, 2, 2, 3, 3);
    PZ_I8_CASE(9, 2, 2, 1, 4, 2, 2, 2);
    PZ_I8_CASE(10, 4, 2, 1, 4, 2, 2, 2);
    PZ_I8_CASE(11, 1, 4, 2, 1, 2, 4, 4);
    PZ_I8_CASE(12, 1, 4, 2, 2, 2, 3, 3);
    PZ_I8_CASE(13, 2, 2, 1, 2, 4, 2, 2);
    PZ_I8_CASE(14, 4, 2, 1, 4, 4, 3, 3);
    PZ_I8_CASE(15, 1, 4, 2, 1, 4, 2, 2);
    PZ_I8_CASE(16, 1, 8, 1, 2, 2, 2, 2);
    PZ_I8_CASE(17, 2, 4, 1, 2, 4, 2, 2);
    PZ_I8_CASE(18, 2, 4, 1, 4, 4, 3, 3);
    default: return launch<2, 4, 1, 8, 4, 3, 2, MODE, true>(s, c);
#undef PZ_I8_CASE
  }
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
