// pz_beamexp.h -- the exponential of beam selection in 64 bits.  Plain arithmetic, for the
// kernels and for a test of it without a device.
//
// Table-driven, after P. T. P. Tang's method (ACM Transactions on Mathematical Software 15,
// 1989): exp(x) = 2^(n / 32) exp(r), n the whole number nearest to 32 x / ln 2 (which the sum
// with 1.5 2^52 leaves in its last bits) and |r| <= ln 2 / 64: 2^(n % 32 / 32) from a table,
// n / 32 into its exponent, and exp(r) from its series up to r^4, with r^5 / 120 replaced by
// the cubic that is nearest on the interval (Chebyshev's).  A result is off by at most 2^-43 of
// itself: 0.7 of that by the series, 0.2 by n ln 2 / 32, whose factor is rounded, for the
// largest |x|.
#pragma once
#include <stdint.h>

#include "pz_pages.h"

namespace {

typedef uint32_t be_u32x2 __attribute__((vector_size(8)));  // low, high

// The bits of 2^(i / 32) less i 2^47, so that all of n may be added.
#ifdef __HIPCC__
__constant__ const uint64_t be_roots[32] = {
#else
const uint64_t be_roots[32] = {
#endif
    0x3ff0000000000000ull, 0x3fefd9b0d3158574ull, 0x3fefb5586cf9890full, 0x3fef9301d0125b51ull,
    0x3fef72b83c7d517bull, 0x3fef54873168b9aaull, 0x3fef387a6e756238ull, 0x3fef1e9df51fdee1ull,
    0x3fef06fe0a31b715ull, 0x3feef1a7373aa9cbull, 0x3feedea64c123422ull, 0x3feece086061892dull,
    0x3feebfdad5362a27ull, 0x3feeb42b569d4f82ull, 0x3feeab07dd485429ull, 0x3feea47eb03a5585ull,
    0x3feea09e667f3bcdull, 0x3fee9f75e8ec5f74ull, 0x3feea11473eb0187ull, 0x3feea589994cce13ull,
    0x3feeace5422aa0dbull, 0x3feeb737b0cdc5e5ull, 0x3feec49182a3f090ull, 0x3feed503b23e255dull,
    0x3feee89f995ad3adull, 0x3feeff76f2fb5e47ull, 0x3fef199bdd85529cull, 0x3fef3720dcef9069ull,
    0x3fef5818dcfba487ull, 0x3fef7c97337b9b5full, 0x3fefa4afa2a490daull, 0x3fefd0765b6e4540ull};
constexpr double BE_PER = 46.1662413084468290355, BE_STEP = 0.0216608493924982909193;
constexpr double BE_C1 = 0.999999999964169676946, BE_C3 = 0.166667888521865636702;

// sum + exp(d), |d| <= 700.  roots: be_roots, as low and high words.
template <class TABLE>
PZ_HD double be_add_exp(double sum, double d, TABLE roots) {
  constexpr double ROUND = 6755399441055744.0;  // 1.5 2^52
  const double t = __builtin_fma(d, BE_PER, ROUND), n = t - ROUND;
  const double r = __builtin_fma(n, -BE_STEP, d);
  const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, t);
  be_u32x2 root = roots[k & 31u];
  root[1] += k << 15;
  const double scale = __builtin_bit_cast(double, root);
  double p = __builtin_fma(r, 1.0 / 24.0, BE_C3);
  p = __builtin_fma(r, p, 0.5);
  p = __builtin_fma(r, p, BE_C1);
  p = __builtin_fma(r, p, 1.0);
  return __builtin_fma(p, scale, sum);
}
// exp(x - m), x <= m
template <class TABLE>
PZ_HD double be_exp(float x, float m, TABLE roots) {
  const double d = (double)x - (double)m;
  return be_add_exp(0.0, d < -700.0 ? -700.0 : d, roots);  // (10^-304 at least; a NaN stays)
}

}  // namespace
