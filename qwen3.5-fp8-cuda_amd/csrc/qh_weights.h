// Weights of a row's logits as whole numbers in the units of bins, a quarter of an octave each, below the
// row's largest (sample_rows.hip).  Plain arithmetic, the same on the host and in a kernel: each fused
// operation is written as one, so that no bin depends on what a compiler contracts.
#pragma once

#include <math.h>
#include <stdint.h>

#if defined(__HIPCC__)
#define QH_HD __host__ __device__ __forceinline__
#else
#define QH_HD inline
#endif

namespace {

constexpr int kBins = 256;
// 2^(g / 4) by the polynomial through its seven Chebyshev points of [-1/2, 1/2], scaled so that g = 0
// gives a whole number: weights of equal logits add up without a rounding.
constexpr uint64_t kOne = 31508019007;        // about 2^35 2^(-1/8)
constexpr double kP1 = 5459923634.982943, kP2 = 473066334.20437115, kP3 = 27325381.376510937, kP4 = 1183781.9759320344,
                 kP5 = 41039.59278978226, kP6 = 1185.1772411226116;
constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: added to |t| < 2^50, the sum's low bits are the nearest integer
constexpr double kWhole = 4503599627370496.0;  // 2^52

QH_HD uint64_t bits(double d) { return __builtin_bit_cast(uint64_t, d); }

// e + 2^52 of a weight e in its bin's units, rounded to an integer by the last addition.
QH_HD double power(double g) {
  double e = fma(kP6, g, kP5);
  e = fma(e, g, kP4);
  e = fma(e, g, kP3);
  e = fma(e, g, kP2);
  e = fma(e, g, kP1);
  return fma(e, g, (double)kOne + kWhole);
}

// The weights below a largest logit; t = x c4, x = t c4_inv.
struct Scale {
  double c4, base;  // base: the largest's bin
  float top;        // the largest
  bool far;         // |t| of it is 2^50 or more (or it is infinite): no other logit is near enough to have a weight
  // Logits far below the largest are lifted to `least`, 400 bins below it, and go to a bin that nobody reads:
  // no branch a logit, and no number that its bin's 32 bits do not hold.  Not `quick`, where that is not a
  // number, or 24 bits of a logit do not tell bins apart: then each is looked at.
  bool quick;
  float least;
  uint32_t first;
  QH_HD Scale(double c4_, double c4_inv, float top_) : c4(c4_), top(top_) {
    const double t = (double)top * c4;
    far = !(fabs(t) < 1125899906842624.0);
    // from the same fused product as every logit's bin: of a product rounded on its own the nearest integer may
    // be one below, and the largest logit's bin -1
    base = fabsf(top) == INFINITY ? (double)top : far ? t : fma((double)top, c4, kRound) - kRound;
    least = (float)((base - 400.0) * c4_inv);
    quick = !far && fabs(base) < 67108864.0 && least > -INFINITY;
    first = (uint32_t)bits(kRound + base);
  }
  // The bin of a logit below `base` and its weight in the bin's units; false where it has none.
  QH_HD bool weigh(float x, int& bin, uint64_t& fx) const {
    if (far) {
      bin = 0;
      fx = kOne;
      return x == top && top > -INFINITY;
    }
    const double tm = fma((double)x, c4, kRound), d = (kRound + base) - tm;
    if (!(d < (double)kBins)) return false;
    bin = (int)d;
    fx = bits(power(fma((double)x, c4, -(tm - kRound)))) & 0xFFFFFFFFFull;
    return true;
  }
  // The same where `quick`: bin kBins without a weight, the weight with 2^52 added.
  QH_HD double weigh_quick(float x, int& bin) const {
    const double v = x > least ? x : least;
    const double tm = fma(v, c4, kRound);
    const uint32_t below = first - (uint32_t)bits(tm);
    bin = (int)(below < (uint32_t)kBins ? below : (uint32_t)kBins);
    return power(fma(v, c4, -(tm - kRound)));
  }
};

}  // namespace
