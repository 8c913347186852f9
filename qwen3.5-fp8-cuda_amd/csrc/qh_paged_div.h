// Quotients of the paged cache's kernels without a division: the launch derives what the
// kernel multiplies by.  Plain arithmetic, the same on the host and in a kernel.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define QH_HD __host__ __device__ __forceinline__
#else
#define QH_HD inline
#endif

// x / d for 0 <= x < 2^31 and d = 8 .. 2^31 - 1: with s = ceil(log2 d) >= 3,
// m = floor(2^(31+s) / d) + 1 is below 2^32 and floor(x m / 2^(31+s)) = floor(x / d),
// as m d - 2^(31+s) <= d <= 2^s.
struct QhDiv {
  uint32_t mul;
  int shift;
};
inline QhDiv qh_div_by(uint32_t d) {
  int s = 3;
  while ((1ull << s) < d) ++s;
  return QhDiv{(uint32_t)((1ull << (31 + s)) / d + 1), s - 1};
}
QH_HD int qh_quotient(int x, uint32_t mul, int shift) {
  return (int)((uint32_t)((uint64_t)(uint32_t)x * mul >> 32) >> shift);
}

// i / group for 0 <= i < 1024 and group = 1 .. 16: floor(i mul / 2^20) with
// mul = ceil(2^20 / group), as mul group - 2^20 < 16.
inline uint32_t qh_group_mul(int group) { return ((1u << 20) + group - 1) / group; }
QH_HD int qh_group_quotient(int i, uint32_t mul) { return (int)((uint32_t)i * mul >> 20); }

// a / b for a >= 0, b > 0 and quotients below 2^20, from a reciprocal of b that is off by an
// ulp at most: the product is off by less than 1.
QH_HD int qh_quotient_near(int a, int b, float reciprocal) {
  const int q = (int)((float)a * reciprocal);
  const int rest = (int)((uint32_t)a - (uint32_t)q * (uint32_t)b);
  return rest < 0 ? q - 1 : rest >= b ? q + 1 : q;
}
