// Prefix sums and extremes over a wave by moves between lanes within the registers (DPP), where a
// butterfly of __shfl calls goes through LDS.
#pragma once

#include "qh_common.h"

template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T dpp_or_zero(T v) {
  static_assert(sizeof(T) == 8, "two registers");
  const u32x2 u = __builtin_bit_cast(u32x2, v);
  const u32x2 r = {(uint32_t)__builtin_amdgcn_update_dpp(0, (int)u.x, CTRL, ROWS, 0xF, false),
                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u.y, CTRL, ROWS, 0xF, false)};
  return __builtin_bit_cast(T, r);
}
template <typename T>
__device__ __forceinline__ T lane63(T v) {
  const u32x2 u = __builtin_bit_cast(u32x2, v);
  const u32x2 r = {(uint32_t)__builtin_amdgcn_readlane((int)u.x, 63), (uint32_t)__builtin_amdgcn_readlane((int)u.y, 63)};
  return __builtin_bit_cast(T, r);
}
// Exclusive prefix over the wave and its total (64-bit values), by moves between lanes within the
// registers: shifts within rows of 16, then the rows' last lanes handed on.
template <typename T>
__device__ __forceinline__ T wave_excl(T v, T& all) {
  T x = v;
  x += dpp_or_zero<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8
  x += dpp_or_zero<0x112, 0xF>(x);
  x += dpp_or_zero<0x114, 0xF>(x);
  x += dpp_or_zero<0x118, 0xF>(x);
  x += dpp_or_zero<0x142, 0xA>(x);  // row_bcast 15 into rows 1 and 3
  x += dpp_or_zero<0x143, 0xC>(x);  // row_bcast 31 into rows 2 and 3
  all = lane63(x);
  return dpp_or_zero<0x138, 0xF>(x);  // wave_shr 1
}
constexpr int kNone = 0x7FFFFFFF;  // larger than any value that wave_min looks at

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_min(int v) {
  return min(v, __builtin_amdgcn_update_dpp(kNone, v, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ int wave_min(int v) {
  v = dpp_min<0x111, 0xF>(v);
  v = dpp_min<0x112, 0xF>(v);
  v = dpp_min<0x114, 0xF>(v);
  v = dpp_min<0x118, 0xF>(v);
  v = dpp_min<0x142, 0xA>(v);
  v = dpp_min<0x143, 0xC>(v);
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ int wave_max_int(int v) { return -wave_min(-v); }
