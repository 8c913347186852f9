// Low-rank adapters of many requests at once, beside a projection that they share (gfx950):
//
//   out[t] = y[t] + scale[a] * B_a (A_a x[t]),   a = ids[t];   out[t] = y[t] without an adapter
//
// with A_a [R][K], B_a [N][R] and all of x, y, A, B, out in bf16.  Two launches: the first
// multiplies by A (h, [slices][T][rank] fp32, each slice of K a partial sum), the second by B
// and adds.  Both run on the matrix cores over tiles of tokens and, within a tile, over the
// adapters that its tokens name, each loaded once: tokens need no sorting, a prompt's tile has
// one adapter or two, a decode tile up to one a token.  A tile is multiplied by an adapter as
// a whole; a token keeps the product of its own and drops the others, so that what another
// request's adapter holds, NaN included, never reaches it.
//
// Bound by bytes: A and B of the adapters in use (decode), x, y and out (prompts), and by the two
// launches, as the second waits for the first.  3700 tokens, K 2560, N 9216, rank 32: 12 + 34 us,
// 158 MB, 3.4 TB/s (a copy: 30.6 us); a token (rank 16) 7.5 us, 48 of decode 10.3.
//
// h stays in fp32 between the launches and enters the second product as two bf16 numbers,
// high and low, which together lose 2^-16 of it: one rounding would cost as much as the
// rounding of the output.  The high part is cut off, not rounded: so both have h's sign, an
// infinity of B times either is the same infinity, and no finite h becomes an infinite one.
// Products and sums are fp32, the output is rounded once.
#include "qh_common.h"
#include "qh_serve.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ u32x4 load16(const uint16_t* p) { return *(const u32x4*)p; }

// The upper 8 bits of x and y, side by side (a NaN that arithmetic gave has its mark among them).
__device__ __forceinline__ uint32_t high_parts(float x, float y) {
  return __float_as_uint(x) >> 16 | (__float_as_uint(y) & 0xFFFF0000u);
}
// What the high part leaves of x, never quite nothing (2^-30 of x, of an infinity too) but of a zero: an infinity
// of B times nothing would be NaN.
__device__ __forceinline__ float low_part(float x, float high) {
  const float least = fmaxf(0x1p-30f * fminf(fabsf(x), 0x1p127f), 0x1p-133f);
  return x == 0.0f ? 0.0f : copysignf(fmaxf(fabsf(x - high), least), x);
}

// The adapters that a tile's tokens name, one after the other: lane i of the wave holds token
// i's (below 0: none).
struct TileIds {
  int id;
  uint64_t left;
  __device__ __forceinline__ TileIds(const QhAdaptersParams& p, int t0, int tokens) {
    const int lane = threadIdx.x & 63;
    id = -1;
    if (lane < tokens && t0 + lane < p.T) id = p.ids[t0 + lane];
    if (id >= p.n) id = -1;
    left = __ballot(id >= 0);
  }
  // The next adapter and the tokens (bits) that name it; only while `left`.
  __device__ __forceinline__ int next(uint64_t& tokens) {
    const int a = __builtin_amdgcn_readlane(id, (int)__builtin_ctzll(left));
    tokens = __ballot(id == a);
    left &= ~tokens;
    return a;
  }
};

// ---- h = A x -----------------------------------------------------------------------------
// A workgroup: 16 MT tokens, one slice of K, the tile's adapters z, z + gridDim.z, ...  Its eight
// waves take the slice's blocks of 64 in turn, BLOCKS of them with all loads on their way at once,
// and add up through LDS.
constexpr int kShrinkWaves = 8;

template <int MT, int RT, int BLOCKS>  // RT: tiles of 16 ranks
__global__ __launch_bounds__(64 * kShrinkWaves) void adapters_shrink_kernel(QhAdaptersParams p, int slice) {
  __shared__ f32x4 s_part[kShrinkWaves][MT * RT][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.y * 16 * MT, k0 = blockIdx.x * slice, k1 = min(p.K, k0 + slice);
  TileIds tile(p, t0, 16 * MT);
  const uint16_t* xr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = p.x + (long long)min(t0 + 16 * m + row, p.T - 1) * p.x_ts;
  const int Rp = 16 * ((p.R + 15) / 16);
  const u32x4 zero = {0, 0, 0, 0};
  for (int j = 0; tile.left != 0; ++j) {
    uint64_t mine;
    const int a = tile.next(mine);
    if (j % gridDim.z != blockIdx.z) continue;
    const uint16_t* ar[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) ar[r] = p.a + ((size_t)a * p.R + min(16 * r + row, p.R - 1)) * p.K;
    f32x4 acc[MT][RT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[m][r] = f32x4{0, 0, 0, 0};
    for (int k = k0 + 64 * wid; k < k1; k += 64 * kShrinkWaves * BLOCKS) {
      u32x4 x[2 * BLOCKS][MT], w[2 * BLOCKS][RT];
#pragma unroll
      for (int i = 0; i < 2 * BLOCKS; ++i) {
        const int c = k + 64 * kShrinkWaves * (i / 2) + 32 * (i % 2) + 8 * g;
        const bool in = c < k1;
#pragma unroll
        for (int r = 0; r < RT; ++r) w[i][r] = in ? load16(ar[r] + c) : zero;
#pragma unroll
        for (int m = 0; m < MT; ++m) x[i][m] = in ? load16(xr[m] + c) : zero;
      }
#pragma unroll
      for (int i = 0; i < 2 * BLOCKS; ++i)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m][r] = mfma(w[i][r], x[i][m], acc[m][r]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < RT; ++r) s_part[wid][m * RT + r][lane] = acc[m][r];
    __syncthreads();
    // lane: token row of its tile of 16, ranks 16 r + 4 g .. + 3
    for (int q = wid; q < MT * RT; q += kShrinkWaves) {
      const int m = q / RT, r = q % RT;
      f32x4 s = s_part[0][q][lane];
#pragma unroll
      for (int v = 1; v < kShrinkWaves; ++v) s += s_part[v][q][lane];
      if ((mine >> (16 * m + row)) & 1 && 16 * r < Rp)
        *(f32x4*)(p.h + ((size_t)blockIdx.x * p.T + t0 + 16 * m + row) * Rp + 16 * r + 4 * g) = s;
    }
    __syncthreads();
  }
}

// ---- out = y + scale B h -------------------------------------------------------------------
// The rows of B are the first operand, in an order that leaves each lane 8 consecutive columns of one
// token: of a pair of products, the first has columns 8 m + 0 .. 3 and the second 8 m + 4 .. 7 of each
// eight.  Ranks go 32 to a product, high and low parts one after the other; rank 16 (and 8) has both
// parts in one, side by side (SMALL).
template <int RC, bool SMALL>
__device__ __forceinline__ u32x4 load_b(const QhAdaptersParams& p, int a, int c0, int q, int c) {
  const int row = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4, r0 = SMALL ? 8 * (g & 1) : 32 * c + 8 * g;
  const int col = min(c0 + 32 * (q / 2) + 8 * (row >> 2) + 4 * (q % 2) + (row & 3), p.N - 1);
  return r0 < p.R ? load16(p.b + ((size_t)a * p.N + col) * p.R + r0) : u32x4{0, 0, 0, 0};
}

// A tile's h, summed over the slices of K, scaled and in two parts, once a workgroup: 4 ranks a thread.
// A row's 16 bytes of padding spread its reads over the banks.
template <int TOKENS, int RC, bool SMALL>
struct TileH {
  static constexpr int kRanks = SMALL ? 16 : 32 * RC;
  uint16_t hi[TOKENS][kRanks + 8], lo[TOKENS][kRanks + 8];

  __device__ __forceinline__ void join(const QhAdaptersParams& p, int t0, int token_id, int slices) {
    const int Rp = 16 * ((p.R + 15) / 16);
    for (int i = threadIdx.x; i < TOKENS * kRanks / 4; i += blockDim.x) {
      const int row = i / (kRanks / 4), r = 4 * (i % (kRanks / 4)), id = __shfl(token_id, row, 64);
      f32x4 u = {0, 0, 0, 0};
      if (id >= 0 && r < p.R) {
        const float* h = p.h + (size_t)(t0 + row) * Rp + r;
        for (int q0 = 0; q0 < slices; q0 += 4) {
          f32x4 v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = *(const f32x4*)(h + (size_t)min(q0 + q, slices - 1) * p.T * Rp);
#pragma unroll
          for (int q = 0; q < 4; ++q) u += q0 + q < slices ? v[q] : f32x4{0, 0, 0, 0};
        }
        u *= p.scale[id];
      }
      const u32x2 top = {high_parts(u.x, u.y), high_parts(u.z, u.w)};
      *(u32x2*)&hi[row][r] = top;
      *(u32x2*)&lo[row][r] = u32x2{pack_bf2(low_part(u.x, bf_lo(top.x)), low_part(u.y, bf_hi(top.x))),
                                   pack_bf2(low_part(u.z, bf_lo(top.y)), low_part(u.w, bf_hi(top.y)))};
    }
    __syncthreads();
  }
  // The lane's token of sub-tile m and its 8 ranks of product c.
  __device__ __forceinline__ void get(int m, int c, u32x4& high, u32x4& low) const {
    const int row = 16 * m + (threadIdx.x & 15), g = (threadIdx.x & 63) >> 4, r0 = SMALL ? 8 * (g & 1) : 32 * c + 8 * g;
    low = *(const u32x4*)&lo[row][r0];
    high = SMALL && g >= 2 ? low : *(const u32x4*)&hi[row][r0];
  }
};

// y plus a lane's 8 columns of a product.
__device__ __forceinline__ u32x4 add8(u32x4 y, f32x4 u, f32x4 v) {
  return u32x4{pack_bf2(bf_lo(y.x) + u.x, bf_hi(y.x) + u.y), pack_bf2(bf_lo(y.y) + u.z, bf_hi(y.y) + u.w),
               pack_bf2(bf_lo(y.z) + v.x, bf_hi(y.z) + v.y), pack_bf2(bf_lo(y.w) + v.z, bf_hi(y.w) + v.w)};
}

// Few tokens, or few columns.  A wave: 16 tokens and 32 columns.  What it waits for is B, so the rows of
// AT adapters are on their way at once, and the first of them and y before h is there.
template <int RC, bool SMALL, int AT>
__global__ __launch_bounds__(256) void adapters_expand_few_kernel(QhAdaptersParams p, int slices) {
  __shared__ TileH<16, RC, SMALL> s_h;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.y * 16, c0 = (blockIdx.x * 4 + wid) * 32, t = t0 + row, col = c0 + 8 * g;
  TileIds tile(p, t0, 16);
  const int token_id = tile.id, mine = __shfl(tile.id, row, 64);
  int a[AT], count;
  u32x4 b[AT][RC][2];
  auto load = [&]() {
    count = 0;
#pragma unroll
    for (int n = 0; n < AT; ++n) {
      if (tile.left == 0) continue;
      uint64_t tokens;
      a[n] = tile.next(tokens);
      count = n + 1;
#pragma unroll
      for (int c = 0; c < RC; ++c)
#pragma unroll
        for (int q = 0; q < 2; ++q) b[n][c][q] = load_b<RC, SMALL>(p, a[n], c0, q, c);
    }
  };
  load();
  u32x4 y = {0, 0, 0, 0};
  if (t < p.T && col < p.N) y = load16(p.y + t * p.y_ts + col);
  s_h.join(p, t0, token_id, slices);
  if (c0 >= p.N) return;
  u32x4 hi[RC], lo[RC];
#pragma unroll
  for (int c = 0; c < RC; ++c) s_h.get(0, c, hi[c], lo[c]);
  f32x4 acc[2] = {};
  while (count > 0) {
#pragma unroll
    for (int n = 0; n < AT; ++n) {
      if (n >= count) continue;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        f32x4 d = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < RC; ++c) {
          d = mfma(b[n][c][q], hi[c], d);
          if (!SMALL) d = mfma(b[n][c][q], lo[c], d);
        }
        if (mine == a[n]) acc[q] = d;
      }
    }
    load();
  }
  if (t >= p.T || col >= p.N || (mine < 0 && p.out == p.y)) return;
  // a row without an adapter is copied as it is
  *(u32x4*)(p.out + t * p.out_ts + col) = mine >= 0 ? add8(y, acc[0], acc[1]) : y;
}

// Prompts.  A wave: 16 MT tokens and 32 CG columns, whose rows of B stay in registers while the tokens go
// by, 16 at a time; eight waves side by side share h.  What counts is y and out: y is on its way at
// once, behind h (loads come back in order).
template <int MT, int RC, bool SMALL, int CG>
__global__ __launch_bounds__(512, 4) void adapters_expand_kernel(QhAdaptersParams p, int slices) {
  __shared__ TileH<16 * MT, RC, SMALL> s_h;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.y * 16 * MT, c0 = (blockIdx.x * 8 + wid) * 32 * CG, col = c0 + 8 * g;
  TileIds tile(p, t0, 16 * MT);
  const int token_id = tile.id;
  s_h.join(p, t0, token_id, slices);
  if (c0 >= p.N) return;
  int mine[MT];
  u32x4 y[MT][CG];
  bool asked = false;
  do {
    uint64_t tokens = 0;
    const int a = tile.left != 0 ? tile.next(tokens) : -1;
    u32x4 b[RC][2 * CG];
    if (a >= 0) {
#pragma unroll
      for (int c = 0; c < RC; ++c)
#pragma unroll
        for (int q = 0; q < 2 * CG; ++q) b[c][q] = load_b<RC, SMALL>(p, a, c0, q, c);
    }
    if (!asked) {
      asked = true;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        mine[m] = __shfl(token_id, 16 * m + row, 64);
#pragma unroll
        for (int q = 0; q < CG; ++q) {
          const int t = min(t0 + 16 * m + row, p.T - 1);
          y[m][q] = col + 32 * q < p.N ? load16(p.y + t * p.y_ts + col + 32 * q) : u32x4{0, 0, 0, 0};
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (((tokens >> (16 * m)) & 0xFFFF) == 0) continue;
      f32x4 d[2 * CG] = {};
#pragma unroll
      for (int c = 0; c < RC; ++c) {
        u32x4 hi, lo;
        s_h.get(m, c, hi, lo);
#pragma unroll
        for (int q = 0; q < 2 * CG; ++q) {
          d[q] = mfma(b[c][q], hi, d[q]);
          if (!SMALL) d[q] = mfma(b[c][q], lo, d[q]);
        }
      }
#pragma unroll
      for (int q = 0; q < CG; ++q)
        if (mine[m] == a && col + 32 * q < p.N)
          *(u32x4*)(p.out + (long long)(t0 + 16 * m + row) * p.out_ts + col + 32 * q) = add8(y[m][q], d[2 * q], d[2 * q + 1]);
    }
  } while (tile.left != 0);
  if (p.out == p.y) return;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int q = 0; q < CG; ++q)  // rows without an adapter are copied as they are
      if (mine[m] < 0 && t0 + 16 * m + row < p.T && col + 32 * q < p.N)
        *(u32x4*)(p.out + (long long)(t0 + 16 * m + row) * p.out_ts + col + 32 * q) = y[m][q];
}

// Slices of K whose partial sums the workspace holds.
int max_slices(int T) { return T <= 2048 ? 8 : T <= 16384 ? 16384 / T : 1; }

template <int MT, int RT, int BLOCKS>
void shrink(const QhAdaptersParams& p, int slices, int slice, int z, hipStream_t st) {
  const dim3 grid(slices, (p.T + 16 * MT - 1) / (16 * MT), z);
  adapters_shrink_kernel<MT, RT, BLOCKS><<<grid, 64 * kShrinkWaves, 0, st>>>(p, slice);
}

template <int RC, bool SMALL, int AT>
void expand_few(const QhAdaptersParams& p, int slices, hipStream_t st) {
  adapters_expand_few_kernel<RC, SMALL, AT><<<dim3((p.N + 127) / 128, (p.T + 15) / 16), 256, 0, st>>>(p, slices);
}

template <int MT, int RC, bool SMALL, int CG>
void expand(const QhAdaptersParams& p, int slices, hipStream_t st) {
  const int cols = 256 * CG;
  adapters_expand_kernel<MT, RC, SMALL, CG><<<dim3((p.N + cols - 1) / cols, (p.T + 16 * MT - 1) / (16 * MT)), 512, 0, st>>>(p, slices);
}

}  // namespace

size_t qh_adapters_ws_bytes(int max_tokens, int R) {
  // the most that max_slices(T) * T is for any T up to max_tokens
  const size_t rows = max_tokens <= 2048 ? 8 * (size_t)max_tokens : max_tokens <= 16384 ? 16384 : (size_t)max_tokens;
  return rows * (16 * ((R + 15) / 16)) * sizeof(float);
}

int qh_launch_adapters(const QhAdaptersParams& p, hipStream_t st) {
  const bool few = p.T <= 256;
  const int tiles = (p.T + 15) / 16, wide_tiles = (p.T + 31) / 32;
  // K in slices until there are 512 workgroups, each of eight blocks of 64 at least: a power of two,
  // so that workgroups of a slice meet on the same XCDs (which get them in turn) and find its
  // columns of A in their caches
  // 32 tokens a workgroup read A half as often as 16 (3700 tokens: R 32 13.4 and 16.4 us, R 64 13.4
  // and 17.5); above rank 64 their sums would not leave registers for loads under way
  const bool two = !few && p.R <= 64;
  const int most = min(max_slices(p.T), max(1, min(512 / (two ? wide_tiles : tiles), p.K / 512)));
  int slices = 1;
  while (2 * slices <= most) slices *= 2;
  const int slice = ((p.K + slices - 1) / slices + 63) / 64 * 64;
  slices = (p.K + slice - 1) / slice;
  // Few tokens name an adapter each: one a workgroup; the tiles of long prompts have one, seldom more
  // (3700 tokens: 2, 4 or 8 workgroups a tile take 12.5, 13.6 and 14.4 us).  Between, ids are not known
  // on the host, and 8192 / T lies between its sides.  Both products, N 1024, now / 2 / 4 / 16 workgroups
  // a tile, us:
  //   450 tokens, R 64: 4 runs 11.4 / 10.8 / 10.8 / 10.7, an adapter a token 28 / 45 / 29 / 28; R 128
  //   16.0 / 14.7 / 14.6 / 15.9 and 53 / 53 / 54 / 53;
  //   701 tokens, R 16: 43 runs 10.7 / 10.4 / 9.8 / 9.9, a token 19.3 / 25.7 / 22.7 / 20.9; R 64
  //   15.6 / 16.5 / 15.5 / 15.5 and 40 / 50 / 45 / 39; R 128 4 runs 17.7 / 15.6 / 15.6 / 19.4, a token
  //   81 / 97 / 81 / 83;
  //   2500 tokens, R 64: 156 runs 31 / 32 / 31 / 34, a token 107 / 125 / 105 / 105.
  const int z = max(2, min(min(16, p.T), 8192 / p.T));
  if (two) {
    if (p.R <= 16) shrink<2, 1, 3>(p, slices, slice, z, st);
    else if (p.R <= 32) shrink<2, 2, 2>(p, slices, slice, z, st);
    else shrink<2, 4, 1>(p, slices, slice, z, st);
  } else {
    if (p.R <= 16) shrink<1, 1, 3>(p, slices, slice, z, st);
    else if (p.R <= 32) shrink<1, 2, 2>(p, slices, slice, z, st);
    else if (p.R <= 64) shrink<1, 4, 1>(p, slices, slice, z, st);
    else shrink<1, 8, 1>(p, slices, slice, z, st);
  }

  // B kept in registers while tokens go by, where more than a few name few adapters and 160 pieces of
  // 64 tokens and 512 columns are there; otherwise 16 and 128.  Either side, us, 16 and 128 first:
  //   prompts, N 9216: 450 tokens (144 pieces) R 32 9.9 / 8.8, R 64 13.7 / 14.4; 640 (180) R 16
  //   11.4 / 10.6, R 32 12.2 / 10.6, R 64 17.3 / 15.6, R 128 25.2 / 17.5; 1600 (450) R 32 23.6 / 16.9;
  //   3700 58.9 / 34.8.  N 2560, R 64: 701 tokens (55) 7.6 / 16.4, 3700 (290) 26.8 / 23.9.
  //   300 tokens of 64 adapters, each its own or 40 runs, N 16384: R 32 18.6 / 20.8, R 64 27.6 / 34.3.
  // Adapters at once in the narrow form: as many as leave four waves a SIMD.  Half of them, as they are and
  // twice as many (both products, N 9216, K 512, an adapter a token, us): 48 tokens R 16 11.2 / 11.0 / 11.0,
  // R 32 12.8 / 12.3 / 11.9, R 64 19.1 / 20.2 / 19.9, R 128 28.1 / 29.4 / 30.4; 256 tokens 15.7 / 17.0 / 20.4,
  // 20.5 / 21.9 / 26.7, 47 / 50 / 53, 90 / 95 / 98.
  // Tiles of the wide form at ranks 33 to 64 have five registers too few (24 bytes a thread go to memory).  As
  // they are, of 32 tokens, of 32 columns a wave, and of both (both products, R 64, N 9216, us): 3700 tokens of 4
  // runs 57.5 / 58.5 / 58.2 / 61.7, of 60 70.4 / 72.7 / 67.8 / 72.0; 1600 tokens 31.4 / 33.3 / 31.5 / 33.1 and
  // 40.1 / 46.9 / 41.3 / 43.6; 700 tokens of 4 runs 22.6 / 21.6 / 19.6 / 20.6.
  if (few || ((p.T + 63) / 64) * ((p.N + 511) / 512) < 160) {
    if (p.R <= 16) expand_few<1, true, 8>(p, slices, st);
    else if (p.R <= 32) expand_few<1, false, 8>(p, slices, st);
    else if (p.R <= 64) expand_few<2, false, 4>(p, slices, st);
    else expand_few<4, false, 2>(p, slices, st);
  } else {
    if (p.R <= 16) expand<2, 1, true, 2>(p, slices, st);
    else if (p.R <= 32) expand<2, 1, false, 2>(p, slices, st);
    else if (p.R <= 64) expand<4, 2, false, 2>(p, slices, st);
    else expand<4, 4, false, 1>(p, slices, st);
  }
  return 0;
}
