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
// Bound by bytes: A and B of the adapters in use (decode), x, y and out (prompts).
//
// h stays in fp32 between the launches and enters the second product as two bf16 numbers,
// high and low, which together lose 2^-16 of it: one rounding would cost as much as the
// rounding of the output.  Products and sums are fp32, the output is rounded once.
#include "qh_common.h"
#include "qh_serve.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ u32x4 load16(const uint16_t* p) { return *(const u32x4*)p; }

// What the high part leaves of x: nothing of an infinity.
__device__ __forceinline__ float low_part(float x, float high) { return fabsf(high) < INFINITY ? x - high : 0.0f; }

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
// A wave: 16 MT tokens and 32 CG columns; WAVES of them side by side share the tile's h.  The rows of B
// are the first operand, in an order that leaves each lane 8 consecutive columns of one token: of a
// pair of products, the first has columns 8 m + 0 .. 3 and the second 8 m + 4 .. 7 of each eight.
// Ranks go 32 to a product, high and low parts one after the other; rank 16 (and 8) has both parts in
// one, side by side.  The rows of B of AT adapters are on their way at once.
// Of eight waves two workgroups fit a CU where a wave takes 128 registers at most.
template <int WAVES, int MT, int RC, bool SMALL, int CG, int AT>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 ? 4 : 1) void adapters_expand_kernel(QhAdaptersParams p, int slices) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.y * 16 * MT, c0 = (blockIdx.x * WAVES + wid) * 32 * CG;
  const int Rp = 16 * ((p.R + 15) / 16);
  const u32x4 zero = {0, 0, 0, 0};
  TileIds tile(p, t0, 16 * MT);
  const int token_id = tile.id;

  int a[AT], count;
  u32x4 b[AT][RC][2 * CG];
  auto load_b = [&]() {
    count = 0;
#pragma unroll
    for (int n = 0; n < AT; ++n) {
      if (tile.left == 0) continue;
      uint64_t tokens;
      a[n] = tile.next(tokens);
      count = n + 1;
#pragma unroll
      for (int c = 0; c < RC; ++c) {
        const int r0 = SMALL ? 8 * (g & 1) : 32 * c + 8 * g;
#pragma unroll
        for (int q = 0; q < 2 * CG; ++q) {
          const int col = min(c0 + 32 * (q / 2) + 8 * (row >> 2) + 4 * (q % 2) + (row & 3), p.N - 1);
          b[n][c][q] = r0 < p.R ? load16(p.b + ((size_t)a[n] * p.N + col) * p.R + r0) : zero;
        }
      }
    }
  };
  u32x4 y[MT][CG];
  auto load_y = [&]() {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int q = 0; q < CG; ++q) {
        const int t = min(t0 + 16 * m + row, p.T - 1), c = c0 + 32 * q + 8 * g;
        y[m][q] = c < p.N ? load16(p.y + t * p.y_ts + c) : zero;
      }
  };
  // Few tokens wait for B most: it goes first, y behind it.  Of a prompt y is most of the bytes, and h
  // would wait behind it (loads come back in order): 3700 tokens 44 us against 35.
  constexpr bool kEarly = AT > 1;
  if (kEarly) {
    load_b();
    load_y();
  }

  // The tile's h, summed over the slices of K, scaled and in two parts, once a workgroup: 4 ranks a
  // thread.  A row's 16 bytes of padding spread the reads below over the banks.
  constexpr int kRow = (SMALL ? 16 : 32 * RC) + 8;
  __shared__ uint16_t s_hi[16 * MT][kRow], s_lo[16 * MT][kRow];
  constexpr int kQuads = SMALL ? 4 : 8 * RC;
  for (int i = threadIdx.x; i < 16 * MT * kQuads; i += 64 * WAVES) {
    const int tr = i / kQuads, r = 4 * (i % kQuads), t = t0 + tr, id = __shfl(token_id, tr, 64);
    f32x4 u = {0, 0, 0, 0};
    if (id >= 0 && r < p.R) {
      const float* h = p.h + (size_t)t * Rp + r;
      for (int q0 = 0; q0 < slices; q0 += 4) {
        f32x4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = *(const f32x4*)(h + (size_t)min(q0 + q, slices - 1) * p.T * Rp);
#pragma unroll
        for (int q = 0; q < 4; ++q) u += q0 + q < slices ? v[q] : f32x4{0, 0, 0, 0};
      }
      u *= p.scale[id];
    }
    const u32x2 top = {pack_bf2(u.x, u.y), pack_bf2(u.z, u.w)};
    *(u32x2*)&s_hi[tr][r] = top;
    *(u32x2*)&s_lo[tr][r] = u32x2{pack_bf2(low_part(u.x, bf_lo(top.x)), low_part(u.y, bf_hi(top.x))),
                                  pack_bf2(low_part(u.z, bf_lo(top.y)), low_part(u.w, bf_hi(top.y)))};
  }
  __syncthreads();
  if (c0 >= p.N) return;
  if (!kEarly) {
    load_b();
    load_y();
  }
  // the lane's token and its 8 ranks of each product
  u32x4 hi[MT][RC], lo[MT][RC];
  int mine[MT];
  f32x4 acc[MT][2 * CG];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    mine[m] = __shfl(token_id, 16 * m + row, 64);
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      const int r0 = SMALL ? 8 * (g & 1) : 32 * c + 8 * g;
      lo[m][c] = *(const u32x4*)&s_lo[16 * m + row][r0];
      hi[m][c] = SMALL && g >= 2 ? lo[m][c] : *(const u32x4*)&s_hi[16 * m + row][r0];
    }
  }
  auto product = [&](int n, int m, int q) {
    f32x4 d = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      d = mfma(b[n][c][q], hi[m][c], d);
      if (!SMALL) d = mfma(b[n][c][q], lo[m][c], d);
    }
    return d;
  };
  // The first adapter's product is everybody's at first (and nobody's who has none: such rows are copied).
  bool others = false;
  while (count > 0) {
#pragma unroll
    for (int n = 0; n < AT; ++n) {
      if (n >= count) continue;
      if (n == 0 && !others) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int q = 0; q < 2 * CG; ++q) acc[m][q] = product(n, m, q);
        others = true;
        continue;
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < 2 * CG; ++q) {
          const f32x4 d = product(n, m, q);
          if (mine[m] == a[n]) acc[m][q] = d;
        }
    }
    load_b();
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int q = 0; q < CG; ++q) {
      const int t = t0 + 16 * m + row, c = c0 + 32 * q + 8 * g;
      if (t >= p.T || c >= p.N || (mine[m] < 0 && p.out == p.y)) continue;
      u32x4 z = y[m][q];
      if (mine[m] >= 0) {  // a row without an adapter is copied as it is
        const f32x4 u = acc[m][2 * q], v = acc[m][2 * q + 1];
        z = u32x4{pack_bf2(bf_lo(z.x) + u.x, bf_hi(z.x) + u.y), pack_bf2(bf_lo(z.y) + u.z, bf_hi(z.y) + u.w),
                  pack_bf2(bf_lo(z.z) + v.x, bf_hi(z.z) + v.y), pack_bf2(bf_lo(z.w) + v.z, bf_hi(z.w) + v.w)};
      }
      *(u32x4*)(p.out + t * p.out_ts + c) = z;
    }
}

// Slices of K whose partial sums the workspace holds.
int max_slices(int T) { return T <= 2048 ? 8 : T <= 16384 ? 16384 / T : 1; }

template <int MT, int RT, int BLOCKS>
void shrink(const QhAdaptersParams& p, int slices, int slice, int z, hipStream_t st) {
  const dim3 grid(slices, (p.T + 16 * MT - 1) / (16 * MT), z);
  adapters_shrink_kernel<MT, RT, BLOCKS><<<grid, 64 * kShrinkWaves, 0, st>>>(p, slice);
}

template <int WAVES, int MT, int RC, bool SMALL, int CG, int AT>
void expand(const QhAdaptersParams& p, int slices, hipStream_t st) {
  const int cols = 32 * CG * WAVES;
  const dim3 grid((p.N + cols - 1) / cols, (p.T + 16 * MT - 1) / (16 * MT));
  adapters_expand_kernel<WAVES, MT, RC, SMALL, CG, AT><<<grid, 64 * WAVES, 0, st>>>(p, slices);
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
  const bool two = !few && p.R <= 64;
  const int most = min(max_slices(p.T), max(1, min(512 / (two ? wide_tiles : tiles), p.K / 512)));
  int slices = 1;
  while (2 * slices <= most) slices *= 2;
  const int slice = ((p.K + slices - 1) / slices + 63) / 64 * 64;
  slices = (p.K + slice - 1) / slice;
  // few tokens name an adapter each: one a workgroup; the tiles of long prompts have one, seldom more
  const int z = max(2, min(min(16, p.T), 8192 / p.T));
  if (two) {
    if (p.R <= 16) shrink<2, 1, 3>(p, slices, slice, z, st);
    else if (p.R <= 32) shrink<2, 2, 2>(p, slices, slice, z, st);
    else shrink<2, 4, 2>(p, slices, slice, z, st);
  } else {
    if (p.R <= 16) shrink<1, 1, 3>(p, slices, slice, z, st);
    else if (p.R <= 32) shrink<1, 2, 2>(p, slices, slice, z, st);
    else if (p.R <= 64) shrink<1, 4, 1>(p, slices, slice, z, st);
    else shrink<1, 8, 1>(p, slices, slice, z, st);
  }

  // 32 tokens and 512 columns a workgroup where that leaves two of them a CU, otherwise 16 and 128
  if (wide_tiles * ((p.N + 511) / 512) < 512) {
    if (p.R <= 16) expand<4, 1, 1, true, 1, 8>(p, slices, st);
    else if (p.R <= 32) expand<4, 1, 1, false, 1, 8>(p, slices, st);
    else if (p.R <= 64) expand<4, 1, 2, false, 1, 4>(p, slices, st);
    else expand<4, 1, 4, false, 1, 2>(p, slices, st);
  } else {
    if (p.R <= 16) expand<8, 2, 1, true, 2, 1>(p, slices, st);
    else if (p.R <= 32) expand<8, 2, 1, false, 2, 1>(p, slices, st);
    else if (p.R <= 64) expand<8, 2, 2, false, 1, 1>(p, slices, st);
    else expand<4, 2, 4, false, 1, 1>(p, slices, st);
  }
  return 0;
}
