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
// A wave: 16 MT tokens, 32 CG columns at a time.  The rows of B are the first operand, in an order
// that leaves each lane 8 consecutive columns of one token: of a pair of products, the first has
// columns 8 m + 0 .. 3 and the second 8 m + 4 .. 7 of each eight.  Ranks go 32 to a product, high
// and low parts one after the other; rank 16 (and 8) has both parts in one, side by side.  The rows
// of B of AT adapters are on their way at once, those of y behind them.
template <int MT, int RC, bool SMALL, int CG, int AT>
__global__ __launch_bounds__(256) void adapters_expand_kernel(QhAdaptersParams p, int slices, int cols) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.y * 16 * MT;
  const int Rp = 16 * ((p.R + 15) / 16);
  const TileIds ids(p, t0, 16 * MT);
  // The tile's h, summed over the slices of K, scaled and in two parts, once a workgroup: 4 ranks a
  // thread.  A row's 16 bytes of padding spread the reads below over the banks.
  constexpr int kRow = (SMALL ? 16 : 32 * RC) + 8;
  __shared__ uint16_t s_hi[16 * MT][kRow], s_lo[16 * MT][kRow];
  constexpr int kQuads = SMALL ? 4 : 8 * RC;
  for (int i = threadIdx.x; i < 16 * MT * kQuads; i += 256) {
    const int row = i / kQuads, r = 4 * (i % kQuads), t = t0 + row, a = __shfl(ids.id, row, 64);
    f32x4 u = {0, 0, 0, 0};
    if (a >= 0 && r < p.R) {
      const float* h = p.h + (size_t)t * Rp + r;
      for (int q0 = 0; q0 < slices; q0 += 4) {
        f32x4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = *(const f32x4*)(h + (size_t)min(q0 + q, slices - 1) * p.T * Rp);
#pragma unroll
        for (int q = 0; q < 4; ++q) u += q0 + q < slices ? v[q] : f32x4{0, 0, 0, 0};
      }
      u *= p.scale[a];
    }
    const u32x2 top = {pack_bf2(u.x, u.y), pack_bf2(u.z, u.w)};
    *(u32x2*)&s_hi[row][r] = top;
    *(u32x2*)&s_lo[row][r] = u32x2{pack_bf2(low_part(u.x, bf_lo(top.x)), low_part(u.y, bf_hi(top.x))),
                                   pack_bf2(low_part(u.z, bf_lo(top.y)), low_part(u.w, bf_hi(top.y)))};
  }
  __syncthreads();
  // the lane's token and its 8 ranks of each product
  u32x4 hi[MT][RC], lo[MT][RC];
  int mine[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    mine[m] = __shfl(ids.id, 16 * m + row, 64);
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      const int r0 = SMALL ? 8 * (g & 1) : 32 * c + 8 * g;
      lo[m][c] = *(const u32x4*)&s_lo[16 * m + row][r0];
      hi[m][c] = SMALL && g >= 2 ? lo[m][c] : *(const u32x4*)&s_hi[16 * m + row][r0];
    }
  }
  const u32x4 zero = {0, 0, 0, 0};
  for (int i = 0; i < cols; ++i) {
    const int c0 = ((blockIdx.x * cols + i) * 4 + wid) * 32 * CG;
    if (c0 >= p.N) break;
    f32x4 acc[MT][2 * CG];
    u32x4 y[MT][CG];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int q = 0; q < 2 * CG; ++q) acc[m][q] = f32x4{0, 0, 0, 0};
    TileIds tile = ids;
    bool asked = false;
    do {
      int a[AT], count = 0;
      u32x4 b[AT][RC][2 * CG];
#pragma unroll
      for (int n = 0; n < AT; ++n) {
        if (n > 0 && tile.left == 0) continue;
        uint64_t tokens;
        a[n] = tile.left != 0 ? tile.next(tokens) : 0;
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
      if (!asked) {
        asked = true;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int q = 0; q < CG; ++q) {
            const int t = min(t0 + 16 * m + row, p.T - 1), c = c0 + 32 * q + 8 * g;
            y[m][q] = c < p.N ? load16(p.y + t * p.y_ts + c) : zero;
          }
      }
#pragma unroll
      for (int n = 0; n < AT; ++n) {
        if (n >= count) continue;
        f32x4 d[MT][2 * CG];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int q = 0; q < 2 * CG; ++q) {
            d[m][q] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < RC; ++c) {
              d[m][q] = mfma(b[n][c][q], hi[m][c], d[m][q]);
              if (!SMALL) d[m][q] = mfma(b[n][c][q], lo[m][c], d[m][q]);
            }
            if (mine[m] == a[n]) acc[m][q] = d[m][q];
          }
      }
    } while (tile.left != 0);
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
}

// Slices of K whose partial sums the workspace holds.
int max_slices(int T) { return T <= 2048 ? 8 : T <= 16384 ? 16384 / T : 1; }

template <int MT, int RT, int BLOCKS>
void shrink(const QhAdaptersParams& p, int slices, int slice, int z, hipStream_t st) {
  const dim3 grid(slices, (p.T + 16 * MT - 1) / (16 * MT), z);
  adapters_shrink_kernel<MT, RT, BLOCKS><<<grid, 64 * kShrinkWaves, 0, st>>>(p, slice);
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
  // K in slices until there are 512 workgroups, of a block a wave at least
  const int step = 64 * kShrinkWaves, steps = (p.K + step - 1) / step;
  const bool two = !few && p.R <= 64;
  int slices = min(max_slices(p.T), max(1, min(512 / (two ? wide_tiles : tiles), steps)));
  const int slice = (steps + slices - 1) / slices * step;
  slices = (p.K + slice - 1) / slice;
  // few tokens name an adapter each: one a workgroup; of prompts a tile has one, seldom more
  const int z = few ? min(16, p.T) : 4;
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

  // 32 tokens and 256 columns a workgroup at a time where that leaves four workgroups a CU, and then
  // up to four times; otherwise 16 and 128
  const int wide1 = (p.N + 255) / 256, cols = min(4, wide_tiles * wide1 / 1024);
  if (cols == 0) {
    const dim3 grid((p.N + 127) / 128, tiles);
    if (p.R <= 16) adapters_expand_kernel<1, 1, true, 1, 8><<<grid, 256, 0, st>>>(p, slices, 1);
    else if (p.R <= 32) adapters_expand_kernel<1, 1, false, 1, 8><<<grid, 256, 0, st>>>(p, slices, 1);
    else if (p.R <= 64) adapters_expand_kernel<1, 2, false, 1, 4><<<grid, 256, 0, st>>>(p, slices, 1);
    else adapters_expand_kernel<1, 4, false, 1, 2><<<grid, 256, 0, st>>>(p, slices, 1);
  } else {
    const dim3 grid((wide1 + cols - 1) / cols, wide_tiles);
    if (p.R <= 16) adapters_expand_kernel<2, 1, true, 2, 1><<<grid, 256, 0, st>>>(p, slices, cols);
    else if (p.R <= 32) adapters_expand_kernel<2, 1, false, 2, 1><<<grid, 256, 0, st>>>(p, slices, cols);
    else if (p.R <= 64) adapters_expand_kernel<2, 2, false, 2, 1><<<grid, 256, 0, st>>>(p, slices, cols);
    else adapters_expand_kernel<2, 4, false, 2, 1><<<grid, 256, 0, st>>>(p, slices, cols);
  }
  return 0;
}
