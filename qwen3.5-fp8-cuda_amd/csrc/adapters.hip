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
// A workgroup: 16 tokens, one slice of K, the tile's adapters z, z + gridDim.z, ...  Its four
// waves take the slice's blocks of 64 in turn and add up through LDS.  Per block a lane loads
// 32 bytes of its row of x and of A (128 bytes a row and wave: whole cache lines); which 8 of
// a block's 64 go into which product is the same for both operands, and free.
template <int RT>  // tiles of 16 ranks
__global__ __launch_bounds__(256) void adapters_shrink_kernel(QhAdaptersParams p, int slice) {
  __shared__ f32x4 s_part[4][RT][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.y * 16, k0 = blockIdx.x * slice, k1 = min(p.K, k0 + slice);
  TileIds tile(p, t0, 16);
  const uint16_t* xr = p.x + (long long)min(t0 + row, p.T - 1) * p.x_ts;
  const int Rp = 16 * ((p.R + 15) / 16);
  const u32x4 zero = {0, 0, 0, 0};
  for (int j = 0; tile.left != 0; ++j) {
    uint64_t mine;
    const int a = tile.next(mine);
    if (j % gridDim.z != blockIdx.z) continue;
    const uint16_t* ar[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) ar[r] = p.a + ((size_t)a * p.R + min(16 * r + row, p.R - 1)) * p.K;
    f32x4 acc[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[r] = f32x4{0, 0, 0, 0};
    for (int k = k0 + 64 * wid; k < k1; k += 256) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int c = k + 16 * g + 8 * half;
        const bool in = c < k1;
        const u32x4 x = in ? load16(xr + c) : zero;
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r] = mfma(in ? load16(ar[r] + c) : zero, x, acc[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) s_part[wid][r][lane] = acc[r];
    __syncthreads();
    // lane: token row, ranks 16 r + 4 g .. + 3
    for (int r = wid; r < RT; r += 4) {
      const f32x4 s = (s_part[0][r][lane] + s_part[1][r][lane]) + (s_part[2][r][lane] + s_part[3][r][lane]);
      if ((mine >> row) & 1 && 16 * r < Rp)
        *(f32x4*)(p.h + ((size_t)blockIdx.x * p.T + t0 + row) * Rp + 16 * r + 4 * g) = s;
    }
    __syncthreads();
  }
}

// ---- out = y + scale B h -------------------------------------------------------------------
// A wave: 16 MT tokens, 32 columns at a time.  The rows of B are the first operand, in an order
// that leaves each lane 8 consecutive columns of one token: of a pair of products, the first has
// columns 8 m + 0 .. 3 and the second 8 m + 4 .. 7 of each eight.  Ranks go 32 to a product, high
// and low parts one after the other; rank 16 (and 8) has both parts in one, side by side.
template <int MT, int RC, bool SMALL>
__global__ __launch_bounds__(256) void adapters_expand_kernel(QhAdaptersParams p, int slices, int cols) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.y * 16 * MT;
  const int Rp = 16 * ((p.R + 15) / 16);
  const TileIds ids(p, t0, 16 * MT);
  // the tokens' h, scaled: the lane's token and its 8 ranks of each product
  u32x4 hi[MT][RC], lo[MT][RC];
  int mine[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    mine[m] = __shfl(ids.id, 16 * m + row, 64);
    const int t = t0 + 16 * m + row;
    const float s = mine[m] >= 0 ? p.scale[mine[m]] : 0.0f;
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      const int r0 = SMALL ? 8 * (g & 1) : 32 * c + 8 * g;
      f32x4 u = {0, 0, 0, 0}, v = u;
      if (mine[m] >= 0 && r0 < p.R) {
        const float* h = p.h + (size_t)t * Rp + r0;
        for (int i = 0; i < slices; ++i) {
          u += *(const f32x4*)(h + (size_t)i * p.T * Rp);
          v += *(const f32x4*)(h + (size_t)i * p.T * Rp + 4);
        }
      }
      u *= s;
      v *= s;
      const u32x4 top = {pack_bf2(u.x, u.y), pack_bf2(u.z, u.w), pack_bf2(v.x, v.y), pack_bf2(v.z, v.w)};
      const u32x4 rest = {pack_bf2(low_part(u.x, bf_lo(top.x)), low_part(u.y, bf_hi(top.x))),
                          pack_bf2(low_part(u.z, bf_lo(top.y)), low_part(u.w, bf_hi(top.y))),
                          pack_bf2(low_part(v.x, bf_lo(top.z)), low_part(v.y, bf_hi(top.z))),
                          pack_bf2(low_part(v.z, bf_lo(top.w)), low_part(v.w, bf_hi(top.w)))};
      hi[m][c] = SMALL && g >= 2 ? rest : top;
      lo[m][c] = rest;
    }
  }
  const u32x4 zero = {0, 0, 0, 0};
  for (int i = 0; i < cols; ++i) {
    const int c0 = ((blockIdx.x * cols + i) * 4 + wid) * 32;
    if (c0 >= p.N) break;
    f32x4 acc[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = f32x4{0, 0, 0, 0};
    TileIds tile = ids;
    while (tile.left != 0) {
      uint64_t tokens;
      const int a = tile.next(tokens);
      f32x4 d[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) d[m][0] = d[m][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < RC; ++c) {
        const int r0 = SMALL ? 8 * (g & 1) : 32 * c + 8 * g;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int col = min(c0 + 8 * (row >> 2) + 4 * half + (row & 3), p.N - 1);
          const u32x4 b = r0 < p.R ? load16(p.b + ((size_t)a * p.N + col) * p.R + r0) : zero;
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            d[m][half] = mfma(b, hi[m][c], d[m][half]);
            if (!SMALL) d[m][half] = mfma(b, lo[m][c], d[m][half]);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if (mine[m] == a) {
          acc[m][0] = d[m][0];
          acc[m][1] = d[m][1];
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int t = t0 + 16 * m + row, c = c0 + 8 * g;
      if (t >= p.T || c >= p.N || (mine[m] < 0 && p.out == p.y)) continue;
      u32x4 y = load16(p.y + t * p.y_ts + c);
      if (mine[m] >= 0) {  // a row without an adapter is copied as it is
        const f32x4 u = acc[m][0], v = acc[m][1];
        y = u32x4{pack_bf2(bf_lo(y.x) + u.x, bf_hi(y.x) + u.y), pack_bf2(bf_lo(y.y) + u.z, bf_hi(y.y) + u.w),
                  pack_bf2(bf_lo(y.z) + v.x, bf_hi(y.z) + v.y), pack_bf2(bf_lo(y.w) + v.z, bf_hi(y.w) + v.w)};
      }
      *(u32x4*)(p.out + t * p.out_ts + c) = y;
    }
  }
}

// Slices of K whose partial sums the workspace holds.
int max_slices(int T) { return T <= 1024 ? 8 : T <= 8192 ? 8192 / T : 1; }

}  // namespace

size_t qh_adapters_ws_bytes(int max_tokens, int R) {
  // the most that max_slices(T) * T is for any T up to max_tokens
  const size_t rows = max_tokens <= 1024 ? 8 * (size_t)max_tokens : max_tokens <= 8192 ? 8192 : (size_t)max_tokens;
  return rows * (16 * ((R + 15) / 16)) * sizeof(float);
}

int qh_launch_adapters(const QhAdaptersParams& p, hipStream_t st) {
  const int tiles = (p.T + 15) / 16;
  // K in slices until there are 512 workgroups, of 512 columns at least: two blocks a wave
  int slices = min(max_slices(p.T), max(1, min(512 / tiles, (p.K + 511) / 512)));
  const int slice = ((p.K + slices - 1) / slices + 255) / 256 * 256;
  slices = (p.K + slice - 1) / slice;
  // few tokens name an adapter each: one a workgroup
  const int z = p.T <= 256 ? min(16, p.T) : 1;
  const dim3 grid(slices, tiles, z);
  if (p.R <= 16) adapters_shrink_kernel<1><<<grid, 256, 0, st>>>(p, slice);
  else if (p.R <= 32) adapters_shrink_kernel<2><<<grid, 256, 0, st>>>(p, slice);
  else if (p.R <= 64) adapters_shrink_kernel<4><<<grid, 256, 0, st>>>(p, slice);
  else adapters_shrink_kernel<8><<<grid, 256, 0, st>>>(p, slice);

  const int cols = p.T <= 256 ? 1 : 4;
  const dim3 wide((p.N + 128 * cols - 1) / (128 * cols), p.T <= 256 ? tiles : (p.T + 63) / 64);
  if (p.T <= 256) {
    if (p.R <= 16) adapters_expand_kernel<1, 1, true><<<wide, 256, 0, st>>>(p, slices, cols);
    else if (p.R <= 32) adapters_expand_kernel<1, 1, false><<<wide, 256, 0, st>>>(p, slices, cols);
    else if (p.R <= 64) adapters_expand_kernel<1, 2, false><<<wide, 256, 0, st>>>(p, slices, cols);
    else adapters_expand_kernel<1, 4, false><<<wide, 256, 0, st>>>(p, slices, cols);
  } else {
    if (p.R <= 16) adapters_expand_kernel<4, 1, true><<<wide, 256, 0, st>>>(p, slices, cols);
    else if (p.R <= 32) adapters_expand_kernel<4, 1, false><<<wide, 256, 0, st>>>(p, slices, cols);
    else if (p.R <= 64) adapters_expand_kernel<4, 2, false><<<wide, 256, 0, st>>>(p, slices, cols);
    else adapters_expand_kernel<4, 4, false><<<wide, 256, 0, st>>>(p, slices, cols);
  }
  return 0;
}
