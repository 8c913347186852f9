// Decode attention over a paged KV cache (gfx950): one new token of each sequence
// of a batch, GQA, rows in bf16 or in E4M3 with a scale per row.  No counterpart in
// the reference, whose decode attention reads one dense bf16 cache (layer_mid_attn,
// qwen3_infer/csrc/fused_kernels.cu:1224-1297).
//
//   s_j = q_h . k_j / sqrt(D),  o_h = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max_j s_j,
//   over positions j = 0 .. last[b] on pages that exist;  out_h = bf16(o_h sigmoid(gate_h)),
//   zeros where no position is visible.
//
// Every visible row of K and V is read once: HBM bounds it from a few MB on, latency
// below.  The query heads of a KV head (at most 16) are the columns of 16 x 16 x 32 bf16
// matrix products, so the arithmetic of one head and of 16 is the same and stays out
// of the way.  A wave takes tiles of 32 positions with nothing but its registers:
//   S^T = K Q^T : A = 16 rows of K as they lie in memory (lane (r, g) = (l % 16, l / 16)
//     holds 8 dims of row r), twice a tile.  Row m of product a is position
//     8 (m / 4) + 4 a + m % 4, which leaves lane (r, g) with the scores of head r at
//     positions 8 g .. 8 g + 7 ...
//   O^T = V^T P^T : ... which is what the B operand asks of it.  A = V^T: the lane loads
//     16 bytes or so of each of its 8 positions' rows (whole rows of 128 to 512 bytes to a
//     16-lane group) and gathers the same element of all 8 by byte permutes.
// E4M3 rows widen exactly to bf16; their scales multiply the score (K) and the weight
// (V).  Weights enter the product as the sum of two bf16 numbers (2^-17 of them is
// lost, as against 2^-9 with one, for matrix instructions that have time to spare).
// Scores, maxima, sums and outputs are fp32.  The maximum follows with a slack of 2^8:
// weights up to 256 lose nothing in fp32, and a tile whose scores stay below that
// needs no exchange between lanes and no rescaling.
//
// Work split: the tiles (32 positions of one KV head of one sequence) of the whole
// batch form one line, cut into equal shares of consecutive tiles, one a workgroup (one
// workgroup per CU), so ragged batches load all CUs alike; a share's tiles go round its
// waves in turn wherever sequences end.  The rows of a wave's next tile are on their way
// while it computes, across sequences too, and the page ids of the one after.  A
// (sequence, KV head) inside one share is written out; one that several shares cut
// leaves a partial record a piece (maximum, sum, outputs), and the last piece to arrive
// joins them in their order: the result does not depend on who comes last.
#include <type_traits>

#include "qh_common.h"
#include "qh_paged.h"

namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 32;                    // positions per wave and step
constexpr int kMaxWG = 256;                  // workgroups that hold a share
constexpr int kMaxG = 16;
constexpr int kWhole = 3 * kWaves;           // tiles of a pair that one workgroup takes rather than join pieces

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

// Four E4M3 bytes as two words of two bf16 each.
__device__ __forceinline__ uint32_t widen_lo(uint32_t x) { return __builtin_bit_cast(uint32_t, e4m3x2_lo_bf16(x)); }
__device__ __forceinline__ uint32_t widen_hi(uint32_t x) { return __builtin_bit_cast(uint32_t, e4m3x2_hi_bf16(x)); }

// Sixteen bytes that another workgroup published (device-coherent): two 8-byte atomic
// loads, which the compiler keeps independent of each other.
__device__ __forceinline__ u32x4 coherent_load(const float* src) {
  uint64_t* s = (uint64_t*)const_cast<float*>(src);
  const uint64_t a = __hip_atomic_load(s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint64_t b = __hip_atomic_load(s + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return u32x4{(uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32)};
}

// What a wave holds of one tile.
template <int D, bool FP8>
struct Tile {
  static constexpr int KL = FP8 ? D / 64 : D / 32;   // 16-byte loads of K a row
  static constexpr int VD = FP8 ? D / 64 : D / 32;   // dwords of V a lane and position
  u32x4 k[2][KL];
  uint32_t v[8][VD];
  f32x4 ks[2], vs[2];                                // scales of positions 8 g .. 8 g + 7
};

// Rows of a record: [G][D] outputs, [16] maxima, [16] sums.
__host__ __device__ constexpr int rec_floats(int G, int D) { return G * D + 2 * kMaxG; }

// LDS bytes: the waves' outputs (and the joining of pieces, which comes after them),
// the query rows, per sequence its positions and the running sum of tiles.
constexpr int head_floats(int D) { return D + 4; }   // between heads: no bank conflict
constexpr int q_stride(int D) { return D + 8; }      // between query rows (bf16)
size_t lds_bytes(int G, int D, int B) {
  const size_t outs = (size_t)kWaves * G * head_floats(D) * 4, join = (size_t)2 * kMaxWG * G * 4 + kThreads * 16;
  return (outs > join ? outs : join) + (size_t)kMaxG * q_stride(D) * 2 + (size_t)B * 8;
}

// A tile on the line: its sequence and KV head, and the tiles [u0, u1) of that pair.
struct Place {
  int k, b, kvh, u0, u1, n;
};

// A pair that several workgroups hold pieces of: the first of them, and whether its
// piece is the second record there.
struct Pair {
  int b, kvh, pieces, first, tail;
};

__device__ __forceinline__ int wave_imax(int v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, __shfl_xor(v, d, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_isum(int v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  return __builtin_amdgcn_readfirstlane(v);
}

template <int D, bool FP8>
__global__ __launch_bounds__(kThreads, 2) void paged_attn_kernel(QhPagedAttnParams p) {
  using T = Tile<D, FP8>;
  constexpr int DT = D / 16;                         // 16-dim tiles of the output
  constexpr int HS = D + 4, QS = D + 8;
  __shared__ int s_tot[kWaves];
  __shared__ float s_m[kWaves][kMaxG], s_l[kWaves][kMaxG];
  __shared__ float s_sum[kMaxG];
  __shared__ int s_last[2];
  extern __shared__ __align__(16) float s_o[];       // [kWaves][G][HS]

  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int B = p.c.n_seqs, Hkv = p.c.n_kv, G = p.n_heads / Hkv, ps = p.c.page_size;
  const int wg = blockIdx.x;
  const int out_floats = kWaves * G * HS, join_floats = 2 * kMaxWG * G + kThreads * 4;
  uint16_t* s_q = (uint16_t*)(s_o + (out_floats > join_floats ? out_floats : join_floats));  // [kMaxG][QS]
  int* s_n = (int*)(s_q + kMaxG * QS);               // [B] positions of sequence b
  int* s_cum = s_n + B;                              // [B] tiles (of one KV head) of sequences 0 .. b

  // ---- this workgroup's part of the work: tiles [start, end) from `seg` on ---------------
  Place seg;
  int start = 0, end = 0, share = 0, w0 = -1;        // w0 >= 0: pieces of one pair, the first of them here
  int pieces = 0;
  auto zeros = [&](int b) {                          // an empty sequence
    for (int i = tid; i < p.n_heads * D / 8; i += kThreads)
      *(u32x4*)(p.out + (size_t)b * p.n_heads * D + i * 8) = u32x4{0u, 0u, 0u, 0u};
  };
  auto tiles_to = [&](int b) { return b < 0 ? 0 : __builtin_amdgcn_readfirstlane(s_cum[b]); };
  bool by_pair = false;
  int n_lane = 0;
  if (B <= 64) {
    // Few sequences: lane b of every wave has sequence b, nothing goes through LDS.
    n_lane = lane < B ? max(min(p.last[lane], p.c.capacity - 1) + 1, 0) : 0;
    const int tl = (n_lane + kTile - 1) / kTile, most = wave_imax(tl), sum = wave_isum(tl);
    const int slots = (int)gridDim.x / Hkv;
    if (most <= kWhole && B <= slots) share = kWhole;
    else if (4 * B <= slots) share = max(kWaves, (sum + slots - B - 1) / (slots - B));
    by_pair = share > 0;
    if (by_pair) {
      share = (share + kWaves - 1) / kWaves * kWaves;
      const int pc = (tl + share - 1) / share;
      int cum = pc;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(cum, d, 64);
        cum += lane >= d ? v : 0;
      }
      for (int b = wg; b < B; b += gridDim.x)
        if (__builtin_amdgcn_readlane(n_lane, b) == 0) zeros(b);
      const unsigned long long past = __ballot(cum * Hkv > wg);
      if (past == 0) return;
      seg.b = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
      seg.n = __builtin_amdgcn_readlane(n_lane, seg.b);
      pieces = __builtin_amdgcn_readlane(pc, seg.b);
      const int i = wg - (__builtin_amdgcn_readlane(cum, seg.b) - pieces) * Hkv;
      seg.kvh = i / pieces;
      const int j = i - seg.kvh * pieces;
      w0 = wg - j;
      seg.u0 = 0;
      seg.u1 = (seg.n + kTile - 1) / kTile;
      start = seg.k = j * share;
      end = min(seg.u1, start + share);
    }
  }
  if (!by_pair) {
    // the line of all tiles: a running sum over the sequences, in LDS
    const int per = (B + kThreads - 1) / kThreads, b0 = tid * per;
    int mine = 0;
    for (int i = 0; i < per; ++i) {
      const int b = b0 + i;
      if (b < B) {
        const int n = max(min(p.last[b], p.c.capacity - 1) + 1, 0);
        mine += (n + kTile - 1) / kTile;
        s_n[b] = n;
        s_cum[b] = mine;
      }
    }
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(sum, d, 64);
      sum += lane >= d ? v : 0;
    }
    if (lane == 63) s_tot[wid] = sum;
    __syncthreads();
    int before = sum - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      before += w < wid ? s_tot[w] : 0;
      all += s_tot[w];
    }
    for (int i = 0; i < per; ++i)
      if (b0 + i < B) s_cum[b0 + i] += before;
    const int total = __builtin_amdgcn_readfirstlane(all) * Hkv;
    __syncthreads();
    share = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    share = max(kWaves, (share + kWaves - 1) / kWaves * kWaves);
    for (int b = wg; b < B; b += gridDim.x)
      if (s_n[b] == 0) zeros(b);
    start = wg * share;
    end = min(total, start + share);
    if (start >= end) return;
    int lo = 0, hi = B - 1;  // the sequence of tile `start`: the first whose running sum passes it
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (tiles_to(mid) * Hkv > start) hi = mid;
      else lo = mid + 1;
    }
    const int first = tiles_to(lo - 1), tiles = tiles_to(lo) - first;
    seg.k = start;
    seg.b = lo;
    seg.kvh = (start - first * Hkv) / tiles;
    seg.u0 = first * Hkv + seg.kvh * tiles;
    seg.u1 = seg.u0 + tiles;
    seg.n = __builtin_amdgcn_readfirstlane(s_n[lo]);
  }
  // The pair that holds tile k >= c.u0 of the line, from c on.
  auto walk = [&](Place c, int k) {
    c.k = k;
    while (k >= c.u1) {
      if (++c.kvh == Hkv) {
        c.kvh = 0;
        do ++c.b; while (tiles_to(c.b) == tiles_to(c.b - 1));
        c.n = __builtin_amdgcn_readfirstlane(s_n[c.b]);
      }
      c.u0 = c.u1;
      c.u1 += (c.n + kTile - 1) / kTile;
    }
    return c;
  };
  const float qscale = (D == 256 ? 0.0625f : 0.08838834764831845f) * 1.4426950408889634f;  // log2(e) / sqrt(D)

  // Page ids and slots of the lane's two groups of 8 positions (K: r / 4, V: g) of a tile.
  // A group behind the last position takes the one that holds it.  A wave without a next
  // tile asks for page 0's first rows, which the caches have: a load under a branch
  // would make the compiler wait for V where K is needed.
  struct Ids { int kid, vid, koff, voff; };
  auto ids_of = [&](const Place& c) {
    const int t0 = (c.k - c.u0) * kTile, lastgrp = (c.n - 1) & ~7;
    const int* pages = p.c.pages + (size_t)c.b * p.c.max_pages;
    Ids x;
    const int kp = min(t0 + 8 * (r >> 2), lastgrp), vp = min(t0 + 8 * g, lastgrp);
    const int kq = page_of(p.c, kp), vq = page_of(p.c, vp);
    x.kid = pages[kq];
    x.vid = pages[vq];
    x.koff = kp - kq * ps;
    x.voff = vp - vq * ps;
    return x;
  };
  auto row_of = [&](const Place& c, int id, int off) {
    const bool ok = c.k < end;
    return ((long long)(ok && (unsigned)id < (unsigned)p.c.n_pages ? id : 0) * Hkv + c.kvh) * ps + (ok ? off : 0);
  };
  T t;
  auto load_k = [&](const Place& c, const Ids& x) {
    const long long row = row_of(c, x.kid, x.koff) + (r & 3);
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const char* src = (const char*)p.c.k + (row + 4 * a) * (FP8 ? D : 2 * D) + 16 * g;
#pragma unroll
      for (int j = 0; j < T::KL; ++j) t.k[a][j] = *(const u32x4*)(src + 64 * j);
    }
    if constexpr (FP8) {
      const long long vrow = row_of(c, x.vid, x.voff);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        t.ks[a] = *(const f32x4*)(p.c.ks + vrow + 4 * a);
        t.vs[a] = *(const f32x4*)(p.c.vs + vrow + 4 * a);
      }
    }
  };
  auto load_v = [&](const Place& c, const Ids& x) {
    const char* src = (const char*)p.c.v + row_of(c, x.vid, x.voff) * (FP8 ? D : 2 * D);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const char* s = src + i * (FP8 ? D : 2 * D);
      if constexpr (T::VD == 2) {
        const u32x2 w = *(const u32x2*)(s + 8 * r);
        t.v[i][0] = w.x; t.v[i][1] = w.y;
      } else {
#pragma unroll
        for (int j = 0; j < T::VD / 4; ++j) {
          const u32x4 w = *(const u32x4*)(s + 16 * (r + 16 * j));
          t.v[i][4 * j] = w.x; t.v[i][4 * j + 1] = w.y; t.v[i][4 * j + 2] = w.z; t.v[i][4 * j + 3] = w.w;
        }
      }
    }
  };
  // The 16 bytes of a pair's query rows that this thread moves to LDS (rows above G: none).
  auto q_of = [&](const Place& c) {
    u32x4 x = {0u, 0u, 0u, 0u};
    const int h = tid / (D / 8), d = tid % (D / 8) * 8;
    if (h < G) x = *(const u32x4*)(p.q + c.b * p.q_bs + (long long)(c.kvh * G + h) * p.q_hs + d);
    return x;
  };
  auto q_put = [&](u32x4 x) {
    const int h = tid / (D / 8), d = tid % (D / 8) * 8;
    if (h < kMaxG) *(u32x4*)(s_q + h * QS + d) = x;
  };

  // ---- the first tile on its way, the ids of the second --------------------------------
  Place A = seg, C;           // the tile whose rows are in t; the next one of this wave
  Ids ai = {}, ci = {};
  A.k = start + wid;
  if (A.k < end) A = walk(A, A.k);
  ai = ids_of(A);
  C = A;
  C.k = A.k + kWaves;
  if (C.k < end) C = walk(C, C.k);
  ci = ids_of(C);
  load_k(A, ai);
  load_v(A, ai);
  q_put(q_of(seg));
  __syncthreads();

  f32x4 o[DT];
  float m, l;
  auto step = [&]() {
    // ---- scores ----
    f32x4 s[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
    const uint16_t* qr = s_q + r * QS + (FP8 ? 16 : 8) * g;
#pragma unroll
    for (int j = 0; j < T::KL; ++j) {
      if constexpr (FP8) {
        const u32x4 q0 = *(const u32x4*)(qr + 64 * j), q1 = *(const u32x4*)(qr + 64 * j + 8);
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const u32x4 w = t.k[a][j];
          s[a] = mfma(u32x4{widen_lo(w.x), widen_hi(w.x), widen_lo(w.y), widen_hi(w.y)}, q0, s[a]);
          s[a] = mfma(u32x4{widen_lo(w.z), widen_hi(w.z), widen_lo(w.w), widen_hi(w.w)}, q1, s[a]);
        }
      } else {
        const u32x4 q0 = *(const u32x4*)(qr + 32 * j);
#pragma unroll
        for (int a = 0; a < 2; ++a) s[a] = mfma(t.k[a][j], q0, s[a]);
      }
    }
    const bool there = (unsigned)ai.vid < (unsigned)p.c.n_pages;
    const int left = there ? A.n - ((A.k - A.u0) * kTile + 8 * g) : 0;  // visible positions of this lane's 8
    float x[8], vs[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = FP8 ? t.ks[i >> 2][i & 3] * qscale : qscale;
      x[i] = i < left ? s[i >> 2][i & 3] * f : -INFINITY;
      vs[i] = FP8 ? t.vs[i >> 2][i & 3] : 1.0f;
    }
    Place nx = A;
    Ids ni = ai;
    load_k(C, ci);
    nx = C;
    ni = ci;
    C.k += kWaves;
    if (C.k < end) C = walk(C, C.k);
    ci = ids_of(C);
    // ---- weights ----
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    if (__any(top > m + 8.0f)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float nm = fmaxf(m, top);
      const float corr = m == -INFINITY ? 0.0f : exp2f(m - nm);
      l *= corr;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= corr;
      m = nm;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = exp2f(x[i] - ref);
      l += e;
      w[i] = FP8 ? (i < left ? e * vs[i] : 0.0f) : e;
    }
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = pack_bf2(w[2 * i], w[2 * i + 1]);
      lo[i] = pack_bf2(w[2 * i] - bf_lo(hi[i]), w[2 * i + 1] - bf_hi(hi[i]));
    }
    // ---- outputs ----
    if (__any(left < 8)) {   // what lies in a masked place may be anything: its weight of 0 must meet a 0
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int d = 0; d < T::VD; ++d) t.v[i][d] = i < left ? t.v[i][d] : 0u;
    }
#pragma unroll
    for (int d = 0; d < T::VD; ++d) {
      if constexpr (FP8) {
        u32x4 e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a01 = __builtin_amdgcn_perm(t.v[2 * i + 1][d], t.v[2 * i][d], 0x05010400u);
          const uint32_t a23 = __builtin_amdgcn_perm(t.v[2 * i + 1][d], t.v[2 * i][d], 0x07030602u);
          e[0][i] = widen_lo(a01);
          e[1][i] = widen_hi(a01);
          e[2][i] = widen_lo(a23);
          e[3][i] = widen_hi(a23);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) o[4 * d + j] = mfma(e[j], hi, o[4 * d + j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[4 * d + j] = mfma(e[j], lo, o[4 * d + j]);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        u32x4 e[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[0][i] = __builtin_amdgcn_perm(t.v[2 * i + 1][d], t.v[2 * i][d], 0x05040100u);
          e[1][i] = __builtin_amdgcn_perm(t.v[2 * i + 1][d], t.v[2 * i][d], 0x07060302u);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) o[2 * d + j] = mfma(e[j], hi, o[2 * d + j]);
#pragma unroll
        for (int j = 0; j < 2; ++j) o[2 * d + j] = mfma(e[j], lo, o[2 * d + j]);
        if (d & 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
    load_v(nx, ni);
    A = nx;
    ai = ni;
  };

  const int rec = rec_floats(G, D);
  Pair open0 = {0, 0, 0, 0, 0}, open1 = {0, 0, 0, 0, 0};
  auto gate_of = [&](const Pair& x, int h, int c) {
    return p.gate ? *(const u32x2*)(p.gate + x.b * p.g_bs + (long long)(x.kvh * G + h) * p.g_hs + c) : u32x2{0u, 0u};
  };
  auto emit = [&](const Pair& x, int h, int c, f32x4 a, float L, u32x2 gt) {
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (L == 0.0f) a = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = a[i] * inv;
    if (p.gate) {
      y[0] *= qh_sigmoid(bf_lo(gt.x)); y[1] *= qh_sigmoid(bf_hi(gt.x));
      y[2] *= qh_sigmoid(bf_lo(gt.y)); y[3] *= qh_sigmoid(bf_hi(gt.y));
    }
    *(u32x2*)(p.out + ((size_t)x.b * p.n_heads + x.kvh * G + h) * D + c) =
        u32x2{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3])};
  };
  while (true) {
    const int s1 = min(seg.u1, end);
    const bool more_seg = s1 < end;
    Place next = seg;
    u32x4 qn = {0u, 0u, 0u, 0u};
    if (more_seg) {
      next = walk(seg, s1);
      qn = q_of(next);
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    m = -INFINITY;
    l = 0.0f;
    while (A.k < s1) step();
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // ---- the waves' parts, joined in LDS ----
    if (g == 0) {
      s_m[wid][r] = m;
      s_l[wid][r] = l;
    }
    if (r < G) {
      float* dst = s_o + ((size_t)wid * G + r) * HS;
      constexpr int RUN = FP8 ? DT : 8;              // consecutive dims of a lane
#pragma unroll
      for (int rr = 0; rr < 4; ++rr)
#pragma unroll
        for (int d = 0; d < DT; d += 4)
          *(f32x4*)(dst + RUN * (4 * g + rr) + (FP8 ? d : 128 * (d / 8) + d % 8)) =
              f32x4{o[d][rr], o[d + 1][rr], o[d + 2][rr], o[d + 3][rr]};
    }
    __syncthreads();
    Pair now;
    now.b = seg.b;
    now.kvh = seg.kvh;
    now.pieces = w0 >= 0 ? pieces : (seg.u1 - 1) / share - seg.u0 / share + 1;
    now.first = w0 >= 0 ? w0 : seg.u0 / share;
    now.tail = w0 < 0 && seg.u0 != now.first * share ? 1 : 0;
    float* mine_rec = p.part + (size_t)(2 * wg + (seg.k != start ? 1 : 0)) * rec;
    const auto out_rsrc = __builtin_amdgcn_make_buffer_rsrc(mine_rec, (short)0, rec * 4, 0x00020000);
    for (int i = tid; i < G * D / 4; i += kThreads) {
      const int h = i / (D / 4), c = (i % (D / 4)) * 4;
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_m[w][h]);
      f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        // a wave that saw nothing (sum 0) counts for nothing; a NaN counts
        const float f = s_l[w][h] == 0.0f ? 0.0f : exp2f(s_m[w][h] - M);
        L += s_l[w][h] * f;
        const f32x4 x = *(const f32x4*)(s_o + ((size_t)w * G + h) * HS + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = f != 0.0f ? fmaf(x[e], f, a[e]) : a[e];
      }
      if (now.pieces == 1) {
        emit(now, h, c, a, L, gate_of(now, h, c));
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, a), out_rsrc, (h * D + c) * 4, 0, 16);
        if (c == 0) {
          pub_store(mine_rec + G * D + h, M);
          pub_store(mine_rec + G * D + kMaxG + h, L);
        }
      }
    }
    // A share holds at most two pairs that others hold too, its first and its last: both
    // arrivals wait for the share's end, when the first one's stores are long done.
    if (now.pieces > 1) {
      if (seg.k == start) open0 = now;
      else open1 = now;
    }
    if (!more_seg) break;
    q_put(qn);                                       // every wave is done with the rows of this pair
    __syncthreads();                                 // the query rows are there, LDS is free
    seg = next;
  }
  if (open0.pieces == 0 && open1.pieces == 0) return;
  wait_mem();
  __syncthreads();
  if (tid < 2) {
    const Pair x = tid == 0 ? open0 : open1;
    if (x.pieces) {
      const unsigned prev = __hip_atomic_fetch_add(p.counters + x.b * Hkv + x.kvh, 1u, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT);
      s_last[tid] = prev == (unsigned)x.pieces - 1;
    } else {
      s_last[tid] = 0;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    if (!s_last[which]) continue;
    const Pair x = which == 0 ? open0 : open1;
    // the pieces' maxima and sums, then their weights, in LDS; then the weighted outputs
    auto rec_of = [&](int j) { return p.part + (size_t)(2 * (x.first + j) + (j == 0 ? x.tail : 0)) * rec; };
    float *s_w = s_o, *s_s = s_o + kMaxWG * G;
    f32x4* s_a = (f32x4*)(s_o + 2 * kMaxWG * G);     // [kThreads]
    for (int i = tid; i < x.pieces * G; i += kThreads) {
      const int j = i / G, h = i - j * G;
      s_w[h * kMaxWG + j] = pub_load(rec_of(j) + G * D + h);
      s_s[h * kMaxWG + j] = pub_load(rec_of(j) + G * D + kMaxG + h);
    }
    __syncthreads();
    for (int h = wid; h < G; h += kWaves) {
      float M = -INFINITY, L = 0.0f;
      for (int j = lane; j < x.pieces; j += 64) M = fmaxf(M, s_w[h * kMaxWG + j]);
      M = wave_max(M);
      for (int j = lane; j < x.pieces; j += 64) {
        const float lj = s_s[h * kMaxWG + j], f = lj == 0.0f ? 0.0f : exp2f(s_w[h * kMaxWG + j] - M);
        s_w[h * kMaxWG + j] = f;
        L += lj * f;
      }
      L = wave_sum(L);
      if (lane == 0) s_sum[h] = L;
    }
    __syncthreads();
    const int items = G * D / 4, subs = items < kThreads ? kThreads / items : 1;
    for (int i0 = 0; i0 < items; i0 += kThreads) {
      const int sub = items < kThreads ? tid / items : 0, i = i0 + tid - sub * items;
      const int h = i / (D / 4), c = (i % (D / 4)) * 4;
      f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
      u32x2 gt = {0u, 0u};
      if (i < items && sub < subs) {
        gt = gate_of(x, h, c);
        constexpr int U = 8;
        for (int j = sub; j < x.pieces; j += U * subs) {
          u32x4 y[U];
#pragma unroll
          for (int u = 0; u < U; ++u) y[u] = coherent_load(rec_of(min(j + u * subs, x.pieces - 1)) + h * D + c);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int jj = j + u * subs;
            const float f = jj < x.pieces ? s_w[h * kMaxWG + jj] : 0.0f;
            const f32x4 z = __builtin_bit_cast(f32x4, y[u]);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = f != 0.0f ? fmaf(z[e], f, a[e]) : a[e];
          }
        }
      }
      if (subs > 1) {
        s_a[tid] = a;
        __syncthreads();
        if (sub == 0)
          for (int k = 1; k < subs; ++k) a += s_a[k * items + i];
      }
      if (i < items && sub == 0) emit(x, h, c, a, s_sum[h], gt);
    }
    if (tid == 0) reset_counter(p.counters + x.b * Hkv + x.kvh);
    __syncthreads();
  }
}

}  // namespace

size_t qh_paged_attn_ws_bytes(int n_heads, int n_kv, int D) {
  if (n_kv < 1 || n_heads < 1 || n_heads % n_kv != 0 || n_heads / n_kv > kMaxG || (D != 128 && D != 256)) return 0;
  return kPagedMaxUnits * sizeof(unsigned) + (size_t)2 * kMaxWG * rec_floats(n_heads / n_kv, D) * sizeof(float);
}

template <int D, bool FP8>
static int launch(const QhPagedAttnParams& p, hipStream_t st) {
  const size_t lds = lds_bytes(p.n_heads / p.c.n_kv, D, p.c.n_seqs);
  hipLaunchKernelGGL((paged_attn_kernel<D, FP8>), dim3(kMaxWG), dim3(kThreads), lds, st, p);
  return 0;
}

int qh_launch_paged_attn(const QhPagedAttnParams& p, int D, hipStream_t st) {
  if (D == 256) return p.c.ks ? launch<256, true>(p, st) : launch<256, false>(p, st);
  return p.c.ks ? launch<128, true>(p, st) : launch<128, false>(p, st);
}
