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
// (V).  Weights enter the product as the sum of two bf16 numbers: what is lost is up to
// 2^-16 of a weight over bf16 rows, whose first part is cut off, not rounded, and 2^-17 over
// E4M3 rows (one bf16 number: 2^-8; a third part that loses nothing: 1 to 2 % of the time of
// every call, for outputs that are rounded by 2^-8).
// Scores, maxima, sums and outputs are fp32.  Weights are 2^(s - m) with an m that a score
// above it raises to 2^8 times that score's: none is above 1, so an output overflows no
// sooner than the sum of the values, and a tile whose scores stay below m needs no exchange
// between lanes and no rescaling.
//
// Work split: the tiles (32 positions of one KV head of one sequence) of the whole
// batch form one line, cut into equal shares of consecutive tiles, one a wave, so ragged
// batches load all CUs alike.  The rows of a wave's next tile are on their way while it
// computes, across sequences too, and the page ids of the one after.  A (sequence, KV
// head) inside one wave's share is written out from its registers.  One that waves of a
// workgroup cut is joined once, at the share's end, through LDS; one that workgroups cut
// leaves a partial record a piece (maximum, sum, outputs) in the workspace, and the last
// piece to arrive joins them.  All joins go in the order of the pieces: the result does
// not depend on who comes last.
//
// Measured: 128 sequences of 500 to 6000 positions (64 / 8 heads of 128, bf16) 184 us, 6.3 TB/s;
// one of 200001 (16 / 4 heads of 256, E4M3) 73 us, 5.7 TB/s, of 4096 11.5 us; 43 of 1 to 8000 29 us,
// 4.6 TB/s.  With the arithmetic taken out the long ones take as long.  Short ones are a chain of
// dependent round trips: length, page ids, rows, LDS join, record, arrival, records.
#include <algorithm>
#include <type_traits>

#include "qh_common.h"
#include "qh_paged.h"

namespace {

constexpr int kTile = 32;    // positions per wave and step
constexpr int kMaxWG = 256;  // workgroups that hold a share (one per CU)
constexpr int kMaxG = 16;
constexpr float kAbove = 1.00000011920928955f;  // 1 + 2^-23
// Waves of a workgroup: two to a SIMD; one where a tile of bf16 rows of 256 fills the
// registers (16 / 4 heads, 300 positions: 11.9 us with four waves, 16.6 with eight), or where
// the LDS has no room for the partial results of eight.
constexpr int waves_of(int G, int D, bool fp8) { return D == 256 && (!fp8 || G > 8) ? 4 : 8; }

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

// Four E4M3 bytes as two words of two bf16 each.
__device__ __forceinline__ uint32_t widen_lo(uint32_t x) { return __builtin_bit_cast(uint32_t, e4m3x2_lo_bf16(x)); }
__device__ __forceinline__ uint32_t widen_hi(uint32_t x) { return __builtin_bit_cast(uint32_t, e4m3x2_hi_bf16(x)); }

// 2^x as the hardware has it (1 ulp; results below 2^-126 are zero).
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Joins U more parts (maximum, sum, outputs) to (a, M, L).  One that saw nothing (sum 0,
// maximum -inf) counts for nothing; a NaN counts.
template <int U>
__device__ __forceinline__ void add_parts(f32x4& a, float& M, float& L, const f32x4 (&x)[U], const float (&mx)[U],
                                          const float (&lx)[U]) {
  float nm = M;
#pragma unroll
  for (int u = 0; u < U; ++u) nm = fmaxf(nm, mx[u]);
  const float fo = L == 0.0f ? 0.0f : exp2_(M - nm);
  a *= fo;
  L *= fo;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float f = lx[u] == 0.0f ? 0.0f : exp2_(mx[u] - nm);
    L = fmaf(lx[u], f, L);
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = fmaf(x[u][e], f, a[e]);
  }
  M = nm;
}

// Cached rows are read once: non-temporal loads, which also reach 6.8 TB/s where plain
// ones reach 6.0 (random 8 KB pages, 2.4 GB), if they ask for whole 128-byte lines.
template <typename V>
__device__ __forceinline__ V stream_load(const void* p) {
  return __builtin_nontemporal_load((const V*)p);
}

// Exchange with the lane whose r differs in bit 1: x becomes the first half, y the second
// half of the own row's line, of what load_k asked for.
__device__ __forceinline__ void unpair(u32x4& x, u32x4& y, bool second) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t xo = __builtin_amdgcn_update_dpp(0, (int)x[i], 0x4E, 0xF, 0xF, true);  // quad_perm [2,3,0,1]
    const uint32_t yo = __builtin_amdgcn_update_dpp(0, (int)y[i], 0x4E, 0xF, 0xF, true);
    const uint32_t a = second ? yo : x[i], b = second ? y[i] : xo;
    x[i] = a;
    y[i] = b;
  }
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

// A partial result, in LDS or in the workspace: the G heads' outputs, 4 dims at a time as
// lane (r < G, g) of a wave holds them ([D / 16][4 G] x 16 bytes), [16] maxima, [16] sums.
__host__ __device__ constexpr int rec_floats(int G, int D) { return G * D + 2 * kMaxG; }

// LDS floats: two partial results a wave (later, the threads' sums), 8 bytes a sequence.
__host__ __device__ constexpr int slot_floats(int G, int D, int waves) {
  const int slots = 2 * waves * rec_floats(G, D), sums = waves * 64 * 6;
  return slots > sums ? slots : sums;
}

// A tile on the line: its sequence and KV head, and the tiles [u0, u1) of that pair.  A place
// of the line is left empty behind each pair: its end costs a wave about a tile's time, and
// waves with many short pairs held up the others (43 sequences of 1 to 8000 positions,
// E4M3, 16 / 4 heads of 256: 43.5 us without it, 34.8 with).
struct Place {
  int k, b, kvh, u0, u1, n;
};

// A pair that several workgroups hold pieces of: the first of them, and whether its
// piece is the second record there.
struct Pair {
  int b, kvh, pieces, first, tail;
};

// Running sum over the wave's lanes, and the maximum of all, of non-negative values by DPP
// moves: within rows of 16 lanes, then from row to row.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_i<0x111, 0xF>(v);  // row_shr:1
  v += dpp_i<0x112, 0xF>(v);
  v += dpp_i<0x114, 0xF>(v);
  v += dpp_i<0x118, 0xF>(v);
  v += dpp_i<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp_i<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_imax(int v) {
  v = max(v, dpp_i<0x111, 0xF>(v));
  v = max(v, dpp_i<0x112, 0xF>(v));
  v = max(v, dpp_i<0x114, 0xF>(v));
  v = max(v, dpp_i<0x118, 0xF>(v));
  v = max(v, dpp_i<0x142, 0xA>(v));
  v = max(v, dpp_i<0x143, 0xC>(v));
  return __builtin_amdgcn_readlane(v, 63);
}

// a / b for quotients below 2^20 (the compiler's division of 32-bit numbers is three times
// as long, and a wave that divides has nothing else to do).
__device__ __forceinline__ int small_quotient(int a, int b) {
  return qh_quotient_near(a, b, __builtin_amdgcn_rcpf((float)b));
}
__device__ __forceinline__ int small_quotient_s(int a, int b) {  // of numbers that the wave's lanes agree on
  return __builtin_amdgcn_readfirstlane(small_quotient(a, b));
}

// Between a wave's LDS accesses to what other lanes of it wrote, or will write: the hardware takes
// a wave's accesses in order, this keeps the compiler from reordering them (no instruction, no wait).
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int D, bool FP8, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves / 4) void paged_attn_kernel(QhPagedAttnParams p) {
  using T = Tile<D, FP8>;
  constexpr int kThreads = 64 * kWaves;
  // Tiles of a pair that one workgroup takes rather than join pieces.  A wave's second tile of
  // 256 E4M3 values takes longer than the join (1 sequence of 400 positions, 16 / 4 heads: 10.3 us
  // in one workgroup, 8.2 in pieces; 16 of them: 11.2 and 9.9); one of 128 hardly, and pieces for all of
  // a batch do not fit (32 / 8 heads: 7.9 and 7.6; 16 of them: 8.7 and 10.8); nor one of bf16, which has
  // a SIMD to itself (200 positions of 256: 8.2 and 8.4; 16 of them: 9.2 and 9.7).
  constexpr int kWhole = D == 256 && kWaves == 8 ? kWaves : 2 * kWaves;
  constexpr int DT = D / 16;                         // 16-dim tiles of the output
  constexpr int KK = D / 32;                         // products of a score tile
  constexpr int RUN = FP8 ? DT : 8;                  // consecutive dims of a lane
  __shared__ int s_tot[kWaves];
  __shared__ int s_last[2];
  extern __shared__ __align__(16) float s_o[];

  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int B = p.c.n_seqs, Hkv = p.c.n_kv, G = p.group, ps = p.c.page_size;
  const int wg = blockIdx.x;
  int* s_n = (int*)(s_o + slot_floats(G, D, kWaves));  // [B] positions of sequence b
  int* s_cum = s_n + B;                              // [B] places on the line (of one KV head) of sequences 0 .. b

  // ---- this workgroup's part of the work: tiles [start, end), each wave's `ws` of them ----
  Place seg;
  int start = 0, end = 0, share = 0, w0 = -1;        // w0 >= 0: pieces of one pair, the first of them here
  int pieces = 0, ws = 0;
  auto zeros = [&](int b) {                          // an empty sequence
    for (int i = tid; i < p.n_heads * D / 8; i += kThreads)
      *(u32x4*)(p.out + (size_t)b * p.n_heads * D + i * 8) = u32x4{0u, 0u, 0u, 0u};
  };
  // Up to 64 sequences: lane b of every wave has sequence b, nothing goes through LDS.
  const bool few = B <= 64;
  int n_lane = 0, cum_lane = 0;                      // its positions; places (of one KV head) of sequences 0 .. b
  auto places_to = [&](int b) {
    return b < 0 ? 0 : few ? __builtin_amdgcn_readlane(cum_lane, b) : __builtin_amdgcn_readfirstlane(s_cum[b]);
  };
  auto length = [&](int b) {
    return few ? __builtin_amdgcn_readlane(n_lane, b) : __builtin_amdgcn_readfirstlane(s_n[b]);
  };
  int total;
  if (few) {
    n_lane = lane < B ? max(min(p.last[lane], p.c.capacity - 1) + 1, 0) : 0;
    const int tl = (n_lane + kTile - 1) / kTile, most = wave_imax(tl), slots = p.slots;
    cum_lane = wave_scan(tl > 0 ? tl + 1 : 0);
    const int sum = __builtin_amdgcn_readlane(cum_lane, 63);
    for (int b = wg; b < B; b += kMaxWG)
      if (length(b) == 0) zeros(b);
    total = sum * Hkv;
    if (most <= kWhole && B <= slots) share = kWhole;
    else if (4 * B <= slots) {
      // equal shares would do if none of them were cut short; that costs a piece a sequence at most
      share = max(4, (sum + slots - 1) / slots);
      if (__builtin_amdgcn_readlane(wave_scan(small_quotient(tl + share - 1, share)), 63) > slots)
        share = max(4, (sum + slots - B - 1) / (slots - B));
      // Four waves have a SIMD each, eight take as long for 5 tiles as for 8 (2 sequences of 4096, 16 / 4
      // heads of 256, E4M3, in shares of 5 and of 8: 13.6 and 12.7 us); and from some length on half the
      // pieces are worth a shared SIMD, the sooner the narrower the rows.  One sequence, shares of 4 and of 8:
      //   16 / 4 of 256, E4M3: 3000 positions 10.8 and 11.3 us, 4096 11.8 and 11.8, 5000 12.8 and 12.5
      //   ... bf16:            3000 12.5 and 13.2, 4096 13.9 and 13.6, 5000 15.3 and 14.5
      //   32 / 8 of 128, E4M3: 1500 8.7 and 9.4, 2000 9.2 and 9.5, 2500 9.9 and 9.7, 3000 10.3 and 10.1
      //   ... bf16:            2000 9.2 and 9.9, 2500 9.9 and 10.1, 3000 10.4 and 10.4, 4096 11.8 and 11.1
      // More pairs want it earlier (2 sequences of 16 / 4 of 256, E4M3: 2500 11.6 and 11.8, 3500 12.9 and
      // 12.3), fewer later (8 / 2: 5000 11.7 and 12.1, 6000 12.4 and 12.3): up to 5 % beside the border.
      if (share < 8 && (share > 4 || most > D / 2)) share = 8;
    }
    if (share > 0) {
      const int pc = small_quotient(tl + share - 1, share), cum = wave_scan(pc);
      const unsigned long long past = __ballot(cum * Hkv > wg);
      if (past == 0) return;
      seg.b = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
      seg.n = length(seg.b);
      pieces = __builtin_amdgcn_readlane(pc, seg.b);
      const int i = wg - (__builtin_amdgcn_readlane(cum, seg.b) - pieces) * Hkv;
      seg.kvh = small_quotient_s(i, pieces);
      const int j = i - seg.kvh * pieces;
      w0 = wg - j;
      seg.u0 = 0;
      seg.u1 = (seg.n + kTile - 1) / kTile;
      start = seg.k = j * share;
      end = min(seg.u1, start + share);
      ws = (end - start + kWaves - 1) / kWaves;
    }
  } else {
    const int per = (B + kThreads - 1) / kThreads, b0 = tid * per;
    int mine = 0;
    for (int i = 0; i < per; ++i) {
      const int b = b0 + i;
      if (b < B) {
        const int n = max(min(p.last[b], p.c.capacity - 1) + 1, 0);
        mine += n > 0 ? (n + kTile - 1) / kTile + 1 : 0;
        s_n[b] = n;
        s_cum[b] = mine;
      }
    }
    const int sum = wave_scan(mine);
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
    total = __builtin_amdgcn_readfirstlane(all) * Hkv;
    __syncthreads();
    for (int b = wg; b < B; b += kMaxWG)
      if (s_n[b] == 0) zeros(b);
  }
  if (w0 < 0) {
    // a share of the line of all tiles
    ws = max(1, (int)((unsigned)(total + kMaxWG * kWaves - 1) / (kMaxWG * kWaves)));
    share = ws * kWaves;
    start = wg * share;
    end = min(total, start + share);
    if (start >= end) return;
    int lo = 0;                                      // the sequence of tile `start`: the first whose running sum passes it
    if (few) {
      lo = __builtin_amdgcn_readfirstlane(__ffsll(__ballot(cum_lane * Hkv > start)) - 1);
    } else {
      int hi = B - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (places_to(mid) * Hkv > start) hi = mid;
        else lo = mid + 1;
      }
    }
    const int first = places_to(lo - 1), places = places_to(lo) - first;
    seg.k = start;
    seg.b = lo;
    seg.kvh = small_quotient_s(start - first * Hkv, places);
    seg.u0 = first * Hkv + seg.kvh * places;
    seg.u1 = seg.u0 + places - 1;
    seg.n = length(lo);
  }
  // The first tile at place k or behind it that is not before pair c, and its pair; .k >= until:
  // there is none before that place.
  auto seek = [&](Place c, int k, int until) {
    k = max(k, c.u0);
    while (k >= c.u1) {
      k = max(k, c.u1 + 1);
      if (k >= until) break;
      if (++c.kvh == Hkv) {
        c.kvh = 0;
        do ++c.b; while (places_to(c.b) == places_to(c.b - 1));
        c.n = length(c.b);
      }
      c.u0 = c.u1 + 1;
      c.u1 = c.u0 + (c.n + kTile - 1) / kTile;
    }
    c.k = k;
    return c;
  };
  seg = seek(seg, start, end);
  if (seg.k >= end) return;
  const int k0 = start + wid * ws, k1 = min(end, k0 + ws);  // this wave's tiles
  const float qscale = (D == 256 ? 0.0625f : 0.08838834764831845f) * 1.4426950408889634f;  // log2(e) / sqrt(D)

  // Page ids and slots of the lane's two groups of 8 positions (K: r / 4, V: g) of a tile.
  // A group behind the last position takes the one that holds it.
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
  auto row_of = [&](const Place& c, int id, int off) {  // of page 0 where there is none: its rows are masked
    return ((long long)((unsigned)id < (unsigned)p.c.n_pages ? id : 0) * Hkv + c.kvh) * ps + off;
  };
  T t;
  // Rows of K come in whole cache lines: in a pair of loads, lanes whose r has bit 1 clear
  // ask for the first half of a line of rows r and r + 2, the others for the second half
  // of rows r - 2 and r; unpair() below hands each lane its own row's two halves.
  const bool second = (r & 2) != 0;
  auto load_k = [&](const Place& c, const Ids& x) {
    const long long row = row_of(c, x.kid, x.koff) + (r & 1);
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const char* src = (const char*)p.c.k + (row + 4 * a) * (FP8 ? D : 2 * D) + 16 * g + (second ? 64 : 0);
#pragma unroll
      for (int j = 0; j < T::KL; j += 2) {
        t.k[a][j] = stream_load<u32x4>(src + 64 * j);
        t.k[a][j + 1] = stream_load<u32x4>(src + 64 * j + 2 * (FP8 ? D : 2 * D));
      }
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
        const u32x2 w = stream_load<u32x2>(s + 8 * r);
        t.v[i][0] = w.x; t.v[i][1] = w.y;
      } else {
#pragma unroll
        for (int j = 0; j < T::VD / 4; ++j) {
          const u32x4 w = stream_load<u32x4>(s + 16 * (r + 16 * j));
          t.v[i][4 * j] = w.x; t.v[i][4 * j + 1] = w.y; t.v[i][4 * j + 2] = w.z; t.v[i][4 * j + 3] = w.w;
        }
      }
    }
  };
  // this lane's query dims: head r (those above G repeat head 0; nothing of theirs is used)
  u32x4 q[KK];
  auto load_q = [&](const Place& c) {
    const uint16_t* src = p.q + c.b * p.q_bs + (long long)(c.kvh * G + (r < G ? r : 0)) * p.q_hs;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      q[kk] = *(const u32x4*)(src + (FP8 ? 64 * (kk / 2) + 16 * g + 8 * (kk & 1) : 32 * kk + 8 * g));
  };

  // ---- the first tile on its way, the ids of the second --------------------------------
  Place A = seg, C;           // the tile whose rows are in t; the next one of this wave
  Ids ai, ci;
  A.k = k0;
  if (k0 < k1) A = seek(A, k0, k1);
  if (A.k < k1) {
    ai = ids_of(A);
    load_q(A);
    C = A;
    C.k = A.k + 1;
    if (C.k < k1) C = seek(C, C.k, k1);
    ci = ids_of(C);
    // in the order of the loop: its waits count the loads behind the one they are for
    asm volatile("" ::: "memory");
    load_k(A, ai);
    asm volatile("" ::: "memory");
    load_v(A, ai);
    asm volatile("" ::: "memory");
  }

  f32x4 o[DT];
  float m, l;
  // One tile of the wave, the next one asked for on the way.  The last one is a copy of its own,
  // without that: loads under a branch would make the compiler wait for V where K is needed, and
  // asking for tiles that are not there costs a microsecond (1 sequence of 300 positions, 16 / 4 heads
  // of 256, bf16: 10.8 us, 9.2 without).
  auto step = [&](auto next) {
    constexpr bool kNext = decltype(next)::value;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int j = 0; j < T::KL; j += 2) unpair(t.k[a][j], t.k[a][j + 1], second);
    // ---- scores ----
    f32x4 s[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int j = 0; j < T::KL; ++j) {
      if constexpr (FP8) {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const u32x4 w = t.k[a][j];
          s[a] = mfma(u32x4{widen_lo(w.x), widen_hi(w.x), widen_lo(w.y), widen_hi(w.y)}, q[2 * j], s[a]);
          s[a] = mfma(u32x4{widen_lo(w.z), widen_hi(w.z), widen_lo(w.w), widen_hi(w.w)}, q[2 * j + 1], s[a]);
        }
      } else {
#pragma unroll
        for (int a = 0; a < 2; ++a) s[a] = mfma(t.k[a][j], q[j], s[a]);
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
    if constexpr (kNext) {
      load_k(C, ci);
      if (C.u0 != A.u0) load_q(C);             // the next pair's: this one's scores are done
      nx = C;
      ni = ci;
      ++C.k;
      if (C.k < k1) C = seek(C, C.k, k1);
      ci = ids_of(C);
    }
    // ---- weights ----
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    if (__any(top > m)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float nm = top > m ? top + 8.0f : m;
      const float corr = m == -INFINITY ? 0.0f : exp2_(m - nm);
      l *= corr;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= corr;
      m = nm;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = exp2_(x[i] - ref);
      l += e;
      w[i] = FP8 ? (i < left ? e * vs[i] : 0.0f) : e;
    }
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (FP8) {
        hi[i] = pack_bf2(w[2 * i], w[2 * i + 1]);
        lo[i] = pack_bf2(w[2 * i] - bf_lo(hi[i]), w[2 * i + 1] - bf_hi(hi[i]));
      } else {  // both parts above zero, or an infinity of V would meet a zero or its own negative
        hi[i] = __builtin_amdgcn_perm(__float_as_uint(w[2 * i + 1]), __float_as_uint(w[2 * i]), 0x07060302u);
        lo[i] = pack_bf2(fmaf(w[2 * i], kAbove, -bf_lo(hi[i])), fmaf(w[2 * i + 1], kAbove, -bf_hi(hi[i])));
      }
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
    if constexpr (kNext) {
      load_v(nx, ni);
      A = nx;
      ai = ni;
    }
  };

  const int rec = rec_floats(G, D);
  // device-coherent (sc1) accesses: pieces pass between workgroups whose L2 caches are not coherent
  const auto parts = __builtin_amdgcn_make_buffer_rsrc(p.part, (short)0, 2 * kMaxWG * rec * 4, 0x00020000);
  auto gate_of = [&](int b, int head, int c) {
    return p.gate ? *(const u32x2*)(p.gate + b * p.g_bs + (long long)head * p.g_hs + c) : u32x2{0u, 0u};
  };
  auto emit = [&](int b, int head, int c, f32x4 a, float L, u32x2 gt) {
    const float inv = 1.0f / L;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = a[i] * inv;
    if (p.gate) {
      y[0] *= qh_sigmoid_bf(bf_lo(gt.x)); y[1] *= qh_sigmoid_bf(bf_hi(gt.x));
      y[2] *= qh_sigmoid_bf(bf_lo(gt.y)); y[3] *= qh_sigmoid_bf(bf_hi(gt.y));
    }
    u32x2 w = {pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3])};
    if (L == 0.0f) w = u32x2{0u, 0u};                // nothing visible, whatever the gate holds
    *(u32x2*)(p.out + ((size_t)b * p.n_heads + head) * D + c) = w;
  };
  // Item i of a partial result: head and first of its 4 dims.
  const int items = G * D / 4;
  struct Item { int h, c; };
  auto item = [&](int i) {
    const int k = qh_group_quotient(i >> 2, p.group_mul), ln = i - k * 4 * G, gg = qh_group_quotient(ln, p.group_mul);
    const int rr = k / (DT / 4), d = k % (DT / 4) * 4;
    return Item{ln - gg * G, RUN * (4 * gg + rr) + (FP8 ? d : 128 * (d / 8) + d % 8)};
  };
  // Where the items need no more than half of the threads, these form groups (whole waves).
  const int gsize = 1 << p.group_shift, groups = kThreads >> p.group_shift;
  const int group = wid >> (p.group_shift - 6), gtid = tid & (gsize - 1);
  auto slot_of = [&](int s) { return s_o + (size_t)s * rec; };  // 2 w: begun before wave w, 2 w + 1: by it
  auto put_slot = [&](int s) {
    if (r < G) {
      f32x4* dst = (f32x4*)slot_of(s) + g * G + r;
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        const int rr = i / (DT / 4), d = i % (DT / 4) * 4;
        dst[i * 4 * G] = f32x4{o[d][rr], o[d + 1][rr], o[d + 2][rr], o[d + 3][rr]};
      }
      if (g == 0) *(float2*)(slot_of(s) + G * D + 2 * r) = float2{m, l};
    }
  };
  // ---- this wave's pairs, one after the other -------------------------------------------
  auto begin = [&]() {
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    m = -INFINITY;
    l = 0.0f;
  };
  auto finish = [&](const Place& done) {
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const bool begun = done.u0 < k0;
    wave_lds_order();                                // the last pair's slot has been read
    put_slot(2 * wid + (begun ? 0 : 1));
    if (begun || done.u1 > k1) return;
    wave_lds_order();
    // all of it is here
    const float* src = slot_of(2 * wid + 1);
    for (int i0 = lane; i0 < items; i0 += 256) {
      u32x2 gt[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const Item it = item(min(i0 + 64 * u, items - 1));
        gt[u] = gate_of(done.b, done.kvh * G + it.h, it.c);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 64 * u;
        if (i >= items) break;
        const Item it = item(i);
        emit(done.b, done.kvh * G + it.h, it.c, ((const f32x4*)src)[i], src[G * D + 2 * it.h + 1], gt[u]);
      }
    }
  };
  if (A.k < k1) {
    Place at = A;
    begin();
    while (C.k < k1) {
      const bool over = C.u0 != A.u0;                // A is the last of its pair here
      step(std::true_type{});
      if (over) {
        finish(at);
        at = A;
        begin();
      }
    }
    step(std::false_type{});                         // the wave's last tile
    finish(at);
  }
  // ---- pairs that waves cut: every thread its items, pair by pair -------------------------
  __syncthreads();
  Pair open0 = {0, 0, 0, 0, 0}, open1 = {0, 0, 0, 0, 0};
  auto pair_of = [&](const Place& c) {
    Pair x;
    x.b = c.b;
    x.kvh = c.kvh;
    x.first = w0 >= 0 ? w0 : small_quotient_s(c.u0, share);
    x.pieces = w0 >= 0 ? pieces : small_quotient_s(c.u1 - 1, share) - x.first + 1;
    x.tail = w0 < 0 && c.u0 != x.first * share ? 1 : 0;
    return x;
  };
  {
    int turn = 0;
    auto wave_of = [&](int k) {                      // place k of the share lies in its tiles
      int w = 0;
#pragma unroll
      for (int u = 1; u < kWaves; ++u) w += k >= start + u * ws ? 1 : 0;
      return w;
    };
    Place c = seg;
    while (true) {
      // pair c lies in waves w .. last; wave w began it, or (w = 0) another workgroup
      const bool begun = c.u0 < start, all = !begun && c.u1 <= end;
      const int w = begun ? 0 : wave_of(c.u0), last = wave_of(min(c.u1, end) - 1);
      if (!all || last > w) {
        const bool here = (turn++ & (groups - 1)) == group;
        const int dst = (2 * wg + (c.u0 > start ? 1 : 0)) * rec * 4;  // bytes from the first record
        for (int i = here ? gtid : items; i < items; i += gsize) {
          const Item it = item(i);
          const int head = c.kvh * G + it.h;
          const u32x2 gt = all ? gate_of(c.b, head, it.c) : u32x2{0u, 0u};
          float M = -INFINITY, L = 0.0f;
          f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
          for (int x0 = w; x0 <= last; x0 += 2) {    // two at a time: the code of eight alone takes 0.5 us
            f32x4 y[2];
            float my[2], ly[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const bool in = x0 + u <= last;
              const int x = min(x0 + u, last);
              const float* src = slot_of(2 * x + (x == w && !begun ? 1 : 0));
              y[u] = in ? ((const f32x4*)src)[i] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
              const float2 ml = *(const float2*)(src + G * D + 2 * it.h);
              my[u] = in ? ml.x : -INFINITY;
              ly[u] = in ? ml.y : 0.0f;
            }
            add_parts(a, M, L, y, my, ly);
          }
          if (all) {
            emit(c.b, head, it.c, a, L, gt);
          } else {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, a), parts, dst + i * 16, 0, 16);
            if (i < G) {                             // items 0 .. G - 1: one of each head
              const u32x2 ml = {__float_as_uint(M), __float_as_uint(L)};
              __builtin_amdgcn_raw_buffer_store_b64(ml, parts, dst + (G * D + 2 * it.h) * 4, 0, 16);
            }
          }
        }
        if (!all) {
          if (c.u0 > start) open1 = pair_of(c);
          else open0 = pair_of(c);
        }
      }
      // the next one that waves may cut holds the last tile of a wave, of this one's last or the one after
      const int kn = min(end, start + (last + 1) * ws);
      if (c.u1 >= end) break;
      c = seek(c, kn > c.u1 ? kn - 1 : min(end, kn + ws) - 1, end);
      if (c.k >= end) break;
    }
  }
  // A share holds at most two pairs that other workgroups hold too, its first and its last.
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
    auto rec_of = [&](int j) { return (2 * (x.first + j) + (j == 0 ? x.tail : 0)) * rec * 4; };
    // a thread takes an item, of every subs-th piece where there are groups enough for that
    const int subs = min(groups, x.pieces);
    f32x4* s_a = (f32x4*)s_o;                        // [kThreads]
    float2* s_ml = (float2*)(s_a + kThreads);        // [kThreads]
    for (int i0 = 0; i0 < items; i0 += gsize) {
      const int i = i0 + gtid;
      const Item it = item(min(i, items - 1));
      const int head = x.kvh * G + it.h, off = min(i, items - 1) * 16, ml_off = (G * D + 2 * it.h) * 4;
      float M = -INFINITY, L = 0.0f;
      f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
      const u32x2 gt = gate_of(x.b, head, it.c);
      if (group < subs) {
        // 8 pieces under way together, 4 where there are few
        auto read = [&](auto n) {
          constexpr int U = decltype(n)::value;
          for (int j = group; j < x.pieces; j += U * subs) {
            f32x4 y[U];
            float my[U], ly[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              y[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
              my[u] = -INFINITY;
              ly[u] = 0.0f;
              if (j + u * subs < x.pieces) {
                const int src = rec_of(j + u * subs);
                y[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, off, src, 16));
                const u32x2 ml = __builtin_amdgcn_raw_buffer_load_b64(parts, ml_off, src, 16);
                my[u] = __uint_as_float(ml.x);
                ly[u] = __uint_as_float(ml.y);
              }
            }
            add_parts(a, M, L, y, my, ly);
          }
        };
        if (x.pieces <= 4 * subs) read(std::integral_constant<int, 4>{});
        else read(std::integral_constant<int, 8>{});
      }
      if (subs > 1) {
        s_a[tid] = a;
        s_ml[tid] = float2{M, L};
        __syncthreads();
        if (group == 0)
          for (int k = 1; k < subs; ++k) {
            const int src = (k << p.group_shift) + gtid;
            const f32x4 y[1] = {s_a[src]};
            const float my[1] = {s_ml[src].x}, ly[1] = {s_ml[src].y};
            add_parts(a, M, L, y, my, ly);
          }
      }
      if (i < items && group == 0) emit(x.b, head, it.c, a, L, gt);
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

template <int D, bool FP8, int kWaves>
static int launch(QhPagedAttnParams p, hipStream_t st) {
  const int items = p.group * D / 4;
  p.group_shift = 6;
  while ((1 << p.group_shift) < std::min(items, 64 * kWaves)) ++p.group_shift;
  const size_t lds = (size_t)slot_floats(p.group, D, kWaves) * sizeof(float) + (size_t)p.c.n_seqs * 8;
  hipLaunchKernelGGL((paged_attn_kernel<D, FP8, kWaves>), dim3(kMaxWG), dim3(64 * kWaves), lds, st, p);
  return 0;
}

int qh_launch_paged_attn(QhPagedAttnParams p, int D, hipStream_t st) {
  p.group = p.n_heads / p.c.n_kv;
  p.group_mul = qh_group_mul(p.group);
  p.slots = kMaxWG / p.c.n_kv;
  const bool four = waves_of(p.group, D, p.c.ks != nullptr) == 4;
  if (D == 256) {
    if (!p.c.ks) return launch<256, false, 4>(p, st);
    return four ? launch<256, true, 4>(p, st) : launch<256, true, 8>(p, st);
  }
  return p.c.ks ? launch<128, true, 8>(p, st) : launch<128, false, 8>(p, st);
}
