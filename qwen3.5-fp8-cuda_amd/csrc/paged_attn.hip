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
// Work split: the granules (128 positions of one KV head of one sequence) of the whole
// batch form one line, cut into equal shares of consecutive granules, one a workgroup,
// so ragged batches load all CUs alike.  A (sequence, KV head) inside one share is
// written out; one that several shares cut leaves a partial record a piece (maximum,
// sum, outputs), and the last piece to arrive joins them in order: the result does not
// depend on who comes last.
#include <type_traits>

#include "qh_common.h"
#include "qh_paged.h"

namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;                    // positions per wave and step
constexpr int kGranule = kWaves * kTile;     // positions per workgroup and step
constexpr int kMaxWG = 512;                  // workgroups that hold a share (two per CU)
constexpr int kMaxG = 16;

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

// Four E4M3 bytes as two words of two bf16 each.
__device__ __forceinline__ uint32_t widen_lo(uint32_t x) { return __builtin_bit_cast(uint32_t, e4m3x2_lo_bf16(x)); }
__device__ __forceinline__ uint32_t widen_hi(uint32_t x) { return __builtin_bit_cast(uint32_t, e4m3x2_hi_bf16(x)); }

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

template <int D, bool FP8>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(QhPagedAttnParams p) {
  using T = Tile<D, FP8>;
  constexpr int DT = D / 16;                         // 16-dim tiles of the output
  constexpr int KK = D / 32;                         // products of a score tile
  constexpr int HS = D + 4;                          // floats between heads in LDS
  __shared__ int s_tot[256];
  __shared__ float s_m[kWaves][kMaxG], s_l[kWaves][kMaxG];
  __shared__ int s_last;
  extern __shared__ __align__(16) float s_o[];       // [kWaves][G][HS], then s_cum

  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int B = p.c.n_seqs, Hkv = p.c.n_kv, G = p.n_heads / Hkv, ps = p.c.page_size;
  const int wg = blockIdx.x;
  int* s_cum = (int*)(s_o + kWaves * G * HS);        // [B] granules (of one KV head) of sequences 0 .. b

  // ---- the line of granules: a running sum over the sequences ----------------------
  const int per = (B + 255) / 256, b0 = tid * per;
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = b0 + i;
    if (b < B) {
      const int n = min(p.last[b], p.c.capacity - 1) + 1;
      mine += n > 0 ? (n + kGranule - 1) / kGranule : 0;
      s_cum[b] = mine;
    }
  }
  s_tot[tid] = mine;
  __syncthreads();
#pragma unroll
  for (int d = 1; d < 256; d <<= 1) {
    const int add = tid >= d ? s_tot[tid - d] : 0;
    __syncthreads();
    s_tot[tid] += add;
    __syncthreads();
  }
  const int before = tid > 0 ? s_tot[tid - 1] : 0;
  for (int i = 0; i < per; ++i)
    if (b0 + i < B) s_cum[b0 + i] += before;
  const long long total = (long long)s_tot[255] * Hkv;
  __syncthreads();
  const long long share = max(1ll, (total + gridDim.x - 1) / gridDim.x);

  // empty sequences: zeros
  for (int b = wg; b < B; b += gridDim.x) {
    if (s_cum[b] != (b > 0 ? s_cum[b - 1] : 0)) continue;
    for (int i = tid; i < p.n_heads * D / 8; i += 256)
      *(u32x4*)(p.out + (size_t)b * p.n_heads * D + i * 8) = u32x4{0u, 0u, 0u, 0u};
  }

  long long at = wg * share;
  const long long end = min(total, at + share);
  if (at >= end) return;
  int b;
  {  // the sequence of granule `at`: the first whose running sum passes it
    int lo = 0, hi = B - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((long long)s_cum[mid] * Hkv > at) hi = mid;
      else lo = mid + 1;
    }
    b = lo;
  }
  const float qscale = (D == 256 ? 0.0625f : 0.08838834764831845f) * 1.4426950408889634f;  // log2(e) / sqrt(D)

  while (at < end) {
    const int first = b > 0 ? s_cum[b - 1] : 0, gran = s_cum[b] - first;
    if (gran == 0) { ++b; continue; }
    const int kvh = (int)((at - (long long)first * Hkv) / gran);
    const long long u0 = (long long)first * Hkv + (long long)kvh * gran;  // this (b, kvh) on the line
    const int g0 = (int)(at - u0), g1 = (int)min((long long)gran, end - u0);
    const int n = min(p.last[b], p.c.capacity - 1) + 1;
    const int p1 = min(n, g1 * kGranule);
    const int* pages = p.c.pages + (size_t)b * p.c.max_pages;

    // this lane's query dims: head r (those above G repeat head 0; nothing of theirs is used)
    u32x4 q[KK];
    {
      const uint16_t* src = p.q + b * p.q_bs + (long long)(kvh * G + (r < G ? r : 0)) * p.q_hs;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        q[kk] = *(const u32x4*)(src + (FP8 ? 64 * (kk / 2) + 16 * g + 8 * (kk & 1) : 32 * kk + 8 * g));
    }
    f32x4 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;

    // Page ids of the lane's two groups of 8 positions (K: r / 4, V: g) of the tile at t0.
    // A group behind the last position takes the one that holds it.
    const int lastgrp = (n - 1) & ~7;
    struct Ids { int kid, vid, koff, voff; };
    auto ids_of = [&](int t0) {
      Ids x;
      const int kp = min(t0 + 8 * (r >> 2), lastgrp), vp = min(t0 + 8 * g, lastgrp);
      const int kq = page_of(p.c, kp), vq = page_of(p.c, vp);
      x.kid = pages[kq];
      x.vid = pages[vq];
      x.koff = kp - kq * ps;
      x.voff = vp - vq * ps;
      return x;
    };
    auto row_of = [&](int id, int off) {
      return ((long long)((unsigned)id < (unsigned)p.c.n_pages ? id : 0) * Hkv + kvh) * ps + off;
    };
    T t;
    auto load_k = [&](const Ids& x) {
      const long long row = row_of(x.kid, x.koff + (r & 3));
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const char* src = (const char*)p.c.k + (row + 4 * a) * (FP8 ? D : 2 * D) + 16 * g;
#pragma unroll
        for (int j = 0; j < T::KL; ++j) t.k[a][j] = *(const u32x4*)(src + 64 * j);
      }
      if constexpr (FP8) {
        const long long vrow = row_of(x.vid, x.voff);
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          t.ks[a] = *(const f32x4*)(p.c.ks + vrow + 4 * a);
          t.vs[a] = *(const f32x4*)(p.c.vs + vrow + 4 * a);
        }
      }
    };
    auto load_v = [&](const Ids& x) {
      const char* src = (const char*)p.c.v + row_of(x.vid, x.voff) * (FP8 ? D : 2 * D);
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

    auto step = [&](int t0, const Ids& cur, auto more) {
      constexpr bool MORE = decltype(more)::value;
      // ---- scores ----
      f32x4 s[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        s[a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < T::KL; ++j) {
          if constexpr (FP8) {
            const u32x4 w = t.k[a][j];
            s[a] = mfma(u32x4{widen_lo(w.x), widen_hi(w.x), widen_lo(w.y), widen_hi(w.y)}, q[2 * j], s[a]);
            s[a] = mfma(u32x4{widen_lo(w.z), widen_hi(w.z), widen_lo(w.w), widen_hi(w.w)}, q[2 * j + 1], s[a]);
          } else {
            s[a] = mfma(t.k[a][j], q[j], s[a]);
          }
        }
      }
      const bool there = (unsigned)cur.vid < (unsigned)p.c.n_pages;
      const int left = there ? p1 - (t0 + 8 * g) : 0;         // visible positions of this lane's 8
      float x[8], vs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = FP8 ? t.ks[i >> 2][i & 3] * qscale : qscale;
        x[i] = i < left ? s[i >> 2][i & 3] * f : -INFINITY;
        vs[i] = FP8 ? t.vs[i >> 2][i & 3] : 1.0f;
      }
      Ids nxt = cur;
      if constexpr (MORE) {
        nxt = ids_of(t0 + kGranule);
        load_k(nxt);
      }
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
          for (int j = 0; j < 4; ++j) o[4 * d + j] = mfma(e[j], lo, mfma(e[j], hi, o[4 * d + j]));
        } else {
          u32x4 e[2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[0][i] = __builtin_amdgcn_perm(t.v[2 * i + 1][d], t.v[2 * i][d], 0x05040100u);
            e[1][i] = __builtin_amdgcn_perm(t.v[2 * i + 1][d], t.v[2 * i][d], 0x07060302u);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) o[2 * d + j] = mfma(e[j], lo, mfma(e[j], hi, o[2 * d + j]));
        }
      }
      if constexpr (MORE) load_v(nxt);
      return nxt;
    };

    int t0 = g0 * kGranule + wid * kTile;
    if (t0 < p1) {
      Ids cur = ids_of(t0);
      load_k(cur);
      load_v(cur);
      for (; t0 + kGranule < p1; t0 += kGranule) cur = step(t0, cur, std::integral_constant<bool, true>{});
      step(t0, cur, std::integral_constant<bool, false>{});
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // ---- the four waves' parts, joined in LDS ----
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
    const int npieces = (int)((u0 + gran - 1) / share - u0 / share) + 1;
    const int unit = b * Hkv + kvh, rec = rec_floats(G, D);
    float* mine_rec = p.part + (size_t)(2 * wg + (at != (long long)wg * share ? 1 : 0)) * rec;
    const auto out_rsrc = __builtin_amdgcn_make_buffer_rsrc(mine_rec, (short)0, rec * 4, 0x00020000);
    auto emit = [&](int h, int c, f32x4 a, float L) {
      const size_t head = (size_t)(kvh * G + h);
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      if (L == 0.0f) a = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = a[i] * inv;
      if (p.gate) {
        const u32x2 gt = *(const u32x2*)(p.gate + b * p.g_bs + (long long)head * p.g_hs + c);
        y[0] *= qh_sigmoid(bf_lo(gt.x)); y[1] *= qh_sigmoid(bf_hi(gt.x));
        y[2] *= qh_sigmoid(bf_lo(gt.y)); y[3] *= qh_sigmoid(bf_hi(gt.y));
      }
      *(u32x2*)(p.out + ((size_t)b * p.n_heads + head) * D + c) = u32x2{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3])};
    };
    for (int i = tid; i < G * D / 4; i += 256) {
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
      if (npieces == 1) {
        emit(h, c, a, L);
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, a), out_rsrc, (h * D + c) * 4, 0, 16);
        if (c == 0) {
          pub_store(mine_rec + G * D + h, M);
          pub_store(mine_rec + G * D + kMaxG + h, L);
        }
      }
    }
    if (npieces > 1 && arrive_last(p.counters + unit, (unsigned)npieces, &s_last)) {
      const long long w0 = u0 / share;
      const bool tail0 = u0 != w0 * share;           // the first piece is the second record of its workgroup
      for (int i = tid; i < G * D / 4; i += 256) {
        const int h = i / (D / 4), c = (i % (D / 4)) * 4;
        float M = -INFINITY, L = 0.0f;
        f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int j = 0; j < npieces; ++j) {
          float* src = p.part + (size_t)(2 * (w0 + j) + (j == 0 && tail0 ? 1 : 0)) * rec;
          const auto rs = __builtin_amdgcn_make_buffer_rsrc(src, (short)0, rec * 4, 0x00020000);
          const f32x4 x = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (h * D + c) * 4, 0, 16));
          const float mj = pub_load(src + G * D + h), lj = pub_load(src + G * D + kMaxG + h);
          if (lj == 0.0f) continue;
          const float nm = fmaxf(M, mj);
          const float fo = M == -INFINITY ? 0.0f : exp2f(M - nm), fn = exp2f(mj - nm);
          L = L * fo + lj * fn;
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = a[e] * fo + x[e] * fn;
          M = nm;
        }
        emit(h, c, a, L);
      }
      if (tid == 0) reset_counter(p.counters + unit);
    }
    __syncthreads();  // LDS is free for the next (sequence, KV head)
    at = u0 + g1;
    if (kvh == Hkv - 1 && g1 == gran) ++b;
  }
}

}  // namespace

size_t qh_paged_attn_ws_bytes(int n_heads, int n_kv, int D) {
  if (n_kv < 1 || n_heads < 1 || n_heads % n_kv != 0 || n_heads / n_kv > kMaxG || (D != 128 && D != 256)) return 0;
  return kPagedMaxUnits * sizeof(unsigned) + (size_t)2 * kMaxWG * rec_floats(n_heads / n_kv, D) * sizeof(float);
}

template <int D, bool FP8>
static int launch(const QhPagedAttnParams& p, hipStream_t st) {
  const int G = p.n_heads / p.c.n_kv;
  const size_t lds = (size_t)kWaves * G * (D + 4) * sizeof(float) + (size_t)p.c.n_seqs * sizeof(int);
  hipLaunchKernelGGL((paged_attn_kernel<D, FP8>), dim3(kMaxWG), dim3(256), lds, st, p);
  return 0;
}

int qh_launch_paged_attn(const QhPagedAttnParams& p, int D, hipStream_t st) {
  if (D == 256) return p.c.ks ? launch<256, true>(p, st) : launch<256, false>(p, st);
  return p.c.ks ? launch<128, true>(p, st) : launch<128, false>(p, st);
}
