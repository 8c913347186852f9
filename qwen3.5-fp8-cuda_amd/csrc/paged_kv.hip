// Paged KV cache of the full-attention layers (gfx950): tokens written to it and
// read back from it.  No counterpart in the reference, whose cache is one dense
// bf16 buffer for one sequence (main.py:1034-1043); the head norm and the
// rotation are those of its attention layer.
//
// Write (qh_attn_prep_paged), per token and head row x of D values:
//   n_c   = x_c rsqrt(mean(x^2) + eps) (1 + w_c)                 (q and k, optional)
//   y_i   = n_i cos - n_{i+h} sin,  y_{i+h} = n_{i+h} cos + n_i sin,   i < h = rot/2,
//           at the angle of column i and the position on pair i's axis
//   q     : y in bf16 or fp32;   K, V : y to slot (page, head, at % page_size),
//           as bf16, or as E4M3 codes e4m3(448 y / amax) with the scale amax / 448,
//           amax over the row's finite values (E4M3 has no infinity: a value that is
//           not finite is stored as NaN and leaves the rest of its row as it is); where
//           amax / 448 is below 2^-100 the scale is that, and the codes e4m3(y 2^100)
// q and bf16 rows in fp32 with one rounding at the end: the intermediate bf16 roundings
// of the dense path (which the reference's tensors have) would be rounded again to three
// mantissa bits here, and a second rounding moves a value in 16 to another code.
// E4M3 codes of V are those of the exact quotient: it is one of bf16 numbers, often a tie between
// two codes and otherwise further from one than fp32's correct rounding moves it.  K's quotient, in
// which the factor rsqrt(..) cancels, is computed in 64 bits (as fast as 32 here) and rounded to fp32
// then, which puts back the ties that the reciprocal moved; its code may be the exact quotient's
// neighbour where that lies within 2^-24 of itself from the border between the two.
#include <algorithm>
#include <type_traits>

#include "qh_common.h"
#include "qh_paged.h"

namespace {

// The axis whose position turns pair i.
__device__ __forceinline__ int axis_of(const qh_rope_axes& r, int i) {
  if (r.interleaved) {
    const int a = i % r.n_axes;
    const int s = a == 0 ? r.section[0] : a == 1 ? r.section[1] : a == 2 ? r.section[2] : r.section[3];
    return i < r.n_axes * s ? a : 0;
  }
  int a = 0, end = 0;
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    end += r.section[j];
    a += (j + 1 < r.n_axes && i >= end) ? 1 : 0;
  }
  return a;
}

constexpr float kMinScale = 7.8886090522101181e-31f;  // 2^-100

// Sum and maximum over the row's LPR (16 or 32) lanes, in all of them: DPP moves within
// 16 lanes, then the neighbouring 16.
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
  v = column_sum<16>(v);
  if constexpr (LPR == 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  return v;
}
template <int LPR>
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp_src<0xB1, 0xF>(v));
  v = fmaxf(v, dpp_src<0x4E, 0xF>(v));
  v = fmaxf(v, dpp_src<0x141, 0xF>(v));
  v = fmaxf(v, dpp_src<0x140, 0xF>(v));
  if constexpr (LPR == 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
  }
  return v;
}

__device__ __forceinline__ void unpack8(float (&x)[8], u32x4 u) {
  x[0] = bf_lo(u.x); x[1] = bf_hi(u.x); x[2] = bf_lo(u.y); x[3] = bf_hi(u.y);
  x[4] = bf_lo(u.z); x[5] = bf_hi(u.z); x[6] = bf_lo(u.w); x[7] = bf_hi(u.w);
}
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(x[4], x[5]), pack_bf2(x[6], x[7])};
}

// Rows that are written go past the L2 cache, where those of a prompt would push out the ones
// still to be read (3700 tokens, 16 / 4 heads of 256, fp32 q: 33.3 us with plain stores, 27.0; loads
// of this kind take 31.9, as they miss what the GEMM before left in the memory-side cache).
template <typename V>
__device__ __forceinline__ void put(V x, void* p) {
  __builtin_nontemporal_store(x, (V*)p);
}

constexpr int kPrepTokens = 4;  // tokens of a workgroup, at most
constexpr int kPrepMaxT = (1 << 26) - 64;  // 256 threads of every fourth token: fewer than 2^32 of a launch

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// row_max of 64-bit values.
template <int LPR>
__device__ __forceinline__ double row_max(double v) {
  v = fmax(v, dpp_f64<0xB1>(v));
  v = fmax(v, dpp_f64<0x4E>(v));
  v = fmax(v, dpp_f64<0x141>(v));
  v = fmax(v, dpp_f64<0x140>(v));
  if constexpr (LPR == 32) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    v = fmax(__builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]),
             __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]));
  }
  return v;
}

// A row's 8 values of this lane as codes, and its scale (without the factor that cancels).
// V: 448 x / amax as (x 7/8) / (amax 2^-9), both exact: the quotient by a reciprocal,
// corrected by its residual.
__device__ __forceinline__ u32x2 e4m3_row(const float (&x)[8], float amax, float& scale) {
  const float s0 = amax * (1.0f / 448.0f);         // amax / 448, with its residual's correction
  scale = fmaf(fmaf(-s0, 448.0f, amax), 1.0f / 448.0f, s0);
  const bool tiny = scale < kMinScale;
  if (tiny) scale = kMinScale;
  const float num = tiny ? 1.0f : 0.875f, den = tiny ? kMinScale : amax * 0.001953125f;
  const float r0 = __builtin_amdgcn_rcpf(den), r = fmaf(fmaf(-den, r0, 1.0f), r0, r0);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = x[i] * num, q0 = v * r;
    q[i] = copysignf(fmaf(fmaf(-q0, den, v), r, q0), v);  // of -0 the correction makes +0
  }
  return u32x2{e4m3x4(q[0], q[1], q[2], q[3]), e4m3x4(q[4], q[5], q[6], q[7])};
}
// K: 64 bits; `factor` is what the values were not multiplied by (the norm's rsqrt, or 1).
__device__ __forceinline__ u32x2 e4m3_row(const double (&x)[8], double amax, float factor, float& scale) {
  const double s = amax * factor * (1.0 / 448.0);
  const bool tiny = !(s >= (double)kMinScale);     // or a NaN: every value is one
  scale = tiny ? kMinScale : (float)s;
  const double r = tiny ? (double)factor / kMinScale : 448.0 / amax;
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = (float)(x[i] * r);
  return u32x2{e4m3x4(q[0], q[1], q[2], q[3]), e4m3x4(q[4], q[5], q[6], q[7])};
}

// D / 8 lanes take a row, 16 bytes of input each.  A thread has the same R heads in each of
// its workgroup's tokens (blockIdx.y: which heads), so that what a head needs is found
// once; the next token's rows are under way while one is computed.  Where the tokens'
// rows go and the cos and sin of their pairs (which the axes gather from up to four rows
// of the tables) are found once a token and kept in LDS, behind the request for the
// first rows.  For prompts HBM bounds it, with the arithmetic close behind (3700 tokens of 16 / 4
// heads of 256 into E4M3 with fp32 q: 27 to 30 us, 3.9 to 4.2 TB/s, the VALU busy half of
// it); for single tokens the chain position -> table and index -> page -> row (4.9 us).
template <int D, int R>
__global__ __launch_bounds__(256) void paged_prep_kernel(QhPagedPrepParams p, int tokens) {
  constexpr int LPR = D / 8, RPB = 256 / LPR;  // lanes of a row, rows of a pass
  __shared__ __align__(16) float s_cos[kPrepTokens * D / 2], s_sin[2][kPrepTokens * D / 2];  // [0]: -sin
  __shared__ __align__(16) float s_w[2][D];    // 1 + w of q and k (E4M3: w of k)
  __shared__ long long s_row[kPrepTokens];     // the token's slot in its page's first head, -1: left out
  const int tid = threadIdx.x, t0 = blockIdx.x * tokens, nt = min(tokens, p.T - t0);
  const int nq = p.q ? p.n_heads : 0, Hkv = p.c.n_kv, rows = nq + 2 * Hkv;
  const int half = p.rope.rot >> 1;
  const int ln = tid % LPR, c0 = ln * 8;

  // The thread's heads: q (kind 0), k (1), v (2) or none (3).
  int kind[R], head[R];
  const uint16_t* src[R];
  long long ts[R];
  u32x4 next[R];
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int row = (int)(blockIdx.y * R + u) * RPB + tid / LPR;
    kind[u] = row < nq ? 0 : row < nq + Hkv ? 1 : row < rows ? 2 : 3;
    head[u] = row - (kind[u] == 0 ? 0 : kind[u] == 1 ? nq : nq + Hkv);
    if (kind[u] == 3) head[u] = 0;
    src[u] = kind[u] == 0 ? p.q + head[u] * p.q_hs : (kind[u] == 1 ? p.k : p.v) + (long long)head[u] * D;
    ts[u] = kind[u] == 0 ? p.q_ts : kind[u] == 1 ? p.k_ts : p.v_ts;
    src[u] += t0 * ts[u] + c0;
    next[u] = *(const u32x4*)src[u];
  }
  // Where token t's rows go.  A row of padding, or an index outside its range: nowhere (it looks
  // at the table's first entry, which is there: no launch without a sequence or a page of its table).
  if (tid < nt) {
    const int t = t0 + tid, s = p.seq ? p.seq[t] : t, at = p.at[t];
    bool ok = s >= 0 && s < p.c.n_seqs && at >= 0 && at < p.c.capacity;
    const int pg = page_of(p.c, ok ? at : 0), id = p.c.pages[(size_t)(ok ? s : 0) * p.c.max_pages + pg];
    ok = ok && id >= 0 && id < p.c.n_pages;
    for (int a = 0; a < p.rope.n_axes; ++a) {
      const int x = p.pos[(size_t)a * p.T + t];
      ok = ok && x >= 0 && x < p.rope.max_pos;
    }
    s_row[tid] = ok ? (long long)id * Hkv * p.c.page_size + (at - pg * p.c.page_size) : -1;
  }
  for (int i = tid; i < nt * half; i += 256) {
    const int t = i / half, pair = i - t * half;
    const int x = p.pos[(size_t)axis_of(p.rope, pair) * p.T + t0 + t];
    const size_t e = (size_t)min(max(x, 0), p.rope.max_pos - 1) * p.rope.rot + pair;
    const float sn = p.rope.sin_t[e];
    s_cos[i] = p.rope.cos_t[e];
    s_sin[0][i] = -sn;
    s_sin[1][i] = sn;
  }
  if (tid < D) {
    s_w[0][tid] = p.q_norm_w ? 1.0f + p.q_norm_w[tid] : 1.0f;
    const float w = p.k_norm_w ? p.k_norm_w[tid] : 0.0f;
    s_w[1][tid] = p.c.ks ? w : 1.0f + w;       // E4M3: 1 + w in 64 bits, below
  }
  __syncthreads();

  const int lane = tid & 63, dl = half / 8;    // rot % 16 == 0: a pair's two halves are whole lanes apart
  const bool lower = c0 < half, turned = c0 < 2 * half;
  const int from = 4 * (lower ? lane + dl : turned ? lane - dl : lane);
  for (int t = 0; t < nt; ++t) {
    u32x4 raw[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      raw[u] = next[u];
      if (t + 1 < nt) next[u] = *(const u32x4*)(src[u] + (t + 1) * ts[u]);
    }
    const long long base = s_row[t];
    if (base < 0) continue;
#pragma unroll
    for (int u = 0; u < R; ++u) {
      float x[8];
      unpack8(x, raw[u]);
      const bool normed = kind[u] == 0 ? p.q_norm_w != nullptr : kind[u] == 1 && p.k_norm_w;
      const bool wide = kind[u] == 1 && p.c.ks;  // E4M3 rows of K: x stays as it is for now
      float rs = 1.0f;
      if (normed) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
        rs = rsqrtf(row_sum<LPR>(ss) * (1.0f / D) + p.eps);
        if (!wide) {
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const f32x4 w = *(const f32x4*)(s_w[kind[u]] + c0 + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i + k] = x[i + k] * rs * w[k];
          }
        }
      }
      float y[8] = {};
      const bool turn = half > 0 && kind[u] < 2 && turned;
      const int e = turn ? t * half + (lower ? c0 : c0 - half) : 0;
      if (half > 0 && __any(kind[u] < 2)) {
        // every lane of the wave takes part: its rows may be of different kinds
#pragma unroll
        for (int i = 0; i < 8; ++i)
          y[i] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(x[i])));
        if (turn && !wide) {
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const f32x4 cs = *(const f32x4*)(s_cos + e + i), sn = *(const f32x4*)(s_sin[lower ? 0 : 1] + e + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i + k] = x[i + k] * cs[k] + y[i + k] * sn[k];
          }
        }
      }
      if (kind[u] == 0) {
        const size_t o = ((size_t)(t0 + t) * p.n_heads + head[u]) * D + c0;
        if (p.q_f32) {
          put(f32x4{x[0], x[1], x[2], x[3]}, (float*)p.q_out + o);
          put(f32x4{x[4], x[5], x[6], x[7]}, (float*)p.q_out + o + 4);
        } else {
          put(pack8(x), (uint16_t*)p.q_out + o);
        }
        continue;
      }
      if (kind[u] == 3) continue;
      void* dst = kind[u] == 1 ? p.c.k : p.c.v;
      const long long row = base + (long long)head[u] * p.c.page_size;
      if (!p.c.ks) {
        put(pack8(x), (uint16_t*)dst + row * D + c0);
        continue;
      }
      float scale;
      u32x2 codes;
      if (wide && (normed || half > 0)) {
        double z[8];
        const int other = turn ? (lower ? c0 + half : c0 - half) : c0;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const f32x4 w = *(const f32x4*)(s_w[1] + c0 + i), wo = *(const f32x4*)(s_w[1] + other + i);
          const f32x4 cs = *(const f32x4*)(s_cos + e + i), sn = *(const f32x4*)(s_sin[lower ? 0 : 1] + e + i);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const double v = x[i + k] * (1.0 + w[k]);
            z[i + k] = turn ? v * cs[k] + y[i + k] * (1.0 + wo[k]) * sn[k] : v;
            if (!(rs < INFINITY)) z[i + k] = NAN;  // a NaN in the row: the norm is NaN
          }
        }
        double a = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmax(a, fabs(z[i]));   // of a NaN and a number: the number
        a = row_max<LPR>(a);
        if (a == INFINITY) {                   // the scale is that of the finite values, an infinity a NaN
          a = 0.0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            z[i] = fabs(z[i]) < INFINITY ? z[i] : NAN;
            a = fmax(a, fabs(z[i]));
          }
          a = row_max<LPR>(a);
        }
        codes = e4m3_row(z, a, rs, scale);
      } else {
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(x[i]));
        a = row_max<LPR>(a);
        if (a == INFINITY) {
          a = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = fabsf(x[i]) < INFINITY ? x[i] : NAN;
            a = fmaxf(a, fabsf(x[i]));
          }
          a = row_max<LPR>(a);
        }
        codes = e4m3_row(x, a, scale);
      }
      if (ln == 0) (kind[u] == 1 ? p.c.ks : p.c.vs)[row] = scale;
      put(codes, (uint8_t*)dst + row * D + c0);
    }
  }
}

// Read back (qh_kv_read_paged): 8 values of a cached row a lane, so that each store writes
// whole cache lines, K and V side by side, kReadRows rows of each under way together.  A
// workgroup takes positions blockIdx.x, blockIdx.x + gridDim.x, ... (in units of its rows) of
// one sequence and KV head.  HBM bounds it: 61700 positions of 4 heads of 256 in E4M3 take 69 us
// (5.5 TB/s), 82 with 16 values a lane, whose stores write half lines, and 75 with plain stores
// (bf16, which asks for twice as much for each store: 35 us with plain ones, 37 without).
constexpr int kReadRows = 2;
template <int D, bool FP8>
__global__ __launch_bounds__(256) void paged_read_kernel(QhPagedReadParams p) {
  using W = typename std::conditional<FP8, u32x2, u32x4>::type;  // 8 values
  constexpr int LPR = D / 8, RPB = 256 / LPR * kReadRows;
  const int pair = blockIdx.y, b = pair / p.c.n_kv, head = pair - b * p.c.n_kv;
  const int n = min(min(p.last[b], p.max_seq - 1), p.c.capacity - 1) + 1;
  const int* pages = p.c.pages + (size_t)b * p.c.max_pages;
  const int mine = threadIdx.x / LPR, c = threadIdx.x % LPR * 8;
  for (int p0 = blockIdx.x * RPB; p0 < n; p0 += gridDim.x * RPB) {
    long long row[kReadRows];
    W k[kReadRows], v[kReadRows];
    float ks[kReadRows], vs[kReadRows];
    bool ok[kReadRows];
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
      const int pos = p0 + mine + u * (256 / LPR), at = min(pos, n - 1), pg = page_of(p.c, at), id = pages[pg];
      ok[u] = pos < n && (unsigned)id < (unsigned)p.c.n_pages;
      row[u] = ((long long)(ok[u] ? id : 0) * p.c.n_kv + head) * p.c.page_size + (at - pg * p.c.page_size);
    }
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
      const size_t o = (size_t)row[u] * D + c;
      k[u] = __builtin_nontemporal_load((const W*)((const char*)p.c.k + o * (FP8 ? 1 : 2)));
      v[u] = __builtin_nontemporal_load((const W*)((const char*)p.c.v + o * (FP8 ? 1 : 2)));
      ks[u] = FP8 ? p.c.ks[row[u]] : 1.0f;
      vs[u] = FP8 ? p.c.vs[row[u]] : 1.0f;
    }
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
      if (!ok[u]) continue;
      const size_t o = ((size_t)pair * p.max_seq + p0 + mine + u * (256 / LPR)) * D + c;
      if constexpr (FP8) {
        auto four = [](uint32_t x, float s) {
          const qh_f32x2 lo = e4m3x2_lo_f32(x), hi = e4m3x2_hi_f32(x);
          return u32x2{pack_bf2(lo.x * s, lo.y * s), pack_bf2(hi.x * s, hi.y * s)};
        };
        const u32x2 k0 = four(k[u].x, ks[u]), k1 = four(k[u].y, ks[u]);
        const u32x2 v0 = four(v[u].x, vs[u]), v1 = four(v[u].y, vs[u]);
        put(u32x4{k0.x, k0.y, k1.x, k1.y}, p.k_out + o);
        put(u32x4{v0.x, v0.y, v1.x, v1.y}, p.v_out + o);
      } else {
        *(u32x4*)(p.k_out + o) = k[u];
        *(u32x4*)(p.v_out + o) = v[u];
      }
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int qh_paged_view(const qh_paged_cache* c, const int* pages, int n_seqs, int max_pages, const char* what,
                  QhPagedView* out) {
  if (!c || !c->k || !c->v) {
    qh_set_error("%s: null cache", what);
    return -1;
  }
  if (c->head_dim != 128 && c->head_dim != 256) {
    qh_set_error("%s: head_dim=%d unsupported (128 or 256)", what, c->head_dim);
    return -1;
  }
  if (c->n_pages < 1 || c->n_kv < 1 || c->n_kv > kPagedMaxUnits || c->page_size < 8 || c->page_size % 8 != 0) {
    qh_set_error("%s: n_pages=%d n_kv=%d page_size=%d (page_size must be a positive multiple of 8)", what, c->n_pages,
                 c->n_kv, c->page_size);
    return -1;
  }
  if (c->fp8 ? (!c->k_scale || !c->v_scale) : (c->k_scale || c->v_scale)) {
    qh_set_error("%s: scales belong to an E4M3 cache, and to every one", what);
    return -1;
  }
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale)) {
    qh_set_error("%s: cache pointers must be 16-byte aligned", what);
    return -1;
  }
  if (n_seqs < 0 || n_seqs > 65535 || max_pages < 1 ||
      (long long)max_pages * c->page_size > 0x7FFF0000LL || (n_seqs > 0 && !pages)) {
    qh_set_error("%s: n_seqs=%d max_pages=%d page_size=%d (at most 65535 sequences, 2^31 - 65536 positions each), or "
                 "no page table", what, n_seqs, max_pages, c->page_size);
    return -1;
  }
  QhPagedView v;
  v.k = c->k;
  v.v = c->v;
  v.ks = c->fp8 ? c->k_scale : nullptr;
  v.vs = c->fp8 ? c->v_scale : nullptr;
  v.n_pages = c->n_pages;
  v.page_size = c->page_size;
  v.n_kv = c->n_kv;
  const QhDiv by_page = qh_div_by((uint32_t)c->page_size);
  v.div_mul = by_page.mul;
  v.div_shift = by_page.shift;
  v.pages = pages;
  v.n_seqs = n_seqs;
  v.max_pages = max_pages;
  v.capacity = max_pages * c->page_size;
  *out = v;
  return 0;
}

int qh_launch_paged_prep(const QhPagedPrepParams& p, int D, hipStream_t st) {
  const char* what = "attn_prep_paged";
  if (p.T < 0 || p.T > kPrepMaxT || (p.q && (p.n_heads < 1 || p.n_heads > 4096)) || p.c.n_kv > 4096) {
    qh_set_error("%s: T=%d n_heads=%d n_kv=%d (at most 2^26 - 64 tokens, 4096 heads)", what, p.T, p.n_heads, p.c.n_kv);
    return -1;
  }
  if (!p.seq && p.T > p.c.n_seqs) {
    qh_set_error("%s: T=%d tokens without seq are one per sequence, n_seqs=%d", what, p.T, p.c.n_seqs);
    return -1;
  }
  if (p.T == 0) return 0;
  if (!p.k || !p.v || !p.at || (p.q && !p.q_out)) {
    qh_set_error("%s: null pointer", what);
    return -1;
  }
  if (p.q && p.q_out == p.q) {
    qh_set_error("%s: q_out must not alias q", what);
    return -1;
  }
  if (!aligned16(p.q) || !aligned16(p.k) || !aligned16(p.v) || !aligned16(p.q_out) || !aligned16(p.q_norm_w) ||
      !aligned16(p.k_norm_w) || p.q_ts % 8 || p.q_hs % 8 || p.k_ts % 8 || p.v_ts % 8) {
    qh_set_error("%s: pointers must be 16-byte aligned and strides multiples of 8", what);
    return -1;
  }
  const qh_rope_axes& r = p.rope;
  if (r.rot != 0) {
    const int half = r.rot / 2;
    if (r.rot < 0 || r.rot > D || r.rot % 16 != 0 || r.max_pos < 1 || !r.cos_t || !r.sin_t || !p.pos) {
      qh_set_error("%s: rot=%d (a multiple of 16, at most head_dim=%d) max_pos=%d, or a null table", what, r.rot, D,
                   r.max_pos);
      return -1;
    }
    if (r.n_axes < 1 || r.n_axes > 4) {
      qh_set_error("%s: n_axes=%d (1 to 4)", what, r.n_axes);
      return -1;
    }
    long long sum = 0;
    for (int a = 0; a < r.n_axes; ++a) {
      // interleaved: axis a > 0 turns pairs a, a + n_axes, ...: its last one has to exist
      if (r.section[a] < 0 || r.section[a] > half ||
          (r.interleaved && a > 0 && r.section[a] > 0 && a + r.n_axes * (r.section[a] - 1) >= half)) {
        qh_set_error("%s: section[%d]=%d does not fit rot/2=%d pairs", what, a, r.section[a], half);
        return -1;
      }
      sum += r.section[a];
    }
    if (sum != half) {
      qh_set_error("%s: the sections add up to %lld, not to rot/2=%d", what, sum, half);
      return -1;
    }
  }
  if (p.c.n_seqs == 0) return 0;  // every token is left out, and there may be no table to look at
  const int rows = (p.q ? p.n_heads : 0) + 2 * p.c.n_kv, pass = 256 / (D / 8), passes = (rows + pass - 1) / pass;
  // A head a thread while that leaves no more than six workgroups a CU (16 / 4 heads of 256: 400
  // tokens, 1200 workgroups, 6.4 us against 7.1 with three heads a thread; 700 tokens, 2100, 10.7
  // against 8.5); then up to 4 of them, and workgroups of up to 4 tokens that still fill the CUs
  // three times (3700 tokens: 34.6 us with one, 29.8 with 2, 29.5 with 4, 32.8 with 8).
  int tokens = 1, groups = passes;
  if ((long long)p.T * passes > 1536) {
    groups = (passes + 3) / 4;
    tokens = (int)std::min<long long>(kPrepTokens, std::max<long long>(1, (long long)p.T * groups / 768));
  }
  const dim3 grid((p.T + tokens - 1) / tokens, groups);
  const int R = (passes + groups - 1) / groups;
  void (*fn)(QhPagedPrepParams, int);
  if (D == 256)
    fn = R == 1 ? paged_prep_kernel<256, 1> : R == 2 ? paged_prep_kernel<256, 2>
         : R == 3 ? paged_prep_kernel<256, 3> : paged_prep_kernel<256, 4>;
  else
    fn = R == 1 ? paged_prep_kernel<128, 1> : R == 2 ? paged_prep_kernel<128, 2>
         : R == 3 ? paged_prep_kernel<128, 3> : paged_prep_kernel<128, 4>;
  hipLaunchKernelGGL(fn, grid, dim3(256), 0, st, p, tokens);
  return 0;
}

int qh_launch_paged_read(const QhPagedReadParams& p, int D, hipStream_t st) {
  const char* what = "kv_read_paged";
  if (p.max_seq < 1 || (long long)p.c.n_seqs * p.c.n_kv > 65535) {
    qh_set_error("%s: max_seq=%d n_seqs=%d n_kv=%d (at most 65535 pairs)", what, p.max_seq, p.c.n_seqs, p.c.n_kv);
    return -1;
  }
  if (p.c.n_seqs == 0) return 0;
  if (!p.last || !p.k_out || !p.v_out) {
    qh_set_error("%s: null pointer", what);
    return -1;
  }
  if (!aligned16(p.k_out) || !aligned16(p.v_out)) {
    qh_set_error("%s: outputs must be 16-byte aligned", what);
    return -1;
  }
  const int most = std::min(p.max_seq, p.c.capacity), pairs = p.c.n_seqs * p.c.n_kv;
  const int rows = 256 / (D / 8) * kReadRows;
  const dim3 grid(std::max(1, std::min((most + rows - 1) / rows, 16384 / pairs)), pairs);
  if (D == 256) {
    if (p.c.ks) hipLaunchKernelGGL((paged_read_kernel<256, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_read_kernel<256, false>), grid, dim3(256), 0, st, p);
  } else {
    if (p.c.ks) hipLaunchKernelGGL((paged_read_kernel<128, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_read_kernel<128, false>), grid, dim3(256), 0, st, p);
  }
  return 0;
}
