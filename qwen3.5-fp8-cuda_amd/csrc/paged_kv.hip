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
//           as bf16, or as E4M3 codes e4m3(y / s) with s = max(amax / 448, 2^-100),
//           amax over the row's finite values (E4M3 has no infinity: a value that is
//           not finite is stored as NaN and leaves the rest of its row as it is)
// All in fp32 with one rounding at the end: the intermediate bf16 roundings of the
// dense path (which the reference's tensors have) would be rounded again to three
// mantissa bits here, and a second rounding moves a value in 16 to another code.
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

// Where a token's rows go: the page and the slot in it, or page -1 for a token
// that is left out (a row of padding, or an index outside its range).
struct Slot {
  int page, off;
};
__device__ __forceinline__ Slot slot_of(const QhPagedPrepParams& p, int t) {
  const int s = p.seq ? p.seq[t] : t, at = p.at[t];
  Slot r = {-1, 0};
  if (s < 0 || s >= p.c.n_seqs || at < 0 || at >= p.c.capacity) return r;
  for (int a = 0; a < p.rope.n_axes; ++a) {
    const int x = p.pos[(size_t)a * p.T + t];
    if (x < 0 || x >= p.rope.max_pos) return r;
  }
  const int pg = page_of(p.c, at);
  const int id = p.c.pages[(size_t)s * p.c.max_pages + pg];
  if (id < 0 || id >= p.c.n_pages) return r;
  r.page = id;
  r.off = at - pg * p.c.page_size;
  return r;
}

constexpr float kMinScale = 7.8886090522101181e-31f;  // 2^-100

// One wave per (token, head row): q heads, then k heads, then v heads.
template <int D>
__global__ __launch_bounds__(256) void paged_prep_kernel(QhPagedPrepParams p) {
  constexpr int NPL = D / 64;
  const int nq = p.q ? p.n_heads : 0, rows = nq + 2 * p.c.n_kv, lane = threadIdx.x & 63;
  const long long idx = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (idx >= (long long)p.T * rows) return;
  const int t = (int)(idx / rows), row = (int)(idx - (long long)t * rows);
  const Slot slot = slot_of(p, t);
  if (slot.page < 0) return;
  const int kind = row < nq ? 0 : row < nq + p.c.n_kv ? 1 : 2;  // q, k, v
  const int head = kind == 0 ? row : kind == 1 ? row - nq : row - nq - p.c.n_kv;
  const uint16_t* src = kind == 0   ? p.q + t * p.q_ts + head * p.q_hs
                        : kind == 1 ? p.k + t * p.k_ts + (long long)head * D
                                    : p.v + t * p.v_ts + (long long)head * D;
  const float* nw = kind == 0 ? p.q_norm_w : kind == 1 ? p.k_norm_w : nullptr;
  float x[NPL];
#pragma unroll
  for (int i = 0; i < NPL; ++i) x[i] = bf2f(src[lane * NPL + i]);
  if (nw) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NPL; ++i) ss = fmaf(x[i], x[i], ss);
    const float r = rsqrtf(wave_sum(ss) / (float)D + p.eps);
#pragma unroll
    for (int i = 0; i < NPL; ++i) x[i] = x[i] * r * (1.0f + nw[lane * NPL + i]);
  }
  if (kind < 2 && p.rope.rot > 0) {
    const int half = p.rope.rot >> 1, dl = half / NPL;  // rot % 16 == 0: partners are whole lanes apart
    const int c0 = lane * NPL;
    const int from = c0 < half ? lane + dl : c0 < 2 * half ? lane - dl : lane;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const float other = __shfl(x[i], from, 64);
      const int c = c0 + i;
      if (c < 2 * half) {
        const int pair = c < half ? c : c - half;
        const size_t e = (size_t)p.pos[(size_t)axis_of(p.rope, pair) * p.T + t] * p.rope.rot + pair;
        const float cs = p.rope.cos_t[e], sn = p.rope.sin_t[e];
        x[i] = c < half ? x[i] * cs - other * sn : x[i] * cs + other * sn;
      }
    }
  }
  if (kind == 0) {
    const size_t o = ((size_t)t * p.n_heads + head) * D + lane * NPL;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      if (p.q_f32) ((float*)p.q_out)[o + i] = x[i];
      else ((uint16_t*)p.q_out)[o + i] = f2bf(x[i]);
    }
    return;
  }
  const size_t r = ((size_t)slot.page * p.c.n_kv + head) * p.c.page_size + slot.off;
  void* dst = kind == 1 ? p.c.k : p.c.v;
  if (!p.c.ks) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) ((uint16_t*)dst)[r * D + lane * NPL + i] = f2bf(x[i]);
    return;
  }
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < NPL; ++i) a = fmaxf(a, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
  const float s = fmaxf(wave_max(a) / 448.0f, kMinScale);
  if (lane == 0) (kind == 1 ? p.c.ks : p.c.vs)[r] = s;
#pragma unroll
  for (int i = 0; i < NPL; i += 2) {
    const float u = fabsf(x[i]) < INFINITY ? x[i] / s : NAN;
    const float w = fabsf(x[i + 1]) < INFINITY ? x[i + 1] / s : NAN;
    ((uint16_t*)dst)[(r * D + lane * NPL + i) / 2] = (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(u, w, 0, false);
  }
}

// Read back (qh_kv_read_paged): one wave per position and KV head.
template <int D, bool FP8>
__global__ __launch_bounds__(256) void paged_read_kernel(QhPagedReadParams p) {
  constexpr int NPL = D / 64;
  const int b = blockIdx.z, head = blockIdx.y, lane = threadIdx.x & 63;
  const int pos = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int n = min(min(p.last[b], p.max_seq - 1), p.c.capacity - 1);
  if (pos > n) return;
  const int pg = page_of(p.c, pos), id = p.c.pages[(size_t)b * p.c.max_pages + pg];
  if (id < 0 || id >= p.c.n_pages) return;
  const size_t r = ((size_t)id * p.c.n_kv + head) * p.c.page_size + (pos - pg * p.c.page_size);
  const size_t o = (((size_t)b * p.c.n_kv + head) * p.max_seq + pos) * D + lane * NPL;
#pragma unroll
  for (int i = 0; i < NPL; i += 2) {
    if constexpr (FP8) {
      const uint32_t kk = ((const uint16_t*)p.c.k)[(r * D + lane * NPL + i) / 2];
      const uint32_t vv = ((const uint16_t*)p.c.v)[(r * D + lane * NPL + i) / 2];
      const qh_f32x2 kf = e4m3x2_lo_f32(kk), vf = e4m3x2_lo_f32(vv);
      const float ks = p.c.ks[r], vs = p.c.vs[r];
      *(uint32_t*)(p.k_out + o + i) = pack_bf2(kf.x * ks, kf.y * ks);
      *(uint32_t*)(p.v_out + o + i) = pack_bf2(vf.x * vs, vf.y * vs);
    } else {
      *(uint32_t*)(p.k_out + o + i) = *(const uint32_t*)((const uint16_t*)p.c.k + r * D + lane * NPL + i);
      *(uint32_t*)(p.v_out + o + i) = *(const uint32_t*)((const uint16_t*)p.c.v + r * D + lane * NPL + i);
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
  // d = page_size, s = ceil(log2 d): m = floor(2^(31+s) / d) + 1 is below 2^32 and
  // floor(x m / 2^(31+s)) = floor(x / d) for 0 <= x < 2^31 (m d - 2^(31+s) <= d <= 2^s)
  const unsigned d = (unsigned)c->page_size;
  int s = 3;
  while ((1ull << s) < d) ++s;
  v.div_mul = (uint32_t)((1ull << (31 + s)) / d + 1);
  v.div_shift = s - 1;
  v.pages = pages;
  v.n_seqs = n_seqs;
  v.max_pages = max_pages;
  v.capacity = max_pages * c->page_size;
  *out = v;
  return 0;
}

int qh_launch_paged_prep(const QhPagedPrepParams& p, int D, hipStream_t st) {
  const char* what = "attn_prep_paged";
  if (p.T < 0 || (p.q && p.n_heads < 1)) {
    qh_set_error("%s: T=%d n_heads=%d", what, p.T, p.n_heads);
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
  const long long rows = (long long)p.T * ((p.q ? p.n_heads : 0) + 2LL * p.c.n_kv), blocks = (rows + 3) / 4;
  if (blocks > 0x7FFFFFFFLL) {
    qh_set_error("%s: T=%d tokens are more than one launch takes", what, p.T);
    return -1;
  }
  if (D == 256) hipLaunchKernelGGL(paged_prep_kernel<256>, dim3((unsigned)blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(paged_prep_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, st, p);
  return 0;
}

int qh_launch_paged_read(const QhPagedReadParams& p, int D, hipStream_t st) {
  const char* what = "kv_read_paged";
  if (p.max_seq < 1 || p.c.n_kv > 65535) {
    qh_set_error("%s: max_seq=%d n_kv=%d", what, p.max_seq, p.c.n_kv);
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
  const int most = p.max_seq < p.c.capacity ? p.max_seq : p.c.capacity;
  const dim3 grid((most + 3) / 4, p.c.n_kv, p.c.n_seqs);
  if (D == 256) {
    if (p.c.ks) hipLaunchKernelGGL((paged_read_kernel<256, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_read_kernel<256, false>), grid, dim3(256), 0, st, p);
  } else {
    if (p.c.ks) hipLaunchKernelGGL((paged_read_kernel<128, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_read_kernel<128, false>), grid, dim3(256), 0, st, p);
  }
  return 0;
}
