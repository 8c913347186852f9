// Decode attention over a paged KV cache (gfx950): one new token of each sequence
// of a batch, GQA, rows in bf16 or in E4M3 with a scale per row.  No counterpart in
// the reference, whose decode attention reads one dense bf16 cache (layer_mid_attn,
// qwen3_infer/csrc/fused_kernels.cu:1224-1297).
//
//   s_j = q_h . k_j / sqrt(D),  o_h = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max_j s_j,
//   over positions j = 0 .. last[b] on pages that exist;  out_h = bf16(o_h sigmoid(gate_h)),
//   zeros where no position is visible.  fp32 throughout, one rounding at the end.
#include "qh_common.h"
#include "qh_paged.h"

namespace {

// One workgroup per (kv head, sequence), one wave per query head, a position at a time.
template <int D, bool FP8>
__global__ __launch_bounds__(256) void paged_attn_kernel(QhPagedAttnParams p) {
  constexpr int NPL = D / 64;
  const int kvh = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int G = p.n_heads / p.c.n_kv, n = min(p.last[b], p.c.capacity - 1);
  const float scale = rsqrtf((float)D);
  for (int gi = wid; gi < G; gi += 4) {
    const int h = kvh * G + gi;
    float q[NPL], o[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      q[i] = bf2f(p.q[b * p.q_bs + h * p.q_hs + lane * NPL + i]);
      o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int pos = 0; pos <= n; ++pos) {
      const int pg = page_of(p.c, pos), id = p.c.pages[(size_t)b * p.c.max_pages + pg];
      if (id < 0 || id >= p.c.n_pages) continue;
      const size_t r = ((size_t)id * p.c.n_kv + kvh) * p.c.page_size + (pos - pg * p.c.page_size);
      float k[NPL], v[NPL], ks = 1.0f, vs = 1.0f;
#pragma unroll
      for (int i = 0; i < NPL; i += 2) {
        if constexpr (FP8) {
          const qh_f32x2 a = e4m3x2_lo_f32(((const uint16_t*)p.c.k)[(r * D + lane * NPL + i) / 2]);
          const qh_f32x2 c = e4m3x2_lo_f32(((const uint16_t*)p.c.v)[(r * D + lane * NPL + i) / 2]);
          k[i] = a.x; k[i + 1] = a.y; v[i] = c.x; v[i + 1] = c.y;
        } else {
          k[i] = bf2f(((const uint16_t*)p.c.k)[r * D + lane * NPL + i]);
          k[i + 1] = bf2f(((const uint16_t*)p.c.k)[r * D + lane * NPL + i + 1]);
          v[i] = bf2f(((const uint16_t*)p.c.v)[r * D + lane * NPL + i]);
          v[i + 1] = bf2f(((const uint16_t*)p.c.v)[r * D + lane * NPL + i + 1]);
        }
      }
      if constexpr (FP8) {
        ks = p.c.ks[r];
        vs = p.c.vs[r];
      }
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < NPL; ++i) dot = fmaf(q[i], k[i], dot);
      const float s = wave_sum(dot) * ks * scale;
      const float nm = fmaxf(m, s);
      const float corr = m == nm ? 1.0f : expf(m - nm), pj = expf(s - nm);
      l = l * corr + pj;
      m = nm;
#pragma unroll
      for (int i = 0; i < NPL; ++i) o[i] = o[i] * corr + pj * vs * v[i];
    }
    uint16_t* dst = p.out + ((size_t)b * p.n_heads + h) * D + lane * NPL;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      float y = l == 0.0f ? 0.0f : o[i] / l;
      if (p.gate) y *= qh_sigmoid(bf2f(p.gate[b * p.g_bs + h * p.g_hs + lane * NPL + i]));
      dst[i] = f2bf(y);
    }
  }
}

}  // namespace

size_t qh_paged_attn_ws_bytes(int n_heads, int n_kv, int D) {
  if (n_kv < 1 || n_heads < 1 || n_heads % n_kv != 0 || n_heads / n_kv > 16 || (D != 128 && D != 256)) return 0;
  return kPagedMaxUnits * sizeof(unsigned);
}

int qh_launch_paged_attn(const QhPagedAttnParams& p, int D, hipStream_t st) {
  const dim3 grid(p.c.n_kv, p.c.n_seqs);
  if (D == 256) {
    if (p.c.ks) hipLaunchKernelGGL((paged_attn_kernel<256, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_attn_kernel<256, false>), grid, dim3(256), 0, st, p);
  } else {
    if (p.c.ks) hipLaunchKernelGGL((paged_attn_kernel<128, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_attn_kernel<128, false>), grid, dim3(256), 0, st, p);
  }
  return 0;
}
