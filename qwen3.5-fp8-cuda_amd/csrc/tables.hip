// Page tables and slot maps of a batch's next step, made on the GPU (gfx950), so that a
// serving loop needs no host round trip between a step's lengths and its cache writes.
//
// With held(n) = ceil(n / page_size), row b (length n_b, t_b new tokens):
//   1. rows that are done push their held(n_b) pages on the stack of free pages, row after
//      row, and n_b = 0;
//   2. need_b = held(n_b + t_b) - held(n_b).  Rows are served in order while the pages and
//      the step's token rows last: t_b = 0 where sum_{i <= b} need_i is above the free pages
//      (and need_b > 0) or sum_{i <= b} t_i above T.  A row that could not be served alone is
//      left out of the sums, so that it holds up nobody.  Both sums grow with b, so the pages
//      of the served rows are one run of the stack;
//   3. page j of that run is the stack's j-th from the top; token i of row b has position
//      n_b + i and flat row start_b + i.
//
// One workgroup does all of it: prefix sums over the rows, a copy of the pages that change hands, the
// flat rows.  What bounds it is latency: a launch, the rows' loads, six barriers (two more where pages
// are given back, two more for flat rows), one search and one round trip a page; so four pages and
// four tokens a thread are on their way at once.  Sums are
// 64-bit: a request of 2^31 - 1 tokens is refused by its size, not by an overflow.
#include "qh_common.h"
#include "qh_scan.h"
#include "qh_serve.h"

namespace {

// Tokens whose flat rows the one workgroup writes itself; above, a second launch does (500 rows, 12000
// tokens: 14.0 us in one launch, 12.2 in two; the second takes 4).
constexpr int kFillInline = 2048;

// Exclusive prefix sum over the workgroup's threads.
template <int NT>
__device__ __forceinline__ int64_t block_excl(int64_t v, int64_t* s_w, int64_t& total) {
  const int wid = threadIdx.x >> 6;
  int64_t all;
  const int64_t excl = wave_excl(v, all);
  if ((threadIdx.x & 63) == 0) s_w[wid] = all;
  __syncthreads();
  int64_t before = 0, tot = 0;
#pragma unroll
  for (int q = 0; q < NT / 64; ++q) {
    if (q == wid) before = tot;
    tot += s_w[q];
  }
  __syncthreads();
  total = tot;
  return before + excl;
}

// The last of N rows (a power of two) whose prefix is at or below i (rows of nothing share their
// successor's prefix): as many steps for every i, so that four searches run side by side.
template <int N>
__device__ __forceinline__ int row_of(const int* prefix, int i) {
  int b = 0;
#pragma unroll
  for (int step = N / 2; step > 0; step /= 2) b = prefix[b + step] <= i ? b + step : b;
  return b;
}

__device__ __forceinline__ int cap_int(int64_t v) { return v < 0x7FFFFFFF ? (int)v : 0x7FFFFFFF; }

// Two rows a thread.
template <int NT>
__global__ __launch_bounds__(NT) void tables_step_kernel(QhTablesParams p) {
  __shared__ int s_back[2 * NT + 1];   // pages given back before row b
  __shared__ int s_need[2 * NT + 1];   // pages taken before row b
  __shared__ int s_tok[2 * NT + 1];    // tokens before row b
  __shared__ int s_held[2 * NT];       // pages row b holds at first, from which its new ones are counted
  __shared__ int s_len[2 * NT];
  __shared__ int64_t s_w[NT / 64];
  __shared__ int2 s_top[NT / 64];
  const int tid = threadIdx.x, S = p.n_rows;
  const int64_t capacity = (int64_t)p.max_pages * p.page_size;
  const bool flat = p.seq != nullptr;
  const int n_free0 = min(max(*p.n_free, 0), p.n_pages);

  int64_t len[2], tok[2], need[2], back[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int b = 2 * tid + e;
    len[e] = tok[e] = back[e] = 0;
    if (b < S) {
      len[e] = min((int64_t)max(p.length[b], 0), capacity);
      tok[e] = max(p.new_tokens[b], 0);
      if (!flat) tok[e] = min(tok[e], (int64_t)1);
      if (p.done && p.done[b] != 0) {
        back[e] = (uint32_t)(len[e] + p.page_size - 1) / (uint32_t)p.page_size;
        len[e] = 0;
      }
    }
  }
  int64_t n_back = 0, off = 0, total;
  if (__syncthreads_or(back[0] + back[1] > 0)) off = block_excl<NT>(back[0] + back[1], s_w, n_back);
  s_back[2 * tid] = cap_int(off);
  s_back[2 * tid + 1] = cap_int(off + back[0]);
  if (tid == NT - 1) s_back[2 * NT] = cap_int(n_back);
  const int n_free = (int)min(n_free0 + n_back, (int64_t)p.n_pages);

#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t held = (uint32_t)(len[e] + p.page_size - 1) / (uint32_t)p.page_size;
    s_held[2 * tid + e] = (int)held;
    const int64_t end = len[e] + tok[e];
    // the sum fits 32 bits where it is not refused
    need[e] = end <= capacity ? (int64_t)((uint32_t)(end + p.page_size - 1) / (uint32_t)p.page_size) - held : 0;
    if (end > capacity || need[e] > n_free || tok[e] > p.T) need[e] = tok[e] = 0;
  }
  // Up to the first row that is left out for its pages (or tokens) the sum of what is asked for is that of
  // what is served, and behind it nothing that would count is: sums cut at the largest one served.
  const int64_t first = block_excl<NT>(need[0] + need[1], s_w, total);
  bool served[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    served[e] = need[e] == 0 || first + (e ? need[0] : 0) + need[e] <= n_free;
    if (!served[e]) tok[e] = 0;
  }
  off = 0;
  if (flat) off = block_excl<NT>(tok[0] + tok[1], s_w, total);
  int top_need = 0, top_tok = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int64_t upto = off + (e ? tok[0] : 0) + tok[e];
    served[e] = served[e] && tok[e] > 0 && (!flat || upto <= p.T);
    if (served[e]) {
      top_need = max(top_need, need[e] > 0 ? (int)(first + (e ? need[0] : 0) + need[e]) : 0);
      top_tok = (int)upto;
    }
  }
  top_need = wave_max_int(top_need);
  top_tok = wave_max_int(top_tok);
  if ((tid & 63) == 0) s_top[tid >> 6] = int2{top_need, top_tok};
  __syncthreads();
  int n_need = 0, n_tok = 0;
#pragma unroll
  for (int q = 0; q < NT / 64; ++q) {
    n_need = max(n_need, s_top[q].x);
    n_tok = max(n_tok, s_top[q].y);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int b = 2 * tid + e;
    s_need[b] = (int)min(first + (e ? need[0] : 0), (int64_t)n_need);
    s_tok[b] = (int)min(off + (e ? tok[0] : 0), (int64_t)n_tok);
    s_len[b] = (int)len[e];
    if (b < S) {
      const int got = served[e] ? (int)tok[e] : 0;
      p.length_out[b] = (int)len[e] + got;
      if (p.last) p.last[b] = (int)len[e] + got - 1;
      if (flat) p.start[b] = s_tok[b];
      else p.at[b] = got > 0 ? (int)len[e] : -1;
    }
  }
  if (tid == NT - 1) {
    s_need[2 * NT] = n_need;
    s_tok[2 * NT] = n_tok;
  }
  if (tid == 0) {
    *p.n_free_out = n_free - n_need;
    if (flat) p.start[S] = n_tok;
  }
  __syncthreads();

  for (int i0 = tid; i0 < n_free - n_free0; i0 += 4 * NT) {
    int id[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = min(i0 + e * NT, n_free - n_free0 - 1), b = row_of<2 * NT>(s_back, i);
      id[e] = p.pages[(size_t)b * p.max_pages + (i - s_back[b])];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i0 + e * NT < n_free - n_free0) p.free_pages[n_free0 + i0 + e * NT] = id[e];
  }
  __syncthreads();  // what was given back may be taken again, into tables that it was read from
  for (int i0 = tid; i0 < n_need; i0 += 4 * NT) {
    int id[4];
    size_t to[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = min(i0 + e * NT, n_need - 1), b = row_of<2 * NT>(s_need, i);
      id[e] = p.free_pages[n_free - 1 - i];
      to[e] = (size_t)b * p.max_pages + s_held[b] + (i - s_need[b]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i0 + e * NT < n_need) p.pages[to[e]] = id[e];
  }
  if (flat && p.T <= kFillInline) {
    for (int t0 = tid; t0 < p.T; t0 += 4 * NT)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = t0 + e * NT, b = row_of<2 * NT>(s_tok, t);  // (above the last: one that is not used)
        const int at = s_len[b] + (t - s_tok[b]);
        if (t < p.T) {
          p.seq[t] = t < n_tok ? b : -1;
          p.at[t] = t < n_tok ? at : -1;
        }
      }
  }
}

// The flat rows of a longer step, from what the workgroup above wrote: row b's tokens end at
// position length_out[b] - 1.
__global__ __launch_bounds__(256) void tables_fill_kernel(QhTablesParams p) {
  __shared__ int s_tok[kTablesMaxRows + 1];
  for (int b = threadIdx.x; b <= kTablesMaxRows; b += 256) s_tok[b] = p.start[min(b, p.n_rows)];
  __syncthreads();
  const int n_tok = s_tok[kTablesMaxRows];
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= p.T) return;
  const bool there = t < n_tok;
  const int b = there ? row_of<kTablesMaxRows>(s_tok, t) : -1;
  p.seq[t] = b;
  p.at[t] = there ? p.length_out[b] - (s_tok[b + 1] - t) : -1;
}

}  // namespace

int qh_launch_tables(const QhTablesParams& p, hipStream_t st) {
  // Two rows a thread, as few threads as that allows: more make every barrier longer, also where pages and
  // tokens are the work.  256 and 1024 threads, us: a token a row, 64 rows 5.1 / 7.7, 256 6.0 / 8.1, 512
  // 7.8 / 8.3; with prompts, 64 rows 8.5 / 11.2, 256 10.0 / 12.4, 512 11.4 / 12.9.
  if (p.n_rows <= 512) tables_step_kernel<256><<<1, 256, 0, st>>>(p);
  else tables_step_kernel<1024><<<1, 1024, 0, st>>>(p);
  if (p.seq && p.T > kFillInline) tables_fill_kernel<<<(p.T + 255) / 256, 256, 0, st>>>(p);
  return 0;
}
