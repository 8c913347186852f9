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
// Everything but the flat rows is one workgroup's work: three prefix sums over the rows and
// a copy of the pages that change hands.  What bounds it is latency: a launch, the rows'
// loads, the sums' barriers.  Sums are 64-bit: a request of 2^31 - 1 tokens is refused by its
// size, not by an overflow.
#include "qh_common.h"
#include "qh_serve.h"

namespace {

// Tokens whose flat rows the one workgroup writes itself; above, a second launch does.
constexpr int kFillInline = 4096;

// Exclusive prefix sum over the workgroup's threads, and the total.
template <int NT>
__device__ __forceinline__ int64_t block_excl(int64_t v, int64_t* s_w, int64_t& total) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) s_w[wid] = x;
  __syncthreads();
  int64_t before = 0, tot = 0;
#pragma unroll
  for (int q = 0; q < NT / 64; ++q) {
    const int64_t t = s_w[q];
    if (q < wid) before += t;
    tot += t;
  }
  __syncthreads();
  total = tot;
  return before + x - v;
}

// The last row whose prefix is at or below i (rows of nothing share their successor's prefix).
__device__ __forceinline__ int row_of(const int* prefix, int n_rows, int i) {
  int lo = 0, hi = n_rows;  // prefix[lo] <= i < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
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
  int64_t n_back;
  int64_t off = block_excl<NT>(back[0] + back[1], s_w, n_back);
  s_back[2 * tid] = cap_int(off);
  s_back[2 * tid + 1] = cap_int(off + back[0]);
  if (tid == NT - 1) s_back[2 * NT] = cap_int(n_back);
  const int64_t n_free = min(n_free0 + n_back, (int64_t)p.n_pages);

#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t held = (uint32_t)(len[e] + p.page_size - 1) / (uint32_t)p.page_size;
    s_held[2 * tid + e] = (int)held;
    const int64_t end = len[e] + tok[e];
    // the sum fits 32 bits where it is not refused
    need[e] = end <= capacity ? (int64_t)((uint32_t)(end + p.page_size - 1) / (uint32_t)p.page_size) - held : 0;
    if (end > capacity || need[e] > n_free || tok[e] > p.T) need[e] = tok[e] = 0;
  }
  int64_t n_need, first = block_excl<NT>(need[0] + need[1], s_w, n_need);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    first += need[e];
    if (need[e] > 0 && first > n_free) tok[e] = need[e] = 0;
  }
  if (flat) {
    int64_t n_tok;
    off = block_excl<NT>(tok[0] + tok[1], s_w, n_tok);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      off += tok[e];
      if (tok[e] > 0 && off > p.T) tok[e] = need[e] = 0;
    }
  }
  // the served rows alone: first those of the pages, then those of the tokens
  first = block_excl<NT>(need[0] + need[1], s_w, n_need);
  int64_t n_tok;
  off = block_excl<NT>(tok[0] + tok[1], s_w, n_tok);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int b = 2 * tid + e;
    s_need[b] = (int)first;
    s_tok[b] = (int)off;
    s_len[b] = (int)len[e];
    if (b < S) {
      p.length_out[b] = (int)(len[e] + tok[e]);
      if (p.last) p.last[b] = (int)(len[e] + tok[e]) - 1;
      if (flat) p.start[b] = (int)off;
      else p.at[b] = tok[e] > 0 ? (int)len[e] : -1;
    }
    first += need[e];
    off += tok[e];
  }
  if (tid == NT - 1) {
    s_need[2 * NT] = (int)n_need;
    s_tok[2 * NT] = (int)n_tok;
  }
  if (tid == 0) {
    *p.n_free_out = (int)(n_free - n_need);
    if (flat) p.start[S] = (int)n_tok;
  }
  __syncthreads();

  for (int i = tid; i < n_free - n_free0; i += NT) {
    const int b = row_of(s_back, 2 * NT, i);
    p.free_pages[n_free0 + i] = p.pages[(size_t)b * p.max_pages + (i - s_back[b])];
  }
  __syncthreads();  // what was given back may be taken again, into tables that it was read from
  for (int i = tid; i < n_need; i += NT) {
    const int b = row_of(s_need, 2 * NT, i);
    p.pages[(size_t)b * p.max_pages + s_held[b] + (i - s_need[b])] = p.free_pages[n_free - 1 - i];
  }
  if (flat && p.T <= kFillInline) {
    for (int t = tid; t < p.T; t += NT) {
      const bool there = t < n_tok;
      const int b = there ? row_of(s_tok, 2 * NT, t) : -1;
      p.seq[t] = b;
      p.at[t] = there ? s_len[b] + (t - s_tok[b]) : -1;
    }
  }
}

// The flat rows of a longer step, from what the workgroup above wrote: row b's tokens end at
// position length_out[b] - 1.
__global__ __launch_bounds__(256) void tables_fill_kernel(QhTablesParams p) {
  __shared__ int s_tok[kTablesMaxRows + 1];
  for (int b = threadIdx.x; b <= p.n_rows; b += 256) s_tok[b] = p.start[b];
  __syncthreads();
  const int n_tok = s_tok[p.n_rows];
  for (int t = blockIdx.x * 1024 + threadIdx.x, e = 0; e < 4 && t < p.T; ++e, t += 256) {
    const bool there = t < n_tok;
    const int b = there ? row_of(s_tok, p.n_rows, t) : -1;
    p.seq[t] = b;
    p.at[t] = there ? p.length_out[b] - (s_tok[b + 1] - t) : -1;
  }
}

}  // namespace

int qh_launch_tables(const QhTablesParams& p, hipStream_t st) {
  if (p.n_rows <= 512) tables_step_kernel<256><<<1, 256, 0, st>>>(p);
  else tables_step_kernel<1024><<<1, 1024, 0, st>>>(p);
  if (p.seq && p.T > kFillInline) tables_fill_kernel<<<(p.T + 1023) / 1024, 256, 0, st>>>(p);
  return 0;
}
