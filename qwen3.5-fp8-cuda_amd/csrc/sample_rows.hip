// A token for each row of logits, drawn with a given random number (gfx950).
//
// For a row x of V logits with the largest M, weights w_i = exp((x_i - M) / T).  In the order of
// falling x, equal ones by their index: the first top_k are kept; of those, the ones before which
// less than top_p of their weight lies; of those, the ones with w_i >= min_p.  The first is always
// kept.  The token is the first kept index whose running sum of kept weights, in index order, is
// above u times the whole.  Temperature 0 (or below): the first of the largest.  The reference's
// sampler (main.py:49-87) is qh_sample_top_p: one row, its bf16 roundings, its own random numbers.
//
// No sort: where the cuts fall is found in a histogram of the weights.
//   1. A workgroup reads 8192 logits (once from memory, which is the bound of the whole) into 256
//      bins of a quarter of an octave of weight below its largest, counts and weights in one 64-bit
//      LDS atomic each.  The last workgroup of a row adds the histograms up.  Without filters it
//      knows in whose sum the draw lies and walks through those 8192 again; with them it knows the
//      bins (the range) in which the cuts fall.
//   2. Launched only where a filter is given: workgroups whose chunk has logits in the range put
//      them on the row's list; the row's last one selects the cuts on it, digit after digit of a
//      key of value and index, adds up what is kept of each chunk and walks through one.  A list
//      longer than its place is not written; the row itself is gone through instead.
//
// Borders between tokens lie as close as the smallest weight, so weights are 64-bit: t = 4 x
// log2(e) / T in double, floor(t) the bin, 2^((t - floor(t) - 1) / 4) from a polynomial (7.8e-14)
// as an integer of 35 bits, which any order of atomics adds up to the same sum.  A weight is
// 2^-36 off its value, alike wherever it is used.  Weights below 2^-63.75 of the largest are none.
#include "qh_common.h"
#include "qh_serve.h"

namespace {

constexpr int NT = 256;
constexpr int kChunk = 8192;           // logits of a workgroup, 32 a thread
constexpr int kRounds = kChunk / (8 * NT);
constexpr int kBins = 256;
constexpr int kList = 32768;           // places of a row's list
constexpr int kMaxChunks = kSampleRowsMaxVocab / kChunk;
constexpr double kInfT = 1e300;        // t of an infinite logit: above every finite one
constexpr uint64_t kMassMask = (1ull << 50) - 1;  // a bin: weights below bit 50, the count above
static_assert(kMaxChunks <= NT, "a thread a chunk");

struct Chunk {      // what a workgroup hands on
  double base;      // the bin of its largest logit; -infinity where there is none
  double mass;      // its weights, as multiples of a weight 2^((base + 1) / 4) / 2^35
  float top;        // the largest
  int top_at;       // its first index, where the row wants it
};

struct RowPlan {    // what the first launch decides for the second
  int done;
  int lo, hi;       // the range: bins below the row's largest
  int by_k, by_p;   // which cuts fall in it
  int n_list;       // logits in it
  int k;            // of which top-k keeps so many
  float top;
  double base;      // the row's first bin
  double total, above, below;  // weights of all bins, of those before and behind the range
};

struct Ws {
  uint64_t* hist;    // [B][chunks][kBins]
  Chunk* chunk;      // [B][chunks]
  double* sure;      // [B][chunks] weights before the range
  RowPlan* plan;     // [B]
  uint64_t* list;    // [B][kList]
  unsigned* count;   // [rows at most][4] arrivals of both launches, places taken: zero between calls
};

int n_chunks(int V) { return (V + kChunk - 1) / kChunk; }

size_t layout(int B, int V, uint8_t* base, Ws* w) {
  const size_t nc = n_chunks(V);
  size_t off = 0;
  auto take = [&](size_t bytes) { const size_t o = off; off = (off + bytes + 255) & ~(size_t)255; return base + o; };
  uint8_t* count = take((size_t)(kSampleRowsMaxRows + 1) * 16);  // in one place for calls of any size: they stay zero
  uint8_t* hist = take(B * nc * kBins * 8);
  uint8_t* chunk = take(B * nc * sizeof(Chunk));
  uint8_t* sure = take(B * nc * 8);
  uint8_t* plan = take(B * sizeof(RowPlan));
  uint8_t* list = take((size_t)B * min(kList, V) * 8);
  if (w) *w = Ws{(uint64_t*)hist, (Chunk*)chunk, (double*)sure, (RowPlan*)plan, (uint64_t*)list, (unsigned*)count};
  return off;
}

// ---- a row's settings ------------------------------------------------------------------------
struct Settings {
  double c4;       // t = x c4
  double heat, p, m;
  int k;           // 0: all
  bool first;      // the first of the largest is the token
  bool by_p, by_m;
  __device__ __forceinline__ Settings(const QhSampleRowsParams& q, int b) {
    const float t = q.temperature ? q.temperature[b] : 1.0f;
    first = !(t > 0.0f);
    heat = first ? 1.0 : (double)t;
    c4 = 4.0 * 1.4426950408889634 / heat;
    k = q.top_k ? q.top_k[b] : 0;
    if (k >= q.V || k < 0) k = 0;
    p = q.top_p ? (double)q.top_p[b] : 1.0;
    m = q.min_p ? (double)q.min_p[b] : 0.0;
    by_p = !(p >= 1.0);
    by_m = !(m <= 0.0);
    // what keeps the first alone (NaN among it)
    if (k == 1 || (by_p && !(p > 0.0)) || (by_m && !(m <= 1.0))) first = true;
  }
  __device__ __forceinline__ bool filtered() const { return !first && (k > 0 || by_p || by_m); }
};

// ---- weights -----------------------------------------------------------------------------------
constexpr double kL = 0.17328679513998632;  // ln(2) / 4
constexpr double kA0 = 34359738368.0 * 0.9170040432046712;  // 2^35 2^(-1/8)

// The bin of a logit below `base` and its weight in the bin's own units (2^35: a whole quarter of an
// octave up); false where it has none.
__device__ __forceinline__ bool weigh(float x, double c4, double base, int& bin, uint64_t& fx) {
  const double t = x == INFINITY ? kInfT : (double)x * c4;
  const double q = floor(t), d = base - q;
  if (!(d < (double)kBins)) return false;
  const double g = (t - q) - 0.5;
  // 2^(g / 4) by its series in g ln(2) / 4, |.| <= 0.0867
  double e = kL * kL * kL * kL * kL * kL * kL / 5040.0 * kA0;
  e = fma(e, g, kL * kL * kL * kL * kL * kL / 720.0 * kA0);
  e = fma(e, g, kL * kL * kL * kL * kL / 120.0 * kA0);
  e = fma(e, g, kL * kL * kL * kL / 24.0 * kA0);
  e = fma(e, g, kL * kL * kL / 6.0 * kA0);
  e = fma(e, g, kL * kL / 2.0 * kA0);
  e = fma(e, g, kL * kA0);
  e = fma(e, g, kA0);
  bin = (int)d;
  fx = (uint64_t)__double_as_longlong(e + 4503599627370496.0) & 0xFFFFFFFFFull;  // + 2^52: rounded to an integer
  return true;
}
// 2^(-j / 4)
__device__ __forceinline__ double quarter(int j) {
  const double s = (j & 2 ? 0.7071067811865476 : 1.0) * (j & 1 ? 0.8408964152537145 : 1.0);
  return ldexp(s, -(j >> 2));
}
// 2^(-j / 4) of a difference of bins that may be far (or infinite)
__device__ __forceinline__ double quarter_far(double j) { return j < 4096.0 ? quarter((int)j) : 0.0; }

// ---- logits ------------------------------------------------------------------------------------
// NaN counts as -infinity, -0 as 0.
__device__ __forceinline__ float tidy(float x) { return x == x ? x + 0.0f : -INFINITY; }

typedef u32x4 u32x4_any __attribute__((aligned(2)));

// Eight logits from index i on (-infinity behind the row's end).
template <bool F32>
__device__ __forceinline__ void load8(const QhSampleRowsParams& p, int b, int i, float (&x)[8]) {
  if constexpr (F32) {
    const float* r = (const float*)p.logits + b * p.stride + i;
    if (i + 8 <= p.V) {
      const u32x4 v = *(const u32x4_any*)r, w = *(const u32x4_any*)(r + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = tidy(__uint_as_float(v[e]));
        x[4 + e] = tidy(__uint_as_float(w[e]));
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i + e < p.V ? tidy(r[e]) : -INFINITY;
  } else {
    const uint16_t* r = (const uint16_t*)p.logits + b * p.stride + i;
    if (i + 8 <= p.V) {
      const u32x4 v = *(const u32x4_any*)r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = tidy(bf_lo(v[e]));
        x[2 * e + 1] = tidy(bf_hi(v[e]));
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i + e < p.V ? tidy(bf2f(r[e])) : -INFINITY;
  }
}
// The first index of round r of a chunk for this thread.
__device__ __forceinline__ int index_of(int chunk, int r) { return chunk * kChunk + (r * NT + (int)threadIdx.x) * 8; }

constexpr int kIndexBits = 24;  // whole digits of 8; an index takes 20 of them

// Sort key of a logit and its index: larger for a larger value, of equal ones for a smaller index.
template <bool F32>
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  const uint32_t u = __float_as_uint(x);
  uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  if (!F32) k >>= 16;
  return (uint64_t)k << kIndexBits | (uint64_t)((1 << kIndexBits) - 1 - i);
}
template <bool F32>
__device__ __forceinline__ float value_of(uint64_t key) {
  uint32_t k = (uint32_t)(key >> kIndexBits);
  if (!F32) k = k << 16 | (k & 0x8000u ? 0u : 0xFFFFu);  // of a negative value the low bits came out inverted
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ int index_of_key(uint64_t key) {
  return (1 << kIndexBits) - 1 - (int)(key & ((1 << kIndexBits) - 1));
}

// ---- workgroup sums ----------------------------------------------------------------------------
// Exclusive prefix over the threads, and the total; a fixed order of additions.
template <typename T>
__device__ __forceinline__ T block_excl(T v, T* s_w, T& total) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  T x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  T before = __shfl_up(x, 1, 64);
  if (lane == 0) before = 0;
  if (lane == 63) s_w[wid] = x;
  __syncthreads();
  T tot = 0, off = 0;
#pragma unroll
  for (int q = 0; q < NT / 64; ++q) {
    if (q == wid) off = tot;
    tot += s_w[q];
  }
  __syncthreads();
  total = tot;
  return off + before;
}
template <typename T>
__device__ __forceinline__ T block_total(T v, T* s_w) {
  T total;
  block_excl(v, s_w, total);
  return total;
}
// The least over the threads of v, the same in all.
__device__ __forceinline__ int block_min(int v, int* s_i) {
  if (threadIdx.x == 0) *s_i = 0x7FFFFFFF;
  __syncthreads();
  if (v != 0x7FFFFFFF) atomicMin(s_i, v);
  __syncthreads();
  const int r = *s_i;
  __syncthreads();
  return r;
}

__device__ __forceinline__ void publish(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t published(const uint64_t* p) {
  return __hip_atomic_load(const_cast<uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t bits(double d) { return (uint64_t)__double_as_longlong(d); }
__device__ __forceinline__ double from_bits(uint64_t u) { return __longlong_as_double((long long)u); }

struct Shared {
  uint64_t hist[kBins];
  double d[NT / 64];
  uint64_t u[NT / 64];
  int i[4];
};

// ---- the draw ----------------------------------------------------------------------------------
// Among the chunks, thread c's weighing `mass`, and then in the one that the draw falls into: the
// first index whose running sum of kept weights is above u times the whole.  kept(x, i) is a logit's
// weight, 0 where it is not kept.
template <bool F32, typename Kept>
__device__ __forceinline__ int draw(const QhSampleRowsParams& p, int b, double mass, int chunks, Shared& s, Kept kept) {
  double total;
  const double before = block_excl(mass, s.d, total);
  const float u = p.u[b];
  const double target = (u > 0.0f ? min((double)u, 1.0) : 0.0) * total;
  const bool some = (int)threadIdx.x < chunks && mass > 0.0;
  int c = block_min(some && before + mass > target ? (int)threadIdx.x : 0x7FFFFFFF, s.i);
  if (c == 0x7FFFFFFF) c = -block_min(some ? -(int)threadIdx.x : 0x7FFFFFFF, s.i);  // u = 1: the last
  if (c < 0 || c >= chunks) return -1;
  if ((int)threadIdx.x == c) s.d[0] = before;
  __syncthreads();
  double run = s.d[0];
  __syncthreads();
  int last = 0x7FFFFFFF;
  for (int r = 0; r < kRounds; ++r) {
    float x[8];
    double w[8], sum = 0.0;
    const int i0 = index_of(c, r);
    load8<F32>(p, b, i0, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = kept(x[e], i0 + e);
      sum += w[e];
      if (w[e] > 0.0) last = -(i0 + e);
    }
    double all;
    double at = run + block_excl(sum, s.d, all);
    int found = 0x7FFFFFFF;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      at += w[e];
      if (found == 0x7FFFFFFF && w[e] > 0.0 && at > target) found = i0 + e;
    }
    found = block_min(found, s.i);
    if (found != 0x7FFFFFFF) return found;
    run += all;
  }
  // the sums in another order fell short of the target: the last kept
  last = block_min(last, s.i);
  return last <= 0 ? -last : -1;
}

template <bool F32>
__device__ __forceinline__ void finish(const QhSampleRowsParams& p, int b, int token, double c4, double base, double total) {
  p.token[b] = token;
  if (!p.logprob) return;
  int bin;
  uint64_t fx;
  float x = -INFINITY;
  if (token >= 0) x = tidy(F32 ? ((const float*)p.logits)[b * p.stride + token] : bf2f(((const uint16_t*)p.logits)[b * p.stride + token]));
  const bool some = token >= 0 && weigh(x, c4, base, bin, fx);
  p.logprob[b] = some ? (float)log((double)fx * quarter(bin) / total) : -INFINITY;
}

// ---- first launch ------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(NT) void sample_rows_scan_kernel(QhSampleRowsParams p, Ws w, int chunks) {
  __shared__ Shared s;
  const int tid = threadIdx.x, b = blockIdx.y, c = blockIdx.x;
  const Settings set(p, b);
  const bool filtered = set.filtered();
  const size_t row = (size_t)b * chunks;

  float x[kRounds][8];
  float top = -INFINITY;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    load8<F32>(p, b, index_of(c, r), x[r]);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, x[r][e]);
  }
  s.hist[tid] = 0;
  top = wave_max(top);
  if ((tid & 63) == 0) s.d[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf((float)s.d[0], (float)s.d[1]), fmaxf((float)s.d[2], (float)s.d[3]));
  const double base = top == INFINITY ? kInfT : floor((double)top * set.c4);
  int top_at = 0x7FFFFFFF;
  if (set.first) {
#pragma unroll
    for (int r = kRounds - 1; r >= 0; --r)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (x[r][e] == top) top_at = index_of(c, r) + e;
    top_at = block_min(top_at, &s.i[0]);
  }
  double mass = 0.0;
  if (!set.first || p.logprob) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        int bin;
        uint64_t fx;
        if (weigh(x[r][e], set.c4, base, bin, fx)) atomicAdd((unsigned long long*)&s.hist[bin], fx | 1ull << 50);
      }
    __syncthreads();
    const uint64_t mine = s.hist[tid];
    if (filtered) publish(&w.hist[(row + c) * kBins + tid], mine);
    mass = block_total((double)(mine & kMassMask) * quarter(tid), s.d);
  }
  if (tid == 0) {
    uint64_t* o = (uint64_t*)&w.chunk[row + c];
    publish(o, bits(base));
    publish(o + 1, bits(mass));
    publish(o + 2, (uint64_t)(uint32_t)top_at << 32 | __float_as_uint(top));
  }
  if (!arrive_last(&w.count[4 * b], chunks, &s.i[0])) return;
  if (tid == 0) reset_counter(&w.count[4 * b]);

  // the row's last workgroup
  double my_base = -INFINITY, my_mass = 0.0;
  float my_top = -INFINITY;
  int my_at = 0x7FFFFFFF;
  if (tid < chunks) {
    const uint64_t* o = (const uint64_t*)&w.chunk[row + tid];
    my_base = from_bits(published(o));
    my_mass = from_bits(published(o + 1));
    const uint64_t v = published(o + 2);
    my_top = __uint_as_float((uint32_t)v);
    my_at = (int)(v >> 32);
  }
  __syncthreads();
  const float wave_top = wave_max(my_top);
  if ((tid & 63) == 0) s.d[tid >> 6] = wave_top;
  __syncthreads();
  const float row_top = fmaxf(fmaxf((float)s.d[0], (float)s.d[1]), fmaxf((float)s.d[2], (float)s.d[3]));
  __syncthreads();
  RowPlan plan = {};
  plan.done = 1;
  if (row_top == -INFINITY) {
    if (tid == 0) {
      p.token[b] = -1;
      if (p.logprob) p.logprob[b] = -INFINITY;
      w.plan[b].done = 1;
    }
    return;
  }
  const double row_base = row_top == INFINITY ? kInfT : floor((double)row_top * set.c4);
  const double scaled = my_mass > 0.0 ? my_mass * quarter_far(row_base - my_base) : 0.0;
  if (!filtered) {
    int token;
    double total;
    if (set.first) {
      token = block_min(my_top == row_top ? my_at : 0x7FFFFFFF, &s.i[0]);
      total = block_total(scaled, s.d);
    } else {
      total = block_total(scaled, s.d);
      token = draw<F32>(p, b, scaled, chunks, s, [&](float v, int) {
        int bin;
        uint64_t fx;
        return weigh(v, set.c4, row_base, bin, fx) ? (double)fx * quarter(bin) : 0.0;
      });
    }
    if (tid == 0) {
      finish<F32>(p, b, token, set.c4, row_base, total);
      w.plan[b].done = 1;
    }
    return;
  }

  // the row's histogram, a bin a thread
  uint64_t mass_fx = 0;
  int count = 0;
  {
    double* bases = (double*)s.hist;  // of up to 128 chunks
    if (tid < chunks) bases[tid] = my_base;
    __syncthreads();
    for (int q = 0; q < chunks; ++q) {
      const double off = row_base - bases[q];  // infinite for a chunk without logits
      if (!(off <= (double)tid)) continue;
      const uint64_t v = published(&w.hist[(row + q) * kBins + (tid - (int)off)]);
      mass_fx += v & kMassMask;
      count += (int)(v >> 50);
    }
    __syncthreads();
  }
  const double weight = (double)mass_fx * quarter(tid);
  double total;
  const double excl = block_excl(weight, s.d, total);
  uint64_t n_all;
  const uint64_t n_excl = block_excl((uint64_t)count, s.u, n_all);
  const int none = 0x7FFFFFFF;
  int lo = none, hi = none;
  plan.by_k = set.k > 0 && (uint64_t)set.k < n_all;
  plan.by_p = set.by_p;
  double p_of = total;
  if (plan.by_k) {
    lo = hi = block_min(n_excl + count >= (uint64_t)set.k ? tid : none, &s.i[0]);
    if (tid == hi) s.d[0] = excl;
    __syncthreads();
    p_of = s.d[0];  // top-p's share is of these at least
    __syncthreads();
  }
  if (plan.by_p) {
    lo = block_min(count > 0 && excl + weight >= set.p * p_of ? tid : none, &s.i[0]);
    if (lo == none) lo = -block_min(count > 0 ? -tid : none, &s.i[0]);
    if (!plan.by_k) hi = lo;
    else lo = min(lo, hi);
  }
  if (set.by_m && row_top != INFINITY) {
    // the bin of the least weight that is kept, and one on both sides
    const double least = row_base - floor((double)row_top * set.c4 + 4.0 * log2(set.m));
    const int jm = least < (double)kBins ? (int)least : kBins;
    const int m_lo = max(jm - 1, 0), m_hi = jm + 1;
    if (m_hi < lo) {  // above the other cuts
      lo = m_lo;
      hi = m_hi;
      plan.by_k = plan.by_p = 0;
    } else {
      lo = min(lo, m_lo);
    }
  }
  if (lo >= kBins) {  // nothing is cut
    const int token = draw<F32>(p, b, scaled, chunks, s, [&](float v, int) {
      int bin;
      uint64_t fx;
      return weigh(v, set.c4, row_base, bin, fx) ? (double)fx * quarter(bin) : 0.0;
    });
    if (tid == 0) {
      finish<F32>(p, b, token, set.c4, row_base, total);
      w.plan[b].done = 1;
    }
    return;
  }
  hi = min(hi, kBins - 1);
  plan.above = block_total(tid < lo ? weight : 0.0, s.d);
  plan.below = block_total(tid > hi ? weight : 0.0, s.d);
  plan.n_list = (int)block_total((uint64_t)(tid >= lo && tid <= hi ? count : 0), s.u);
  const int n_above = (int)block_total((uint64_t)(tid < lo ? count : 0), s.u);
  if (tid == 0) {
    plan.done = 0;
    plan.lo = lo;
    plan.hi = hi;
    plan.k = set.k - n_above;
    plan.top = row_top;
    plan.base = row_base;
    plan.total = total;
    w.plan[b] = plan;
  }
}

// ---- second launch -----------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(NT) void sample_rows_cut_kernel(QhSampleRowsParams p, Ws w, int chunks, int places) {
  __shared__ Shared s;
  __shared__ unsigned s_count[256];
  __shared__ uint64_t s_kept[kMaxChunks];
  const int tid = threadIdx.x, b = blockIdx.y, c = blockIdx.x;
  const RowPlan plan = w.plan[b];
  if (plan.done) return;
  const Settings set(p, b);
  const size_t row = (size_t)b * chunks;
  uint64_t* list = w.list + (size_t)b * places;
  const bool listed = plan.n_list <= places;

  {  // this chunk's weight before the range, and its logits in the range
    const double off = plan.base - w.chunk[row + c].base;
    double sure = 0.0;
    int n = 0;
    if (off < (double)kBins) {
      const uint64_t v = w.hist[(row + c) * kBins + tid];
      const int j = tid + (int)off;
      if (j < plan.lo) sure = (double)(v & kMassMask) * quarter(j);
      else if (j <= plan.hi) n = (int)(v >> 50);
    }
    sure = block_total(sure, s.d);
    n = (int)block_total((uint64_t)n, s.u);
    if (n > 0 && listed) {
      if (tid == 0) {
        s.i[1] = (int)__hip_atomic_fetch_add(&w.count[4 * b + 2], (unsigned)n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s.i[2] = 0;
      }
      __syncthreads();
      const int first = s.i[1];
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        float x[8];
        load8<F32>(p, b, index_of(c, r), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          int bin;
          uint64_t fx;
          if (weigh(x[e], set.c4, plan.base, bin, fx) && bin >= plan.lo && bin <= plan.hi) {
            const int at = first + atomicAdd(&s.i[2], 1);
            if (at < places) publish(&list[at], key_of<F32>(x[e], index_of(c, r) + e));
          }
        }
      }
    }
    if (tid == 0) publish((uint64_t*)&w.sure[row + c], bits(sure));
  }
  if (!arrive_last(&w.count[4 * b + 1], chunks, &s.i[0])) return;
  if (tid == 0) {
    reset_counter(&w.count[4 * b + 1]);
    reset_counter(&w.count[4 * b + 2]);
  }

  // The row's last workgroup.  Weights of the range in units of its first bin's, 2^-unit: whole
  // numbers whose sum stays below 2^53.
  int unit = 53;
  while ((1ll << (53 - unit)) < plan.n_list) --unit;
  const double to_units = ldexp(1.0 / quarter(plan.lo & 3), unit - 35 + (plan.lo >> 2));
  auto in_range = [&](float x, uint64_t& fx) {
    int bin;
    if (!weigh(x, set.c4, plan.base, bin, fx) || bin < plan.lo || bin > plan.hi) return false;
    fx = (uint64_t)rint(ldexp((double)fx, unit - 35) * quarter(bin - plan.lo));
    return true;
  };
  // fn(key, weight) for every logit of the range
  auto each = [&](auto fn) {
    uint64_t fx;
    if (listed) {
      for (int i = tid; i < plan.n_list; i += NT) {
        const uint64_t key = published(&list[i]);
        if (in_range(value_of<F32>(key), fx)) fn(key, fx);
      }
    } else {
      for (int q = 0; q < chunks; ++q)
        for (int r = 0; r < kRounds; ++r) {
          float x[8];
          load8<F32>(p, b, index_of(q, r), x);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (in_range(x[e], fx)) fn(key_of<F32>(x[e], index_of(q, r) + e), fx);
        }
    }
  };
  // The least key such that the keys from it up, of those from `least` up, are `want` (a number of
  // them, or of weight): digit after digit from the top, until one key is left.
  auto select = [&](bool by_weight, uint64_t least, uint64_t want) {
    uint64_t prefix = 0;
    for (int shift = F32 ? 48 : 32;; shift -= 8) {
      s_count[tid] = 0;
      s.hist[tid] = 0;
      __syncthreads();
      each([&](uint64_t key, uint64_t fx) {
        if (key < least || key >> (shift + 8) != prefix) return;
        const int digit = (int)(key >> shift) & 255;
        atomicAdd(&s_count[digit], 1u);
        if (by_weight) atomicAdd((unsigned long long*)&s.hist[digit], fx);
      });
      __syncthreads();
      const int digit = 255 - tid;
      const uint64_t mine = by_weight ? s.hist[digit] : s_count[digit];
      uint64_t all;
      const uint64_t before = block_excl(mine, s.u, all);
      const int at = block_min(s_count[digit] > 0 && before + mine >= want ? tid : 0x7FFFFFFF, &s.i[0]);
      if (at == 0x7FFFFFFF) return least;  // all of them
      if (tid == at) {
        s.u[0] = before;
        s.i[1] = (int)s_count[digit];
      }
      __syncthreads();
      want -= s.u[0];
      const int n = s.i[1];
      __syncthreads();
      prefix = prefix << 8 | (uint64_t)(255 - at);
      const uint64_t cut = prefix << shift;
      if (n == 1 || shift == 0) return cut > least ? cut : least;
    }
  };
  auto sum_from = [&](uint64_t least) {
    uint64_t mine = 0;
    each([&](uint64_t key, uint64_t fx) { mine += key >= least ? fx : 0; });
    return block_total(mine, s.u);
  };

  uint64_t cut = 0;
  if (plan.by_k) cut = select(false, 0, (uint64_t)plan.k);
  if (plan.by_p) {
    const double above = plan.above * to_units;
    const double share = set.p * (above + (double)sum_from(cut) + (plan.by_k ? 0.0 : plan.below * to_units));
    const double want = ceil(share - above);
    cut = select(true, cut, want >= 1.0 ? (uint64_t)want : 1);
  }
  auto kept = [&](uint64_t key) {
    return key >= cut && (!set.by_m || plan.top == INFINITY ||
                          exp(((double)value_of<F32>(key) - (double)plan.top) / set.heat) >= set.m);
  };
  if (tid < chunks) s_kept[tid] = 0;
  __syncthreads();
  each([&](uint64_t key, uint64_t fx) {
    if (kept(key)) atomicAdd((unsigned long long*)&s_kept[index_of_key(key) / kChunk], fx);
  });
  __syncthreads();
  double mass = 0.0;
  // back in the units of the row's first bin: whole numbers too, of that bin's weights
  const double from_units = 1.0 / to_units;
  if (tid < chunks) mass = from_bits(published((const uint64_t*)&w.sure[row + tid])) + (double)s_kept[tid] * from_units;
  const int token = draw<F32>(p, b, mass, chunks, s, [&](float x, int i) {
    int bin;
    uint64_t fx;
    if (!weigh(x, set.c4, plan.base, bin, fx) || bin > plan.hi) return 0.0;
    if (bin < plan.lo) return (double)fx * quarter(bin);
    return kept(key_of<F32>(x, i)) ? rint(ldexp((double)fx, unit - 35) * quarter(bin - plan.lo)) * from_units : 0.0;
  });
  if (tid == 0) finish<F32>(p, b, token, set.c4, plan.base, plan.total);
}

template <bool F32>
void launch(const QhSampleRowsParams& p, const Ws& w, hipStream_t st) {
  const int chunks = n_chunks(p.V);
  const dim3 grid(chunks, p.B);
  sample_rows_scan_kernel<F32><<<grid, NT, 0, st>>>(p, w, chunks);
  if (p.top_k || p.top_p || p.min_p) sample_rows_cut_kernel<F32><<<grid, NT, 0, st>>>(p, w, chunks, min(kList, p.V));
}

}  // namespace

size_t qh_sample_rows_ws_bytes(int rows, int V) { return layout(rows, V, nullptr, nullptr); }

int qh_launch_sample_rows(const QhSampleRowsParams& p, hipStream_t st) {
  Ws w;
  layout(p.B, p.V, p.ws, &w);
  if (p.f32) launch<true>(p, w, st);
  else launch<false>(p, w, st);
  return 0;
}
