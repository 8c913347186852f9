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
//   1. scan: a workgroup reads 8192 logits (once from memory, which is the bound of the whole) into
//      256 bins of a quarter of an octave of weight below its largest, counts and weights in one
//      64-bit LDS atomic each; only their sum where the row has no filter.
//   2. plan: a workgroup a row adds the chunks up.  Without filters it knows in whose sum the draw
//      lies and walks through those 8192 again; with them it knows the bins (the range) in which
//      the cuts fall.
//   3. list: workgroups whose chunk has logits in the range put them on the row's list.
//   4. cut: a workgroup a row selects the cuts on its list, digit after digit of a key of value and
//      index, adds up what is kept of each chunk and walks through one.  A list longer than its
//      place is not written; the row itself is gone through instead.
// The last two are launched only where a filter is given.
//
// Borders between tokens lie as close as the smallest weight, so weights are 64-bit: t = 4 x
// log2(e) / T in double, floor(t) the bin, 2^((t - floor(t) - 1) / 4) from a polynomial (7.8e-14)
// as an integer of 35 bits, which any order of atomics adds up to the same sum.  A weight is
// 2^-36 off its value, alike wherever it is used.  Weights below 2^-63.75 of the largest are none.
#include "qh_common.h"
#include "qh_serve.h"

namespace {

constexpr int NT = 512;
constexpr int kWaves = NT / 64;
constexpr int kChunk = 8192;           // logits of a workgroup, 16 a thread
constexpr int kRounds = kChunk / (8 * NT);
constexpr int kBins = 256;
constexpr int kCopies = 4;             // of the histogram in LDS, by lane: logits crowd in few bins
constexpr int kList = 32768;           // places of a row's list
constexpr int kShort = 4096;           // entries of a list that stays in LDS
constexpr int kMaxChunks = kSampleRowsMaxVocab / kChunk;
constexpr double kInfT = 1e300;        // t of an infinite logit: above every finite one
constexpr uint64_t kMassMask = (1ull << 50) - 1;  // a bin: weights below bit 50, the count above
constexpr int kNone = 0x7FFFFFFF;
static_assert(kMaxChunks <= kBins && NT == 2 * kBins, "a thread a chunk, two a bin");

struct Chunk {      // what a workgroup hands on
  double base;      // the bin of its largest logit; -infinity where there is none
  double mass;      // its weights, as multiples of a weight 2^((base + 1) / 4) / 2^35
  float top;        // the largest
  int top_at;       // its first index, where the row wants it
};

struct RowPlan {    // what the plan says to the launches behind it
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
  unsigned* taken;   // [B] places of the list that are taken
};

int n_chunks(int V) { return (V + kChunk - 1) / kChunk; }

size_t layout(int B, int V, uint8_t* base, Ws* w) {
  const size_t nc = n_chunks(V);
  size_t off = 0;
  auto take = [&](size_t bytes) { const size_t o = off; off = (off + bytes + 255) & ~(size_t)255; return base + o; };
  uint8_t* taken = take((size_t)B * 4);
  uint8_t* hist = take(B * nc * kBins * 8);
  uint8_t* chunk = take(B * nc * sizeof(Chunk));
  uint8_t* sure = take(B * nc * 8);
  uint8_t* plan = take(B * sizeof(RowPlan));
  uint8_t* list = take((size_t)B * min(kList, V) * 8);
  if (w) *w = Ws{(uint64_t*)hist, (Chunk*)chunk, (double*)sure, (RowPlan*)plan, (uint64_t*)list, (unsigned*)taken};
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

// Sort key of a logit and its index: larger for a larger value, of equal ones for a smaller index.
// The index takes `ib` bits.
template <bool F32>
__device__ __forceinline__ uint64_t key_of(float x, int i, int ib) {
  const uint32_t u = __float_as_uint(x);
  uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  if (!F32) k >>= 16;
  return (uint64_t)k << ib | (uint64_t)((1 << ib) - 1 - i);
}
template <bool F32>
__device__ __forceinline__ float value_of(uint64_t key, int ib) {
  uint32_t k = (uint32_t)(key >> ib);
  if (!F32) k = k << 16 | (k & 0x8000u ? 0u : 0xFFFFu);  // of a negative value the low bits came out inverted
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ int index_of_key(uint64_t key, int ib) { return (1 << ib) - 1 - (int)(key & ((1 << ib) - 1)); }

// ---- workgroup sums ----------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ T wave_excl(T v, T& all) {
  const int lane = threadIdx.x & 63;
  T x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  all = __shfl(x, 63, 64);
  const T before = __shfl_up(x, 1, 64);
  return lane == 0 ? T(0) : before;
}
// Exclusive prefixes over the threads of two values, and their totals; a fixed order of additions.
template <typename A, typename B>
__device__ __forceinline__ void block_excl(A a, B b, A* s_a, B* s_b, A& a_excl, A& a_all, B& b_excl, B& b_all) {
  const int wid = threadIdx.x >> 6;
  A wa;
  B wb;
  a_excl = wave_excl(a, wa);
  b_excl = wave_excl(b, wb);
  if ((threadIdx.x & 63) == 0) {
    s_a[wid] = wa;
    s_b[wid] = wb;
  }
  __syncthreads();
  A at = 0, ao = 0;
  B bt = 0, bo = 0;
#pragma unroll
  for (int q = 0; q < kWaves; ++q) {
    if (q == wid) {
      ao = at;
      bo = bt;
    }
    at += s_a[q];
    bt += s_b[q];
  }
  __syncthreads();
  a_excl += ao;
  b_excl += bo;
  a_all = at;
  b_all = bt;
}
// The total over the threads, in a fixed order.
__device__ __forceinline__ double block_total(double v, double* s_d) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) s_d[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int q = 0; q < kWaves; ++q) t += s_d[q];
  __syncthreads();
  return t;
}
// The least over the threads, the same in all.
__device__ __forceinline__ int block_min(int v, int* s_i) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  if ((threadIdx.x & 63) == 0) s_i[threadIdx.x >> 6] = v;
  __syncthreads();
  int r = s_i[0];
#pragma unroll
  for (int q = 1; q < kWaves; ++q) r = min(r, s_i[q]);
  __syncthreads();
  return r;
}
__device__ __forceinline__ float block_max(float v, float* s_f) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) s_f[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = s_f[0];
#pragma unroll
  for (int q = 1; q < kWaves; ++q) r = fmaxf(r, s_f[q]);
  __syncthreads();
  return r;
}

struct Sums {  // LDS of the sums above
  double d[2][kWaves];
  uint64_t u[kWaves];
  float f[kWaves];
  int i[kWaves];
  double at[2];
  uint64_t n[2];
};

// ---- the draw ----------------------------------------------------------------------------------
// Among the chunks, thread c's weighing `mass`, and then in the one that the draw falls into: the
// first index whose running sum of kept weights is above u times the whole.  kept(x, i) is a logit's
// weight, 0 where it is not kept.
template <bool F32, typename Kept>
__device__ __forceinline__ int draw(const QhSampleRowsParams& p, int b, float u, double mass, int chunks, Sums& s, Kept kept,
                                    double& total) {
  double before, none, none_all;
  block_excl(mass, 0.0, s.d[0], s.d[1], before, total, none, none_all);
  const double target = (u > 0.0f ? min((double)u, 1.0) : 0.0) * total;
  const bool some = (int)threadIdx.x < chunks && mass > 0.0;
  int c = block_min(some && before + mass > target ? (int)threadIdx.x : kNone, s.i);
  if (c == kNone) c = -block_min(some ? -(int)threadIdx.x : kNone, s.i);  // u = 1: the last
  if (c < 0 || c >= chunks) return -1;
  if ((int)threadIdx.x == c) s.at[0] = before;
  float x[kRounds][8];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) load8<F32>(p, b, index_of(c, r), x[r]);
  double w[kRounds][8], sum[kRounds] = {};
  int last = kNone;
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[r][e] = kept(x[r][e], index_of(c, r) + e);
      sum[r] += w[r][e];
      if (w[r][e] > 0.0) last = -(index_of(c, r) + e);
    }
  static_assert(kRounds == 2, "two prefixes at once");
  double excl[2], all[2];
  block_excl(sum[0], sum[1], s.d[0], s.d[1], excl[0], all[0], excl[1], all[1]);
  int found = kNone;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    double at = (s.at[0] + (r ? all[0] : 0.0)) + excl[r];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      at += w[r][e];
      if (found == kNone && w[r][e] > 0.0 && at > target) found = index_of(c, r) + e;
    }
  }
  found = block_min(found, s.i);
  if (found != kNone) return found;
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

// ---- scan ------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(NT) void sample_rows_scan_kernel(QhSampleRowsParams p, Ws w, int chunks) {
  __shared__ Sums s;
  __shared__ uint64_t s_hist[kBins * kCopies];
  const int tid = threadIdx.x, b = blockIdx.y, c = blockIdx.x;
  const size_t row = (size_t)b * chunks;

  float x[kRounds][8];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) load8<F32>(p, b, index_of(c, r), x[r]);
  const Settings set(p, b);
  const bool filtered = set.filtered();
  for (int i = tid; i < kBins * kCopies; i += NT) s_hist[i] = 0;
  float top = -INFINITY;
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, x[r][e]);
  top = block_max(top, s.f);
  const double base = top == INFINITY ? kInfT : floor((double)top * set.c4);
  int top_at = kNone;
  if (set.first) {
#pragma unroll
    for (int r = kRounds - 1; r >= 0; --r)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (x[r][e] == top) top_at = index_of(c, r) + e;
    top_at = block_min(top_at, s.i);
  }
  double mass = 0.0;
  if (filtered) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        int bin;
        uint64_t fx;
        if (weigh(x[r][e], set.c4, base, bin, fx))
          atomicAdd((unsigned long long*)&s_hist[bin * kCopies + (tid & (kCopies - 1))], fx | 1ull << 50);
      }
    __syncthreads();
    if (tid < kBins) {
      uint64_t mine = 0;
#pragma unroll
      for (int q = 0; q < kCopies; ++q) mine += s_hist[tid * kCopies + q];
      w.hist[(row + c) * kBins + tid] = mine;
      mass = (double)(mine & kMassMask) * quarter(tid);
    }
  } else if (!set.first || p.logprob) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        int bin;
        uint64_t fx;
        if (weigh(x[r][e], set.c4, base, bin, fx)) mass += (double)fx * quarter(bin);
      }
  }
  mass = block_total(mass, s.d[0]);
  if (tid == 0) w.chunk[row + c] = Chunk{base, mass, top, top_at};
}

// ---- plan ----------------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(NT) void sample_rows_plan_kernel(QhSampleRowsParams p, Ws w, int chunks) {
  __shared__ Sums s;
  __shared__ uint64_t s_other[2 * kBins];
  __shared__ double s_base[kMaxChunks];
  const int tid = threadIdx.x, b = blockIdx.x;
  const size_t row = (size_t)b * chunks;
  const float u = p.u[b];
  const Settings set(p, b);
  const bool filtered = set.filtered();
  Chunk mine = {-INFINITY, 0.0, -INFINITY, kNone};
  if (tid < chunks) mine = w.chunk[row + tid];
  const float row_top = block_max(mine.top, s.f);
  if (row_top == -INFINITY) {
    if (tid == 0) {
      p.token[b] = -1;
      if (p.logprob) p.logprob[b] = -INFINITY;
      w.plan[b].done = 1;
    }
    return;
  }
  const double row_base = row_top == INFINITY ? kInfT : floor((double)row_top * set.c4);
  const double scaled = mine.mass > 0.0 ? mine.mass * quarter_far(row_base - mine.base) : 0.0;
  auto every = [&](float v, int) {
    int bin;
    uint64_t fx;
    return weigh(v, set.c4, row_base, bin, fx) ? (double)fx * quarter(bin) : 0.0;
  };
  double total;
  if (!filtered) {
    int token;
    if (set.first) {
      token = block_min(mine.top == row_top ? mine.top_at : kNone, s.i);
      total = block_total(scaled, s.d[0]);
    } else {
      token = draw<F32>(p, b, u, scaled, chunks, s, every, total);
    }
    if (tid == 0) {
      finish<F32>(p, b, token, set.c4, row_base, total);
      w.plan[b].done = 1;
    }
    return;
  }

  // the row's histogram: two threads a bin, every other chunk each, eight loads on their way at once
  uint64_t mass_fx = 0;
  int count = 0;
  {
    if (tid < chunks) s_base[tid] = mine.base;
    __syncthreads();
    const int j = tid & (kBins - 1);
    for (int q0 = tid / kBins; q0 < chunks; q0 += 16) {
      uint64_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int q = q0 + 2 * e;
        const double off = q < chunks ? row_base - s_base[q] : INFINITY;  // infinite for a chunk without logits
        const bool in = off <= (double)j;
        v[e] = w.hist[in ? (row + q) * kBins + (j - (int)off) : row * kBins];
        if (!in) v[e] = 0;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        mass_fx += v[e] & kMassMask;
        count += (int)(v[e] >> 50);
      }
    }
    if (tid >= kBins) {
      s_other[2 * j] = mass_fx;
      s_other[2 * j + 1] = (uint64_t)count;
      mass_fx = 0;
      count = 0;
    }
    __syncthreads();
    if (tid < kBins) {
      mass_fx += s_other[2 * j];
      count += (int)s_other[2 * j + 1];
    }
  }
  const double weight = tid < kBins ? (double)mass_fx * quarter(tid) : 0.0;
  double excl;
  uint64_t n_excl, n_all;
  block_excl(weight, (uint64_t)count, s.d[0], s.u, excl, total, n_excl, n_all);
  RowPlan plan = {};
  int lo = kNone, hi = kNone;
  plan.by_k = set.k > 0 && (uint64_t)set.k < n_all;
  plan.by_p = set.by_p;
  double p_of = total;
  if (plan.by_k) {
    lo = hi = block_min(n_excl + count >= (uint64_t)set.k ? tid : kNone, s.i);
    if (tid == hi) s.at[0] = excl;
    __syncthreads();
    p_of = s.at[0];  // top-p's share is of these at least
  }
  if (plan.by_p) {
    lo = block_min(count > 0 && excl + weight >= set.p * p_of ? tid : kNone, s.i);
    if (lo == kNone) lo = -block_min(count > 0 ? -tid : kNone, s.i);
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
    const int token = draw<F32>(p, b, u, scaled, chunks, s, every, total);
    if (tid == 0) {
      finish<F32>(p, b, token, set.c4, row_base, total);
      w.plan[b].done = 1;
    }
    return;
  }
  hi = min(hi, kBins - 1);
  if (tid == lo) {
    s.d[0][0] = excl;
    s.n[0] = n_excl;
  }
  if (tid == hi) {
    s.d[0][1] = excl + weight;
    s.n[1] = n_excl + count;
  }
  __syncthreads();
  if (tid == 0) {
    plan.done = 0;
    plan.lo = lo;
    plan.hi = hi;
    plan.above = s.d[0][0];
    plan.below = total - s.d[0][1];
    plan.n_list = (int)(s.n[1] - s.n[0]);
    plan.k = set.k - (int)s.n[0];
    plan.top = row_top;
    plan.base = row_base;
    plan.total = total;
    w.plan[b] = plan;
    w.taken[b] = 0;
  }
}

// ---- list ----------------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(NT) void sample_rows_list_kernel(QhSampleRowsParams p, Ws w, int chunks, int places, int ib) {
  __shared__ Sums s;
  __shared__ unsigned s_n;
  const int tid = threadIdx.x, b = blockIdx.y, c = blockIdx.x;
  const RowPlan plan = w.plan[b];
  if (plan.done) return;
  const size_t row = (size_t)b * chunks;
  uint64_t* list = w.list + (size_t)b * places;

  // this chunk's weight before the range, and how many of its logits are in the range
  const double off = plan.base - w.chunk[row + c].base;
  double sure = 0.0;
  uint64_t n = 0;
  if (off < (double)kBins && tid < kBins) {
    const uint64_t v = w.hist[(row + c) * kBins + tid];
    const int j = tid + (int)off;
    if (j < plan.lo) sure = (double)(v & kMassMask) * quarter(j);
    else if (j <= plan.hi) n = v >> 50;
  }
  double sure_excl, sure_all;
  uint64_t n_excl, n_all;
  block_excl(sure, n, s.d[0], s.u, sure_excl, sure_all, n_excl, n_all);
  if (tid == 0) w.sure[row + c] = sure_all;
  if (n_all == 0 || plan.n_list > places) return;
  float x[kRounds][8];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) load8<F32>(p, b, index_of(c, r), x[r]);
  const Settings set(p, b);
  if (tid == 0) s_n = atomicAdd(&w.taken[b], (unsigned)n_all);
  __syncthreads();
  // the range's ends as logits, a little wide: most logits need no more
  const float x_lo = (float)((plan.base - plan.hi) / set.c4), x_hi = (float)((plan.base - plan.lo + 1.0) / set.c4);
  const float slack = 1e-6f * fmaxf(fabsf(x_lo), fabsf(x_hi));
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (x[r][e] < x_lo - slack || x[r][e] > x_hi + slack) continue;
      int bin;
      uint64_t fx;
      if (weigh(x[r][e], set.c4, plan.base, bin, fx) && bin >= plan.lo && bin <= plan.hi) {
        const unsigned at = atomicAdd(&s_n, 1u);
        if (at < (unsigned)places) list[at] = key_of<F32>(x[r][e], index_of(c, r) + e, ib);
      }
    }
}

// ---- cut -----------------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(NT) void sample_rows_cut_kernel(QhSampleRowsParams p, Ws w, int chunks, int places, int ib) {
  __shared__ Sums s;
  __shared__ uint64_t s_list[kShort];
  __shared__ uint64_t s_mass[NT], s_kept[kMaxChunks];
  __shared__ unsigned s_count[NT];
  const int tid = threadIdx.x, b = blockIdx.x;
  const RowPlan plan = w.plan[b];
  if (plan.done) return;
  const Settings set(p, b);
  const size_t row = (size_t)b * chunks;
  const uint64_t* list = w.list + (size_t)b * places;
  const bool listed = plan.n_list <= places;

  // Weights of the range in units of its first bin's, 2^-unit: whole numbers whose sum stays below 2^53.
  const float u = p.u[b];
  const double sure = tid < chunks ? w.sure[row + tid] : 0.0;
  const int n_list = plan.n_list;
  const int unit = 53 - (n_list > 1 ? 32 - __clz(n_list - 1) : 0);
  const double to_units = ldexp(1.0 / quarter(plan.lo & 3), unit - 35 + (plan.lo >> 2)), from_units = 1.0 / to_units;
  auto in_range = [&](float x, uint64_t& fx) {
    int bin;
    if (!weigh(x, set.c4, plan.base, bin, fx) || bin < plan.lo || bin > plan.hi) return false;
    fx = (uint64_t)rint(ldexp((double)fx, unit - 35) * quarter(bin - plan.lo));
    return true;
  };
  if (tid < chunks) s_kept[tid] = 0;
  const bool brief = listed && n_list <= kShort;
  if (brief) {
    uint64_t v[kShort / NT];
#pragma unroll
    for (int i = 0; i < kShort / NT; ++i) v[i] = i * NT + tid < n_list ? list[i * NT + tid] : 0;
#pragma unroll
    for (int i = 0; i < kShort / NT; ++i)
      if (i * NT + tid < n_list) s_list[i * NT + tid] = v[i];
  }
  __syncthreads();
  // fn(key, weight) for every logit of the range (weight 0 where it is not wanted)
  auto each = [&](bool weights, auto fn) {
    uint64_t fx = 0;
    if (brief) {
      for (int i = tid; i < n_list; i += NT) {
        const uint64_t key = s_list[i];
        if (!weights || in_range(value_of<F32>(key, ib), fx)) fn(key, fx);
      }
    } else if (listed) {
      for (int i0 = tid; i0 < n_list; i0 += 8 * NT) {
        uint64_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = list[min(i0 + e * NT, n_list - 1)];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i0 + e * NT < n_list && (!weights || in_range(value_of<F32>(v[e], ib), fx))) fn(v[e], fx);
      }
    } else {
      for (int q = 0; q < chunks; ++q) {
        float x[kRounds][8];
#pragma unroll
        for (int r = 0; r < kRounds; ++r) load8<F32>(p, b, index_of(q, r), x[r]);
#pragma unroll
        for (int r = 0; r < kRounds; ++r)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (in_range(x[r][e], fx)) fn(key_of<F32>(x[r][e], index_of(q, r) + e, ib), fx);
      }
    }
  };

  uint64_t cut = 0;
  if (plan.by_k || plan.by_p) {
    // what all keys have in common tells nothing: digits are of the distance from the least
    uint64_t least = ~0ull, most = 0;
    each(false, [&](uint64_t key, uint64_t) {
      least = key < least ? key : least;
      most = key > most ? key : most;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t l = __shfl_xor(least, o, 64), m = __shfl_xor(most, o, 64);
      least = l < least ? l : least;
      most = m > most ? m : most;
    }
    if ((tid & 63) == 0) {
      s_mass[tid >> 6] = least;
      s_mass[kWaves + (tid >> 6)] = most;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kWaves; ++q) {
      least = s_mass[q] < least ? s_mass[q] : least;
      most = s_mass[kWaves + q] > most ? s_mass[kWaves + q] : most;
    }
    __syncthreads();
    const int key_bits = most > least ? 64 - __clzll((long long)(most - least)) : 0;
    // The least key such that those from it up, of the ones from `cut` up, are as many (or weigh as
    // much) as wanted(their sum), digit after digit of nine bits, until one key is left.
    auto select = [&](bool by_weight, auto wanted) {
      uint64_t prefix = 0, want = 0;
      int high = key_bits;  // the digits above are settled
      for (int round = 0;; ++round) {
        const int shift = max(high - 9, 0);
        s_count[tid] = 0;
        s_mass[tid] = 0;
        __syncthreads();
        each(by_weight, [&](uint64_t key, uint64_t fx) {
          const uint64_t d = key - least;
          if (key < cut || d >> high != prefix) return;
          const int digit = (int)(d >> shift) & ((1 << (high - shift)) - 1);
          atomicAdd(&s_count[digit], 1u);
          if (by_weight) atomicAdd((unsigned long long*)&s_mass[digit], fx);
        });
        __syncthreads();
        const int digit = NT - 1 - tid;
        const uint64_t n = s_count[digit], mine = by_weight ? s_mass[digit] : n;
        uint64_t before, all;
        double none, none_all;
        block_excl(mine, 0.0, s.u, s.d[0], before, all, none, none_all);
        if (round == 0) want = wanted(all);
        const int at = block_min(n > 0 && before + mine >= want ? tid : kNone, s.i);
        if (at == kNone) return;  // all of them
        if (tid == at) {
          s.n[0] = before;
          s.n[1] = n;
        }
        __syncthreads();
        want -= s.n[0];
        const uint64_t left = s.n[1];
        prefix = prefix << (high - shift) | (uint64_t)(NT - 1 - at);
        high = shift;
        if (left == 1 || shift == 0) break;
      }
      const uint64_t found = least + (prefix << high);
      cut = found > cut ? found : cut;
    };
    if (plan.by_k) select(false, [&](uint64_t) { return (uint64_t)plan.k; });
    if (plan.by_p)
      select(true, [&](uint64_t all) {
        const double above = plan.above * to_units;
        const double share = set.p * (above + (double)all + (plan.by_k ? 0.0 : plan.below * to_units));
        const double want = ceil(share - above);
        return want >= 1.0 ? (uint64_t)want : (uint64_t)1;
      });
  }

  auto kept = [&](float x, uint64_t key) {
    return key >= cut && (!set.by_m || plan.top == INFINITY || exp(((double)x - (double)plan.top) / set.heat) >= set.m);
  };
  each(true, [&](uint64_t key, uint64_t fx) {
    if (kept(value_of<F32>(key, ib), key)) atomicAdd((unsigned long long*)&s_kept[index_of_key(key, ib) / kChunk], fx);
  });
  __syncthreads();
  // back in the units of the row's first bin: whole numbers too, of that bin's weights
  const double mass = tid < chunks ? sure + (double)s_kept[tid] * from_units : 0.0;
  double kept_all;
  const int token = draw<F32>(p, b, u, mass, chunks, s, [&](float x, int i) {
    int bin;
    uint64_t fx;
    if (!weigh(x, set.c4, plan.base, bin, fx) || bin > plan.hi) return 0.0;
    if (bin < plan.lo) return (double)fx * quarter(bin);
    return kept(x, key_of<F32>(x, i, ib)) ? rint(ldexp((double)fx, unit - 35) * quarter(bin - plan.lo)) * from_units : 0.0;
  }, kept_all);
  if (tid == 0) finish<F32>(p, b, token, set.c4, plan.base, plan.total);
}

template <bool F32>
void launch(const QhSampleRowsParams& p, const Ws& w, hipStream_t st) {
  const int chunks = n_chunks(p.V);
  const dim3 grid(chunks, p.B);
  sample_rows_scan_kernel<F32><<<grid, NT, 0, st>>>(p, w, chunks);
  sample_rows_plan_kernel<F32><<<p.B, NT, 0, st>>>(p, w, chunks);
  if (!p.top_k && !p.top_p && !p.min_p) return;
  int ib = 1;  // bits of an index
  while ((1 << ib) < p.V) ++ib;
  sample_rows_list_kernel<F32><<<grid, NT, 0, st>>>(p, w, chunks, min(kList, p.V), ib);
  sample_rows_cut_kernel<F32><<<p.B, NT, 0, st>>>(p, w, chunks, min(kList, p.V), ib);
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
