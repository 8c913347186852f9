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
//      place is not written; the row itself is gone through instead, by the one workgroup: a row of
//      equal logits takes 1.3 ms (bf16; fp32 2.1) with top-p, 1.8 (2.8) with top-k too, and a
//      batch waits for it.
// The last two are launched only where a filter is given.  256 rows of 248320 bf16 logits take
// 58 + 8 + 26 + 53 us, one row 4.8 + 6.1 + 4.9 + 12.7.  The scan is bound by the VALU (28 instructions
// a logit and wave, 16 of them the weight and its bin; 83 % busy), plan and cut by a chain of round
// trips and, in rows whose range crosses zero (thousands of bf16 values), by the weights of one
// workgroup's list.
//
// Borders between tokens lie as close as the smallest weight, so weights are 64-bit: t = 4 x
// log2(e) / T in double, its nearest integer the bin, 2^(g / 4) of what is left (|g| <= 1/2) from a
// polynomial (1.1e-13) as an integer of 35 bits, which any order of atomics adds up to the same
// sum.  A weight is 2^-35.75 of itself off at most, alike wherever it is used.  Weights below 2^-63.75
// of the largest are none.  Weights of one bin are compared and added up as whole numbers; where
// those of several meet it is in doubles, whose sums come in a fixed order.
#include "qh_common.h"
#include "qh_scan.h"
#include "qh_serve.h"
#include "qh_weights.h"

namespace {

constexpr int NT = 512;
constexpr int kWaves = NT / 64;
constexpr int kChunk = 8192;           // logits of a workgroup, 16 a thread
constexpr int kRounds = kChunk / (8 * NT);
constexpr int kCopies = 8;             // of the histogram in LDS, by lane: logits crowd in few bins (1, 2, 4, 8: 118, 79, 60, 56 us)
constexpr int kList = 65536;           // places of a row's list
constexpr int kHeld = 20480;           // 32-bit words of LDS for it
constexpr int kMaxChunks = kSampleRowsMaxVocab / kChunk;
constexpr int kBinBit = 48;            // a value's weight below, its bin above
constexpr int kFine = 13;              // a chunk's 2^13 weights of 2^35 leave so many bits free
constexpr uint64_t kMassMask = (1ull << 50) - 1;  // a bin: weights below bit 50, the count above
static_assert(kMaxChunks <= kBins && NT == 2 * kBins, "a thread a chunk, two a bin");

struct Chunk {      // what a workgroup hands on
  double base;      // the bin of its largest logit; -infinity where there is none
  double mass;      // its weights in units of that bin
  float top;        // the largest
  int top_at;       // its first index, where the row wants it
};

struct RowPlan {    // what the plan says to the launches behind it
  int done;
  int lo, hi;       // the range: bins below the row's largest
  int by_k, by_p;   // which cuts fall in it
  int n_list;       // logits in it
  int k;            // of which top-k keeps so many
  int m_lo;         // the first of the three bins in which min-p's border falls (kNone: there is none)
  float top;        // the row's largest
  double total, before_hi;  // weights of all bins and of those before the range's last
};

struct Ws {
  uint64_t* hist;    // [B][chunks][kBins]
  Chunk* chunk;      // [B][chunks]
  double* sure;      // [B][chunks] weights before the range
  int2* span;        // [B][chunks] a chunk's logits on the list: where they begin, how many
  RowPlan* plan;     // [B]
  double2* bins;     // [B][kBins] the weight before a bin and its own, where top-p's cut may fall in several
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
  uint8_t* span = take(B * nc * 8);
  uint8_t* plan = take(B * sizeof(RowPlan));
  uint8_t* bins = take((size_t)B * kBins * sizeof(double2));
  uint8_t* list = take((size_t)B * min(kList, V) * 8);
  if (w) *w = Ws{(uint64_t*)hist, (Chunk*)chunk, (double*)sure, (int2*)span, (RowPlan*)plan, (double2*)bins, (uint64_t*)list, (unsigned*)taken};
  return off;
}

// ---- a row's settings ------------------------------------------------------------------------
struct Settings {
  double c4, c4_inv;  // t = x c4, x = t c4_inv
  double heat, p, m;
  int k;           // 0: all
  bool first;      // the first of the largest is the token
  bool by_p, by_m;
  __device__ __forceinline__ Settings(const QhSampleRowsParams& q, int b) {
    const float t = q.temperature ? q.temperature[b] : 1.0f;
    first = !(t > 0.0f);
    heat = first ? 1.0 : (double)t;
    c4 = 4.0 * 1.4426950408889634 / heat;
    c4_inv = heat * 0.17328679513998632;  // ln(2) / 4
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
// The logits of bins `hi` to `lo` below the largest lie between these two (a little wide): a test that
// most logits fail without their weight.  Where all have to be looked at, all pass.
struct Ends {
  float lo, hi;
  __device__ __forceinline__ Ends(const Settings& set, const Scale& s, int bin_lo, int bin_hi) {
    lo = (float)((s.base - bin_hi - 0.75) * set.c4_inv);
    hi = (float)((s.base - bin_lo + 0.75) * set.c4_inv);
    const float slack = 1e-6f * fmaxf(fabsf(lo), fabsf(hi));
    lo -= slack;
    hi += slack;
  }
  __device__ __forceinline__ bool out(float x) const { return x < lo || x > hi; }
};
// 2^(-j / 4)
__device__ __forceinline__ double quarter(int j) {
  const double s = (j & 2 ? 0.7071067811865476 : 1.0) * (j & 1 ? 0.8408964152537145 : 1.0);
  return ldexp(s, -(j >> 2));
}
// ... of every bin, and 0 for what has none
__device__ __forceinline__ void fill_quarters(double* s_quarter) {
  if ((int)threadIdx.x <= kBins) s_quarter[threadIdx.x] = (int)threadIdx.x < kBins ? quarter(threadIdx.x) : 0.0;
}
// Bins from a to b below it (they may be far apart, or infinite).
__device__ __forceinline__ double below(double a, double b) { return a == b ? 0.0 : a - b; }

// ---- logits ------------------------------------------------------------------------------------
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// Eight logits from index i on (-infinity behind the row's end).  A NaN among them fails every
// comparison on its way: it has no weight and is no maximum.
template <bool F32>
__device__ __forceinline__ void load8(const QhSampleRowsParams& p, int b, int i, float (&x)[8]) {
  if constexpr (F32) {
    const float* r = (const float*)p.logits + b * p.stride + i;
    if (i + 8 <= p.V) {
      const u32x4 v = *(const u32x4_any*)r, w = *(const u32x4_any*)(r + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = __uint_as_float(v[e]);
        x[4 + e] = __uint_as_float(w[e]);
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i + e < p.V ? r[e] : -INFINITY;
  } else {
    const uint16_t* r = (const uint16_t*)p.logits + b * p.stride + i;
    if (i + 8 <= p.V) {
      const u32x4 v = *(const u32x4_any*)r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = bf_lo(v[e]);
        x[2 * e + 1] = bf_hi(v[e]);
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i + e < p.V ? bf2f(r[e]) : -INFINITY;
  }
}
// The first index of round r of a chunk for this thread.
__device__ __forceinline__ int index_of(int chunk, int r) { return chunk * kChunk + (r * NT + (int)threadIdx.x) * 8; }

// Sort key of a logit and its index: larger for a larger value, of equal ones for a smaller index.
// The index takes `ib` bits.
template <bool F32>
__device__ __forceinline__ uint64_t key_of(float x, int i, int ib) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 is 0
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
// Exclusive prefix over the threads, and the total; a fixed order of additions.
template <typename T>
__device__ __forceinline__ T block_excl(T v, T* s_v, T& all) {
  const int wid = threadIdx.x >> 6;
  T w;
  T excl = wave_excl(v, w);
  if ((threadIdx.x & 63) == 0) s_v[wid] = w;
  __syncthreads();
  T at = 0, off = 0;
#pragma unroll
  for (int q = 0; q < kWaves; ++q) {
    if (q == wid) off = at;
    at += s_v[q];
  }
  __syncthreads();
  all = at;
  return off + excl;
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
  double w;
  wave_excl(v, w);
  if ((threadIdx.x & 63) == 0) s_d[threadIdx.x >> 6] = w;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int q = 0; q < kWaves; ++q) t += s_d[q];
  __syncthreads();
  return t;
}
// The least over the threads, the same in all.
__device__ __forceinline__ int block_min(int v, int* s_i) {
  v = wave_min(v);
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
// Token and log-probability, by the thread that has the logit; `total` is the weight of all logits.
__device__ __forceinline__ void emit(const QhSampleRowsParams& p, int b, int token, float x, const Scale& scale, double total) {
  p.token[b] = token;
  if (!p.logprob) return;
  int bin;
  uint64_t fx;
  p.logprob[b] = scale.weigh(x, bin, fx) ? (float)log((double)fx * quarter(bin) / total) : -INFINITY;
}

// Among the chunks, thread c's weighing `mass`, and then in the one that the draw falls into: the
// first index whose running sum of kept weights is above u times the whole.  keep(x, i, bin) says of a
// logit with a weight whether it is kept, of those below `least` none is; `total` below 0: all are.
// s_quarter[j] is 2^(-j / 4).
template <bool F32, typename Keep>
__device__ __forceinline__ void draw(const QhSampleRowsParams& p, int b, float u, double mass, int chunks, Sums& s,
                                     const double* s_quarter, const Scale& scale, double total, float least, Keep keep) {
  double all_mass;
  const double before = block_excl(mass, s.d[0], all_mass);
  if (total < 0.0) total = all_mass;
  const double target = (u > 0.0f ? min((double)u, 1.0) : 0.0) * all_mass;
  const bool some = (int)threadIdx.x < chunks && mass > 0.0;
  int c = block_min(some && before + mass > target ? (int)threadIdx.x : kNone, s.i);
  if (c == kNone) c = -block_min(some ? -(int)threadIdx.x : kNone, s.i);  // u = 1: the last
  c = min(max(c, 0), chunks - 1);
  if ((int)threadIdx.x == c) s.at[0] = before;
  float x[kRounds][8];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) load8<F32>(p, b, index_of(c, r), x[r]);
  double w[kRounds][8] = {}, sum[kRounds] = {};
  if (scale.quick) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      float most = x[r][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) most = fmaxf(most, x[r][e]);
      if (!__any(most >= least)) continue;  // a wave of logits that are all too small
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        int bin;
        const double v = (scale.weigh_quick(x[r][e], bin) - kWhole) * s_quarter[bin];
        w[r][e] = keep(x[r][e], index_of(c, r) + e, bin) ? v : 0.0;
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        int bin;
        uint64_t fx;
        w[r][e] = scale.weigh(x[r][e], bin, fx) && keep(x[r][e], index_of(c, r) + e, bin) ? (double)fx * s_quarter[bin] : 0.0;
      }
  }
  int last = kNone;
  float x_last = 0.0f;
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum[r] += w[r][e];
      if (w[r][e] > 0.0) {
        last = -(index_of(c, r) + e);
        x_last = x[r][e];
      }
    }
  static_assert(kRounds == 2, "two prefixes at once");
  double excl[2], all[2];
  block_excl(sum[0], sum[1], s.d[0], s.d[1], excl[0], all[0], excl[1], all[1]);
  int found = kNone;
  float x_found = 0.0f;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    double at = (s.at[0] + (r ? all[0] : 0.0)) + excl[r];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      at += w[r][e];
      if (found == kNone && w[r][e] > 0.0 && at > target) {
        found = index_of(c, r) + e;
        x_found = x[r][e];
      }
    }
  }
  int token = block_min(found, s.i);
  if (token != kNone) {
    if (found == token) emit(p, b, token, x_found, scale, total);
    return;
  }
  // the sums in another order fell short of the target: the last kept
  token = block_min(last, s.i);
  if (token != kNone && last == token) emit(p, b, -token, x_last, scale, total);
}

// ---- scan ------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(NT) void sample_rows_scan_kernel(QhSampleRowsParams p, Ws w, int chunks) {
  __shared__ Sums s;
  __shared__ uint64_t s_hist[(kBins + 1) * kCopies];
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
  int top_at = kNone;
  if (set.first) {
#pragma unroll
    for (int r = kRounds - 1; r >= 0; --r)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (x[r][e] == top) top_at = index_of(c, r) + e;
    top_at = block_min(top_at, s.i);
  }
  const Scale scale(set.c4, set.c4_inv, top);
  double mass = 0.0;
  if (!set.first || p.logprob) {
    unsigned long long* mine = (unsigned long long*)&s_hist[tid & (kCopies - 1)];
    if (scale.quick) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          int bin;
          const uint64_t fx = bits(scale.weigh_quick(x[r][e], bin));
          atomicAdd(mine + bin * kCopies, fx + ((1ull << 50) - 0x4330000000000000ull));  // the exponent away, a count in
        }
    } else {
#pragma unroll
      for (int r = 0; r < kRounds; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          int bin;
          uint64_t fx;
          if (scale.weigh(x[r][e], bin, fx)) atomicAdd(mine + bin * kCopies, fx | 1ull << 50);
        }
    }
    __syncthreads();
    if (tid < kBins) {  // four whole waves
      uint64_t v = 0;
#pragma unroll
      for (int q = 0; q < kCopies; ++q) v += s_hist[tid * kCopies + q];
      if (filtered) w.hist[(row + c) * kBins + tid] = v;
      wave_excl((double)(v & kMassMask) * quarter(tid), mass);
      if ((tid & 63) == 0) s.d[0][tid >> 6] = mass;
    }
    __syncthreads();
    mass = (s.d[0][0] + s.d[0][1]) + (s.d[0][2] + s.d[0][3]);
  }
  if (tid == 0) w.chunk[row + c] = Chunk{scale.base, mass, top, top_at};
}

// ---- plan ----------------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(NT) void sample_rows_plan_kernel(QhSampleRowsParams p, Ws w, int chunks) {
  __shared__ Sums s;
  __shared__ uint64_t s_other[2 * kBins];
  __shared__ double s_base[kMaxChunks], s_quarter[kBins + 1];
  const int tid = threadIdx.x, b = blockIdx.x;
  const size_t row = (size_t)b * chunks;
  const float u = p.u[b];
  const Settings set(p, b);
  const bool filtered = set.filtered();
  fill_quarters(s_quarter);
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
  const Scale scale(set.c4, set.c4_inv, row_top);
  // a chunk whose largest has no weight in the row has none: a draw of 0 would fall into it, and find nothing
  const double off = below(scale.base, mine.base);
  const double scaled = mine.mass > 0.0 && off < (double)kBins ? mine.mass * quarter((int)off) : 0.0;
  auto every = [](float, int, int) { return true; };
  if (!filtered) {
    if (set.first) {
      const int token = block_min(mine.top == row_top ? mine.top_at : kNone, s.i);
      const double all = block_total(scaled, s.d[0]);
      if (tid == 0) emit(p, b, token, row_top, scale, all);
    } else {
      draw<F32>(p, b, u, scaled, chunks, s, s_quarter, scale, -1.0, -INFINITY, every);
    }
    if (tid == 0) w.plan[b].done = 1;
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
        const double away = q < chunks ? below(scale.base, s_base[q]) : INFINITY;  // infinite for a chunk without logits
        const bool in = away <= (double)j;
        v[e] = w.hist[in ? (row + q) * kBins + (j - (int)away) : row * kBins];
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
  double excl, total;
  uint64_t n_excl, n_all;
  block_excl(weight, (uint64_t)count, s.d[0], s.u, excl, total, n_excl, n_all);
  RowPlan plan = {};
  plan.m_lo = kNone;
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
  if (set.by_m && !scale.far) {
    // the bin of the least weight that is kept, and one on both sides
    const double least = scale.base - rint((double)row_top * set.c4 + 4.0 * log2(set.m));
    const int jm = least < (double)kBins ? (int)least : kBins;
    const int m_lo = max(jm - 1, 0), m_hi = jm + 1;
    plan.m_lo = m_lo;
    if (m_hi < lo) {  // above the other cuts
      lo = m_lo;
      hi = m_hi;
      plan.by_k = plan.by_p = 0;
    } else {
      lo = min(lo, m_lo);
    }
  }
  if (lo >= kBins) {  // nothing is cut
    draw<F32>(p, b, u, scaled, chunks, s, s_quarter, scale, -1.0, -INFINITY, every);
    if (tid == 0) w.plan[b].done = 1;
    return;
  }
  hi = min(hi, kBins - 1);
  if (plan.by_k && plan.by_p && lo < hi && tid < kBins) w.bins[(size_t)b * kBins + tid] = double2{excl, weight};
  if (tid == lo) s.n[0] = n_excl;
  if (tid == hi) {
    s.d[0][1] = excl;
    s.n[1] = n_excl + count;
  }
  __syncthreads();
  if (tid == 0) {
    plan.done = 0;
    plan.lo = lo;
    plan.hi = hi;
    plan.before_hi = s.d[0][1];
    plan.n_list = (int)(s.n[1] - s.n[0]);
    plan.k = set.k - (int)s.n[0];
    plan.top = row_top;
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
  const Settings set(p, b);
  const Scale scale(set.c4, set.c4_inv, plan.top);
  const double off = below(scale.base, w.chunk[row + c].base);
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
  if (tid == 0) {
    w.sure[row + c] = sure_all;
    if (n_all == 0) w.span[row + c] = int2{0, 0};
  }
  if (n_all == 0 || plan.n_list > places) return;
  float x[kRounds][8];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) load8<F32>(p, b, index_of(c, r), x[r]);
  if (tid == 0) {
    s_n = atomicAdd(&w.taken[b], (unsigned)n_all);
    w.span[row + c] = int2{(int)s_n, (int)n_all};
  }
  __syncthreads();
  const Ends ends(set, scale, plan.lo, plan.hi);
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (ends.out(x[r][e])) continue;
      int bin;
      uint64_t fx;
      if (scale.weigh(x[r][e], bin, fx) && bin >= plan.lo && bin <= plan.hi) {
        const unsigned at = atomicAdd(&s_n, 1u);
        if (at < (unsigned)places) list[at] = key_of<F32>(x[r][e], index_of(c, r) + e, ib);
      }
    }
}

// ---- cut -----------------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(NT) void sample_rows_cut_kernel(QhSampleRowsParams p, Ws w, int chunks, int places, int ib) {
  __shared__ Sums s;
  __shared__ uint64_t s_held[kHeld / 2];
  __shared__ uint64_t s_mass[NT], s_weight[NT], s_kept[kMaxChunks];
  __shared__ unsigned s_count[NT];
  __shared__ double s_quarter[kBins + 1], s_more[kMaxChunks];
  __shared__ int2 s_span[kMaxChunks];
  const int tid = threadIdx.x, b = blockIdx.x;
  const RowPlan plan = w.plan[b];
  if (plan.done) return;
  const Settings set(p, b);
  const Scale scale(set.c4, set.c4_inv, plan.top);
  const Ends ends(set, scale, plan.lo, plan.hi);
  const size_t row = (size_t)b * chunks;
  const uint64_t* list = w.list + (size_t)b * places;
  const int n_list = plan.n_list;
  const bool listed = n_list <= places;
  const float u = p.u[b];
  const double sure = tid < chunks ? w.sure[row + tid] : 0.0;
  if (tid < chunks) {
    s_kept[tid] = 0;
    s_span[tid] = w.span[row + tid];
  }
  fill_quarters(s_quarter);

  auto in_range = [&](float x, int& bin, uint64_t& fx) {
    return !ends.out(x) && scale.weigh(x, bin, fx) && bin >= plan.lo && bin <= plan.hi;
  };

  // fn(key) for every logit of the range, from memory
  uint64_t first[8] = {};
  if (listed) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (tid + e * NT < n_list) first[e] = list[tid + e * NT];
  }
  auto each_far = [&](auto fn) {
    if (listed) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (tid + e * NT < n_list) fn(first[e], tid + e * NT);
      for (int i0 = tid + 8 * NT; i0 < n_list; i0 += 8 * NT) {
        uint64_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = list[min(i0 + e * NT, n_list - 1)];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i0 + e * NT < n_list) fn(v[e], i0 + e * NT);
      }
    } else {
      for (int q = 0; q < chunks; ++q) {
        float x[kRounds][8];
#pragma unroll
        for (int r = 0; r < kRounds; ++r) load8<F32>(p, b, index_of(q, r), x[r]);
#pragma unroll
        for (int r = 0; r < kRounds; ++r)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            int bin;
            uint64_t fx;
            if (in_range(x[r][e], bin, fx)) fn(key_of<F32>(x[r][e], index_of(q, r) + e, ib), 0);
          }
      }
    }
  };

  // What all keys have in common tells nothing: digits are of the distance from the least that the
  // range may have.
  const bool whole = !(ends.lo <= ends.hi);  // ends that are no numbers: the largest alone has a weight
  const uint64_t least_value = key_of<F32>(whole ? plan.top : ends.lo, 0, ib) >> ib;
  const uint64_t values = (key_of<F32>(whole ? plan.top : ends.hi, 0, ib) >> ib) - least_value + 1;
  const uint64_t least = least_value << ib;
  const int key_bits = 64 - __clzll((long long)((values << ib) - 1));
  // Few values (of bf16 logits nearly always): a digit is a value, all its logits weigh the same, and
  // weights come from a table (256 rows: 55 us, without 64), a value a thread.
  const bool few = values <= NT;
  int value_bin = kNone;  // of the digit `tid`
  if (few) {
    uint64_t fx;
    const bool in = in_range(value_of<F32>((least_value + tid) << ib, ib), value_bin, fx);
    if (!in) value_bin = kNone;
    s_weight[tid] = in ? fx | (uint64_t)value_bin << kBinBit : 0;
  }
  // the list stays in LDS where it fits: as distances of 32 bits (few values: 29 at most), or whole
  uint32_t* held32 = (uint32_t*)s_held;
  const bool in32 = listed && key_bits <= 32 && n_list <= kHeld, in64 = listed && !in32 && n_list <= kHeld / 2;
  if (in32) each_far([&](uint64_t key, int i) { held32[i] = (uint32_t)(key - least); });
  else if (in64) each_far([&](uint64_t key, int i) { s_held[i] = key; });
  __syncthreads();
  auto each = [&](auto fn) {
    if (in32) {
      for (int i0 = tid; i0 < n_list; i0 += 4 * NT) {  // four reads on their way at once
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = held32[min(i0 + e * NT, n_list - 1)];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i0 + e * NT < n_list) fn(least + v[e]);
      }
    } else if (in64) {
      for (int i = tid; i < n_list; i += NT) fn(s_held[i]);
    } else {
      each_far([&](uint64_t key, int) { fn(key); });
    }
  };
  // a listed logit's bin and its weight in the bin's units
  auto weight_of = [&](uint64_t key, int& bin) -> uint64_t {
    uint64_t fx = 0;
    if (few) {
      const uint64_t v = s_weight[(key >> ib) - least_value];
      bin = (int)(v >> kBinBit);
      return v & ((1ull << kBinBit) - 1);
    }
    return in_range(value_of<F32>(key, ib), bin, fx) ? fx : 0;
  };
  // Top-p's share within bin `p_bin`, in the bin's units; 0 where it turns out to be an earlier one's.  First of
  // the range's last bin, of which top-k leaves `all` (without top-k the cut is there): what is kept before it is
  // known, and with it the share.  Sums in different bins' units meet in doubles alone, as the draw's do.
  int p_bin = plan.hi;
  double p_before = plan.before_hi, share = -1.0;
  auto p_want = [&](uint64_t all) -> uint64_t {
    if (share < 0.0) {
      share = set.p * (plan.by_k ? p_before + (double)all * s_quarter[p_bin] : plan.total);
      if (plan.by_k && plan.lo < plan.hi) {
        double2 v = {0.0, 0.0};
        if (tid < plan.hi) v = w.bins[(size_t)b * kBins + tid];
        const int at = block_min(v.y > 0.0 && v.x + v.y >= share ? tid : kNone, s.i);
        if (at != kNone) {
          if (tid == at) s.at[0] = v.x;
          __syncthreads();
          p_bin = at;
          p_before = s.at[0];
          return 0;
        }
      }
    }
    const double want = min(ceil((share - p_before) / s_quarter[p_bin]), (double)all);
    return want >= 1.0 ? (uint64_t)want : 1;
  };

  uint64_t cut = 0;  // the least key that is kept, of bin cut_bin; bins before that are kept whole
  int cut_bin = plan.hi;
  // The least key such that those from it up, of the ones from `cut` up that are below `from` + 2^high (by
  // weight: and in bin p_bin), are as many (or weigh as much) as wanted(their sum): digit after digit of nine bits
  // of the distance from `from`, until one key is left.  False where nothing is wanted.
  auto select = [&](bool by_weight, uint64_t from, int high, auto wanted) {
    uint64_t want = 0, prefix = 0;
    for (int round = 0;; ++round) {
      const int shift = max(high - 9, 0);
      s_count[tid] = 0;
      s_mass[tid] = 0;
      __syncthreads();
      each([&](uint64_t key) {
        const uint64_t d = key - from;
        if (key < cut || d >> high != prefix) return;
        const int digit = (int)(d >> shift) & ((1 << (high - shift)) - 1);
        if (by_weight) {
          int bin = kNone;
          const uint64_t fx = weight_of(key, bin);
          if (bin != p_bin) return;
          atomicAdd((unsigned long long*)&s_mass[digit], fx);
        }
        atomicAdd(&s_count[digit], 1u);
      });
      __syncthreads();
      const int digit = NT - 1 - tid;
      const uint64_t n = s_count[digit], mine = by_weight ? s_mass[digit] : n;
      uint64_t all;
      const uint64_t before = block_excl(mine, s.u, all);
      if (round == 0) want = wanted(all);
      if (want == 0) return false;
      const int at = block_min(n > 0 && before + mine >= want ? tid : kNone, s.i);
      if (at == kNone) return true;  // all of them
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
    const uint64_t found = from + (prefix << high);
    cut = found > cut ? found : cut;
    return true;
  };
  if (few && (plan.by_k || plan.by_p)) {
    // how many logits each value has: both cuts as a value and how many of its logits are kept
    s_count[tid] = 0;
    __syncthreads();
    each([&](uint64_t key) { atomicAdd(&s_count[(key >> ib) - least_value], 1u); });
    __syncthreads();
    const int value = NT - 1 - tid;
    const uint64_t fx = s_weight[value] & ((1ull << kBinBit) - 1);
    const int bin = (int)(s_weight[value] >> kBinBit);
    uint64_t n = s_count[value], n_before, n_all, before, all;  // n: how many top-k leaves
    block_excl(n, bin == p_bin ? n * fx : 0, s.u, (uint64_t*)s.d[0], n_before, n_all, before, all);
    int cut_at = kNone, cut_n = 0;  // the value, by its thread
    if (plan.by_k) {
      cut_at = block_min(n > 0 && n_before + n >= (uint64_t)plan.k ? tid : kNone, s.i);
      if (tid == cut_at) {
        n = plan.k - n_before;
        s.n[0] = n;
        s.n[1] = before + n * fx;
      } else if (tid > cut_at) {
        n = 0;
      }
      __syncthreads();
      if (cut_at != kNone) {
        cut_n = (int)s.n[0];
        all = s.n[1];
      }
      __syncthreads();
    }
    if (plan.by_p) {
      uint64_t want = p_want(all);
      if (want == 0) {
        before = block_excl(bin == p_bin ? n * fx : 0, s.u, all);
        want = p_want(all);
        cut_bin = p_bin;
      }
      const int at = block_min(n > 0 && bin == p_bin && before + n * fx >= want ? tid : kNone, s.i);
      if (tid == at) s.n[0] = (want - before + fx - 1) / fx;
      __syncthreads();
      if (at != kNone && (at < cut_at || (at == cut_at && (int)s.n[0] < cut_n))) {
        cut_at = at;
        cut_n = (int)s.n[0];
      }
      __syncthreads();
    }
    if (cut_at != kNone) {
      const uint64_t at = least_value + (uint64_t)(NT - 1 - cut_at);
      cut = at << ib;
      if (cut_n < (int)s_count[NT - 1 - cut_at]) {  // of equal ones the first: by the index's digits
        __syncthreads();
        select(false, cut, ib, [&](uint64_t) { return (uint64_t)cut_n; });
      }
    }
  } else {
    if (plan.by_k) select(false, least, key_bits, [&](uint64_t) { return (uint64_t)plan.k; });
    if (plan.by_p && !select(true, least, key_bits, p_want)) {
      select(true, least, key_bits, p_want);
      cut_bin = p_bin;
    }
  }

  // Bins before part_lo are kept whole, those behind part_hi not at all; of the up to three between, a key
  // from the cut up (as a comparison of logits) that min-p leaves.
  const int part_lo = min(cut_bin, plan.m_lo), part_hi = plan.m_lo == kNone ? cut_bin : min(cut_bin, plan.m_lo + 2);
  const float x_cut = cut > 0 ? value_of<F32>(cut, ib) : -INFINITY;
  const int i_cut = index_of_key(cut, ib);
  auto kept = [&](float x, int i, int bin) {
    return (bin < cut_bin || x > x_cut || (x == x_cut && i <= i_cut)) &&
           (bin < plan.m_lo || exp(((double)x - (double)plan.top) / set.heat) >= set.m);
  };
  // What is kept of each chunk.  Of whole bins by the chunk's histogram, four threads a chunk,
  if (part_lo > plan.lo) {
    static_assert(NT >= 4 * kMaxChunks, "four threads a chunk");
    const int c = tid >> 2;
    // (infinite for a chunk without logits)
    const double off = c < chunks ? below(scale.base, w.chunk[row + c].base) : INFINITY;
    double more = 0.0;
    if (off < (double)part_lo)
#pragma unroll 4
      for (int j = max(plan.lo, (int)off) + (tid & 3); j < part_lo; j += 4)
        more += (double)(w.hist[(row + c) * kBins + (j - (int)off)] & kMassMask) * s_quarter[j];
    more += __shfl_xor(more, 1, 64);
    more += __shfl_xor(more, 2, 64);
    if (c < chunks && (tid & 3) == 0) s_more[c] = more;
  }
  // of the others by its logits, which lie together on the list, a wave a chunk: in units of 2^-kFine of bin
  // part_lo's, 62 bits for all of a chunk; a weight of the next two bins loses 2^-48 of it.
  auto weight_kept = [&](uint64_t key) -> uint64_t {
    int bin = kNone;
    const uint64_t fx = weight_of(key, bin);
    if (bin < part_lo || bin > part_hi || !kept(value_of<F32>(key, ib), index_of_key(key, ib), bin)) return 0;
    return bin == part_lo ? fx << kFine : (uint64_t)rint((double)(fx << kFine) * s_quarter[bin - part_lo]);
  };
  if (listed) {
    const bool by_value = in32 && few && plan.m_lo == kNone;
    if (by_value) {
      __syncthreads();
      if (value_bin != cut_bin) s_weight[tid] = 0;
      else s_weight[tid] &= (1ull << kBinBit) - 1;
      __syncthreads();
    }
    for (int c = tid >> 6; c < chunks; c += kWaves) {
      const int2 span = s_span[c];
      uint64_t mine = 0, all;
      const int end = span.x + span.y;
      if (by_value) {
        const uint32_t cut32 = cut > least ? (uint32_t)(cut - least) : 0;  // the cut is not above the largest key
        for (int i0 = span.x + (tid & 63); i0 < end; i0 += 256) {
          uint32_t v[4];
          uint64_t fx[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = held32[min(i0 + 64 * e, end - 1)];
#pragma unroll
          for (int e = 0; e < 4; ++e) fx[e] = s_weight[v[e] >> ib];
#pragma unroll
          for (int e = 0; e < 4; ++e) mine += i0 + 64 * e < end && v[e] >= cut32 ? fx[e] : 0;
        }
        mine <<= kFine;
      } else {
        for (int i = span.x + (tid & 63); i < end; i += 64)
          mine += weight_kept(in32 ? least + held32[i] : in64 ? s_held[i] : list[i]);
      }
      wave_excl(mine, all);
      if ((tid & 63) == 0) s_kept[c] = all;
    }
  } else {
    each([&](uint64_t key) {
      const uint64_t fx = weight_kept(key);
      if (fx) atomicAdd((unsigned long long*)&s_kept[index_of_key(key, ib) / kChunk], fx);
    });
  }
  __syncthreads();
  // in the units of the row's first bin: whole numbers where all is in that bin
  double mass = 0.0;
  if (tid < chunks) {
    mass = sure + (double)s_kept[tid] * (s_quarter[part_lo] * (1.0 / (1 << kFine)));
    if (part_lo > plan.lo) mass += s_more[tid];
  }
  draw<F32>(p, b, u, mass, chunks, s, s_quarter, scale, plan.total, ends.lo,
            [&](float x, int i, int bin) { return bin < part_lo || (bin <= part_hi && kept(x, i, bin)); });
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
