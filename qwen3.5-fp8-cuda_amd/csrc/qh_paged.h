// Launch descriptors of the paged KV-cache kernels (paged_kv.hip: write and read
// back, paged_attn.hip: decode attention).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/qh_paged_types.h"
#include "qh_paged_div.h"

// A cache and the page tables of a batch, as the kernels see them.
struct QhPagedView {
  void* k;
  void* v;
  float* ks;              // null: bf16 rows
  float* vs;
  int n_pages;
  int page_size;
  int n_kv;
  uint32_t div_mul;       // of a position by page_size (qh_quotient)
  int div_shift;
  const int* pages;       // [n_seqs][max_pages]
  int n_seqs;
  int max_pages;
  int capacity;           // max_pages * page_size: positions that a table can name
};

struct QhPagedPrepParams {
  QhPagedView c;
  const uint16_t* q;      // token t, head h at q + t * q_ts + h * q_hs (elements); null: no q
  long long q_ts, q_hs;
  const uint16_t* k;      // token t, head h at k + t * k_ts + h * D
  long long k_ts;
  const uint16_t* v;
  long long v_ts;
  const float* q_norm_w;  // optional (1+w) head norm weights [D]
  const float* k_norm_w;
  float eps;
  qh_rope_axes rope;      // rot == 0: no rotation
  const int* pos;         // [n_axes][T]
  const int* seq;         // [T]; null: token t belongs to sequence t
  const int* at;          // [T] cache positions
  int T;
  void* q_out;            // [T][n_heads][D] bf16 or fp32
  int q_f32;
  int n_heads;
};

struct QhPagedReadParams {
  QhPagedView c;
  const int* last;        // [n_seqs] newest position
  uint16_t* k_out;        // [n_seqs][n_kv][max_seq][D] bf16
  uint16_t* v_out;
  int max_seq;
};

struct QhPagedAttnParams {
  QhPagedView c;
  const uint16_t* q;      // sequence b, head h at q + b * q_bs + h * q_hs
  long long q_bs, q_hs;
  const uint16_t* gate;   // optional output gate
  long long g_bs, g_hs;
  const int* last;        // [n_seqs]
  int n_heads;
  uint16_t* out;          // [n_seqs][n_heads][D] bf16
  unsigned* counters;     // [kPagedMaxUnits] zero between calls
  float* part;
  // what the launch derives for the kernel, which would spend its time on divisions
  int group;              // heads of a KV head
  uint32_t group_mul;     // of i < 1024 by group (qh_group_quotient)
  int group_shift;        // log2 of the threads that take a pair's items together
  int slots;              // workgroups of each KV head
};

// (sequence, kv head) pairs that one call of the decode attention takes, and its sequences.
constexpr int kPagedMaxUnits = 65536;
constexpr int kPagedMaxSeqs = 2048;

int qh_paged_view(const qh_paged_cache* c, const int* pages, int n_seqs, int max_pages, const char* what,
                  QhPagedView* out);
int qh_launch_paged_prep(const QhPagedPrepParams& p, int D, hipStream_t st);
int qh_launch_paged_read(const QhPagedReadParams& p, int D, hipStream_t st);
size_t qh_paged_attn_ws_bytes(int n_heads, int n_kv, int D);
int qh_launch_paged_attn(QhPagedAttnParams p, int D, hipStream_t st);
void qh_set_error(const char* fmt, ...);

#if defined(__HIPCC__)
// The page of a position, counted in the sequence's table.
__device__ __forceinline__ int page_of(const QhPagedView& c, int pos) {
  return qh_quotient(pos, c.div_mul, c.div_shift);
}
#endif
