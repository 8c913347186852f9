// Launch descriptors of what a serving step needs around the paged cache: its page
// tables and slot maps (tables.hip), the adapters of its requests (adapters.hip), a token
// for each row of logits (sample_rows.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

struct QhTablesParams {
  int* pages;             // [n_rows][max_pages]
  int n_rows;
  int max_pages;
  int page_size;
  const int* length;      // [n_rows] positions held; may be length_out
  const int* new_tokens;  // [n_rows]
  const int* done;        // optional [n_rows]: rows that give their pages back first
  int* free_pages;        // [n_pages] ids of the free pages, the last of them taken first
  int n_pages;
  const int* n_free;      // how many there are; may be n_free_out
  int* length_out;
  int* n_free_out;
  int* at;                // [T]
  int* seq;               // [T]; null: token t is row t's
  int T;
  int* start;             // [n_rows + 1], with seq
  int* last;              // optional [n_rows]
};

constexpr int kTablesMaxRows = 2048;

struct QhAdaptersParams {
  const uint16_t* a;      // [n][R][K] bf16
  const uint16_t* b;      // [n][N][R] bf16
  const float* scale;     // [n]
  int n, R, K, N;
  const uint16_t* x;      // token t at x + t * x_ts
  long long x_ts;
  const int* ids;         // [T] adapter of each token; outside [0, n): none
  int T;
  const uint16_t* y;
  long long y_ts;
  uint16_t* out;          // may be y itself
  long long out_ts;
  float* h;               // workspace [slices][T][rank rounded up to 16]
};

constexpr int kAdaptersMaxRank = 128;
constexpr int kAdaptersMaxWidth = 1 << 30;         // a workgroup's columns end behind the last one, in 32 bits
constexpr int kAdaptersMaxTokens = (1 << 20) - 64;  // 16 to a workgroup along one axis of the grid

size_t qh_adapters_ws_bytes(int max_tokens, int R);
int qh_launch_adapters(const QhAdaptersParams& p, hipStream_t st);

struct QhSampleRowsParams {
  const void* logits;        // row b at logits + b * stride (elements), bf16 or fp32
  long long stride;
  int f32;
  int B, V;
  const float* u;            // [B] random numbers of [0, 1)
  const float* temperature;  // optional [B]; 0 or below: the largest
  const int* top_k;          // optional [B]; 0 or below: all
  const float* top_p;        // optional [B]; 1 or above: all
  const float* min_p;        // optional [B]; 0 or below: all
  int64_t* token;            // [B]
  float* logprob;            // optional [B]
  uint8_t* ws;
};

constexpr int kSampleRowsMaxVocab = 1 << 20;  // 128 workgroups a row
constexpr int kSampleRowsMaxRows = 65535;     // the grid's second axis

size_t qh_sample_rows_ws_bytes(int rows, int V);
int qh_launch_sample_rows(const QhSampleRowsParams& p, hipStream_t st);

int qh_launch_tables(const QhTablesParams& p, hipStream_t st);
void qh_set_error(const char* fmt, ...);
