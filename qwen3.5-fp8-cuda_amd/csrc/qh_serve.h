// Launch descriptors of what a serving step needs around the paged cache: its page
// tables and slot maps (tables.hip), the adapters of its requests (adapters.hip).
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
constexpr int kAdaptersMaxTokens = (1 << 20) - 64;  // 16 to a workgroup along one axis of the grid

size_t qh_adapters_ws_bytes(int max_tokens, int R);
int qh_launch_adapters(const QhAdaptersParams& p, hipStream_t st);

int qh_launch_tables(const QhTablesParams& p, hipStream_t st);
void qh_set_error(const char* fmt, ...);
