// Launch descriptors of what a serving step needs around the paged cache: its page
// tables and slot maps (tables.hip).
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

int qh_launch_tables(const QhTablesParams& p, hipStream_t st);
void qh_set_error(const char* fmt, ...);
