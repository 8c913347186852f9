/* Descriptors of the paged KV-cache entry points (host structures, read during
 * the call; the pointers in them are device pointers). */
#ifndef QH_PAGED_TYPES_H
#define QH_PAGED_TYPES_H

/* One layer's cache as a pool of pages.  Row (page, kv head, slot) of k and v
 * holds head_dim values: bf16, or with fp8 != 0 E4M3FN bytes that stand for
 * byte * scale, one fp32 scale per row.  page_size is a multiple of 8;
 * head_dim 128 or 256; 16-byte aligned pointers. */
typedef struct qh_paged_cache {
  void* k;        /* [n_pages][n_kv][page_size][head_dim] */
  void* v;
  float* k_scale; /* [n_pages][n_kv][page_size], null for bf16 */
  float* v_scale;
  int n_pages;
  int page_size;
  int n_kv;
  int head_dim;
  int fp8;
} qh_paged_cache;

/* Rotary positions on several axes (1 to 4).  Dimension pair (i, i + rot/2),
 * i < rot/2, is turned by the angle of column i and row pos[axis(i)] of the
 * tables.  axis(i): interleaved == 0: the first section[0] pairs take axis 0,
 * the next section[1] axis 1, ...; interleaved != 0: i % n_axes while
 * i < n_axes * section[i % n_axes], otherwise 0.  The sections add up to rot/2.
 * rot is a multiple of 16, at most head_dim. */
typedef struct qh_rope_axes {
  const float* cos_t; /* [max_pos][rot] fp32, of which columns [0, rot/2) are read */
  const float* sin_t;
  int max_pos;
  int rot;
  int n_axes;
  int interleaved;
  int section[4];
} qh_rope_axes;

#endif /* QH_PAGED_TYPES_H */
