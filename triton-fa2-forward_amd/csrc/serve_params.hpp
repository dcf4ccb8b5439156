// serve_params.hpp - argument blocks of the serving kernels (rotary positions, the paged K/V cache,
// attention over packed sequences and over pages), shared by host and device code.
#pragma once

#include <stdint.h>

namespace fa2 {

// Rotation of the first 2 * half values of a row: pairs (i, i + half), or (2 i, 2 i + 1) when interleaved,
// by the angle freqs[i] * position (float64 radians), times scale. half 0: none.
struct RotaryPlan {
  const double* freqs;
  int32_t half;
  int32_t interleaved;
  double scale;
};

struct RotaryParams {
  const uint16_t* x;
  uint16_t* out;
  int64_t sxb, sxh, sxn;
  int64_t sob, soh, son;
  const void* positions;  // int32 or int64, element strides spb, spn
  int64_t spb, spn;
  int32_t positions64;
  int32_t batch, heads, n;
  int32_t tokens_per_wg;
  RotaryPlan rot;
};

// Sequences over a paged cache: sequence s owns packed rows cu[s] .. cu[s + 1] - 1, its last tokens of
// lens[s] in the cache; token p of it lies in page table[s * table_stride + p / page_size], row p % page_size.
// Everything read from the device is checked there: rows outside every sequence are skipped, a page
// outside [0, n_pages) is never accessed.
struct Sequences {
  const int32_t* cu;    // [n_seq + 1]
  const int32_t* lens;  // [n_seq]
  const int32_t* table;
  int64_t table_stride;
  int32_t n_seq, n_tokens;
  int32_t max_pages, n_pages, page_shift;
};

// One of the cache's two tensors: 16-bit elements, or e4m3 bytes with a scale byte e per row (value
// times 2^(e - 127)). Element strides (bytes for e4m3 and the scales).
struct CacheTensor {
  char* data;
  uint8_t* scale;
  int64_t page, head, token;
  int64_t scale_page, scale_head, scale_token;
};

struct CacheParams {
  CacheTensor kc, vc;
  Sequences seq;
  // cache_write: sources; cache_read: destinations. Strides [token, head].
  uint16_t *k, *v;
  int64_t skt, skh, svt, svh;
  const uint16_t* q;  // cache_write: rotated into q_out beside it, or null
  uint16_t* q_out;
  int64_t sqt, sqh, sot, soh;
  int32_t h_kv, h_q;
  int32_t tokens_per_wg;
  RotaryPlan rot;
};

// What rows of q and k are turned by, beyond a rotation by one position: each head first divided by its root mean
// square, x / sqrt(mean x^2 + eps) * weight (float32 [head_dim]; null: not), and pair i rotated by the position on
// axis axes[i] of n_axes (null: all by the first; an entry outside them by the nearest).
struct TurnParams {
  const int32_t* axes;
  int32_t n_axes;
  int32_t positions64;
  const void* positions;  // int32 or int64, element strides [axis, batch, token]; null: the place in the sequence
  int64_t spa, spb, spn;
  const float *q_weight, *k_weight;
  double q_eps, k_eps;
};

struct RotaryQkParams {
  const uint16_t *q, *k;
  uint16_t *q_out, *k_out;
  int64_t sqb, sqh, sqn, skb, skh, skn;
  int64_t sqob, sqoh, sqon, skob, skoh, skon;
  int32_t batch, h_q, h_k, n;
  int32_t tokens_per_wg;
  RotaryPlan rot;
  TurnParams turn;
};

struct CacheTurnParams : CacheParams {
  TurnParams turn;
};

// A step's pages (serve_pages.hip): free_pages[0 .. count) are free; results in memory of their own, but the table's.
struct PagesParams {
  const int32_t* free_pages;
  const int32_t* count;
  int32_t* table;
  const int32_t *lens, *fresh;  // [n_seq]: tokens in the cache, and new ones
  int64_t table_stride;
  int32_t n_pages, n_seq, max_pages, page_shift, n_tokens;
  int32_t *count_out, *lens_out, *cu_out, *positions;
  int64_t* slots;
};

struct ReleaseParams {
  int32_t* free_pages;
  const int32_t *count, *table, *first, *last;
  int64_t table_stride;
  int32_t n_pages, n_seq, max_pages;
  int32_t* count_out;
  int32_t* counts;  // [n_seq + 1]
};

constexpr int kMergeBytes = 32;

// What keys the rows of a ragged attention launch take: all up to their last; those of a window and the first
// few; of sequences with a common prefix, the prefix's (all rows as those of one sequence), or their own behind it.
constexpr int kModeAll = 0, kModeWindow = 1, kModePrefix = 2, kModeOwn = 3;

// Attention of packed rows. K and V are packed rows too (source 0), pages of 16-bit elements (1) or of
// e4m3 (2).
struct RaggedParams {
  const uint16_t* q;
  uint16_t* o;
  float* lse;  // [h_q][n_tokens], or null
  int64_t sqt, sqh, sot, soh;
  CacheTensor kc, vc;     // packed rows: data, head and token strides
  Sequences seq;          // packed rows: cu, n_seq, n_tokens
  const int32_t* cu_kv;   // packed rows: [n_seq + 1]
  int32_t kv_tokens;
  int32_t h_kv, group, causal;
  float qk_scale;
  int32_t xcd_shift;
  // 0: a workgroup per row tile. Above: that many workgroups per KV head share its work evenly by
  // cutting the row tiles' key ranges; the pieces of a cut row tile meet in `parts`.
  int32_t shares;
  double per_share;  // 1 / shares
  float* parts;  // [h_kv * shares][2][block_m][head_dim + 4]: O, then m, l, exact l
  void* merges;  // [h_kv * shares] of kMergeBytes: the tile that ends in each share
  // kModeWindow: a row sees the `window` newest keys up to its last, and the first `sinks`
  int32_t window, sinks;
  // kModePrefix and kModeOwn: the leading tokens that all sequences have in common, on the device; every row's results over
  // them and over its own keys, [2][n_tokens * h_q][head_dim + 4]; the rows of a partial result
  const int32_t* shared;
  float* rows;
  int32_t part_rows;
};

}  // namespace fa2
