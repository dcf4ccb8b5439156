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

constexpr int kMergeBytes = 32;

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
};

}  // namespace fa2
