// serve_launch.hpp - launchers of the serving kernels. Each returns a hipError_t value.
#pragma once

#include <hip/hip_runtime.h>

#include "serve_params.hpp"

namespace fa2 {

// Tokens of one workgroup of the rotary and cache kernels: as many as its 256 lanes take rows of at once, and more
// while at least `least_wgs` workgroups are left.
int serve_tokens_per_wg(int lanes_per_token, int64_t tokens, int64_t least_wgs);

int launch_rotary(int dtype, int head_dim, const RotaryParams& p, unsigned grid, hipStream_t stream);
int launch_cache(bool write, int dtype, int head_dim, bool e4m3, const CacheParams& p, unsigned grid,
                 hipStream_t stream);

int launch_rotary_qk(int dtype, int head_dim, const RotaryQkParams& p, unsigned grid, hipStream_t stream);
int launch_cache_write_turn(int dtype, int head_dim, bool e4m3, const CacheTurnParams& p, unsigned grid, hipStream_t stream);

int launch_pages_extend(const PagesParams& p, unsigned blocks, unsigned stripes, hipStream_t stream);
int launch_pages_release(const ReleaseParams& p, hipStream_t stream);

// Where K and V of a ragged attention launch lie: packed rows, 16-bit pages, e4m3 pages.
constexpr int kSourcePacked = 0, kSourcePages = 1, kSourceE4m3 = 2;

// Its workgroups per CU (waves per SIMD), by registers: packed rows keep nothing from tile to tile (128 VGPRs at
// head_dim 64). Measured at head_dim 64 on MI355X: packed prompts of 3k to 8k, 2 / 3 / 4 a CU 394 / 390 / 384 us; a chunk of
// 2000 over 8k keys, 16-bit pages 170 / 165 / 223 (spilled), e4m3 pages 193 / 195 / 359. 32-row workgroups keep 32 KiB of LDS up
// to head_dim 32 and 64 above: steps of 195 e4m3 sequences of up to 8000, 8 heads of 32, 123 / 104 / 121 us; of 97
// 16-bit ones 84 / 90 / 93, of 195 with heads of 16 95 / 88 / 91.
constexpr int ragged_waves(int head_dim, int source, int row_waves) {
  if (row_waves == 1) return head_dim <= 32 ? 3 : 2;
  return head_dim == 128 || source == kSourceE4m3 ? 2 : source == kSourcePages ? 3 : 4;
}

// Keys that a tile costs beside its own: its rows' loads, its merge and stores. Measured on MI355X, in keys of cost
// 64 / 128 / 256 / 384: 4 prompts of 2000 in 128-row tiles (a share of short tiles alone holds many of them)
// 201 / 185 / 164 / 166 us; steps of 64 sequences of 1000 keys in 32-row tiles 46.5 / 47.8 / 48.0 / 49.0.
template <int BM>
constexpr int kTileCost = BM == 32 ? 64 : 256;
// ... and what sharing the tiles out costs a 128-row workgroup: more pieces, the partial results, their merge
constexpr int kShareCost = 640;

// The ragged attention kernel with 32 * row_waves (1 or 4) rows per workgroup, and after it, with p.shares > 0,
// the merge of the row tiles that its shares cut.
template <int DT, int D, int MODE>
int launch_ragged(const RaggedParams& p, int source, int row_waves, unsigned grid, hipStream_t stream);

// Workgroups per CU of the kernels that hold two forms' code (three would spill up to 64 registers at head_dim 64), and workgroups that join its rows' results (8 rows each)
constexpr int kSharedWaves = 2;
inline int64_t shared_join_grid(const RaggedParams& p) {
  return ((int64_t)p.seq.n_tokens * p.group + 7) / 8 * p.h_kv;
}

// Attention within a window over pages, chunks beside single tokens: p.shares workgroups per head for sequences of more than 32 rows, and
// one for each sequence (grid: both), then the merge of the tiles that the shares cut.
template <int DT, int D>
int launch_window_mixed(const RaggedParams& p, int source, unsigned grid, hipStream_t stream);

// The kernel for batches with a common prefix with 32 * prefix_waves rows per workgroup for the prefix and 32 * own_waves for the keys behind it (1 and 1, 4 and 1, or 4
// and 4), and after it the join of its rows' results.
template <int DT, int D>
int launch_shared(const RaggedParams& p, int source, int prefix_waves, int own_waves, unsigned grid, hipStream_t stream);

#define FA2_DECLARE_RAGGED(DT, D)                                                              \
  template <>                                                                                  \
  int launch_ragged<DT, D, kModeAll>(const RaggedParams&, int, int, unsigned, hipStream_t);    \
  template <>                                                                                  \
  int launch_ragged<DT, D, kModeWindow>(const RaggedParams&, int, int, unsigned, hipStream_t); \
  template <>                                                                                  \
  int launch_window_mixed<DT, D>(const RaggedParams&, int, unsigned, hipStream_t);             \
  template <>                                                                                  \
  int launch_shared<DT, D>(const RaggedParams&, int, int, int, unsigned, hipStream_t);
FA2_DECLARE_RAGGED(0, 16)
FA2_DECLARE_RAGGED(0, 32)
FA2_DECLARE_RAGGED(0, 64)
FA2_DECLARE_RAGGED(0, 128)
FA2_DECLARE_RAGGED(1, 16)
FA2_DECLARE_RAGGED(1, 32)
FA2_DECLARE_RAGGED(1, 64)
FA2_DECLARE_RAGGED(1, 128)
#undef FA2_DECLARE_RAGGED

}  // namespace fa2
