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

// The ragged attention kernel with 32 * row_waves (1 or 4) rows per workgroup, and after it, with p.shares > 0,
// the merge of the row tiles that its shares cut.
template <int DT, int D>
int launch_ragged(const RaggedParams& p, int source, int row_waves, unsigned grid, hipStream_t stream);

#define FA2_DECLARE_RAGGED(DT, D) \
  template <>                     \
  int launch_ragged<DT, D>(const RaggedParams&, int, int, unsigned, hipStream_t);
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
