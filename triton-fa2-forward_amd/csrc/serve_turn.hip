// serve_turn.hip - queries and keys of a layer made ready for attention in one pass: every head divided by its root
// mean square, then rotated, by one position a token or by the positions of several axes (images, video).
//
//   x_hat = x / sqrt(mean_d x_d^2 + eps) * weight_d
//   (a, b) of pair i -> scale * (a cos t - b sin t, b cos t + a sin t),  t = freqs[i] * position[axes[i]]
//
// Squares are summed in float where the sum is well inside its range (a bf16 value's square is past it from 1.8e19 on), in
// float64 elsewhere; products in float, or all of it in float64 for keys on their way into an e4m3 cache, and rounded once.
// Angles as in serve_cache.hip, in float64, once per token for all heads.
//
// Bound by HBM and, beside it, by the vector instructions (about 110 for 16 bytes of a row). Measured on MI355X: 16384 tokens of 32 + 8 heads of
// 128, three axes, both normalised 82 us, 4.1 TB/s (the same with LDS conflicts of the angles 121, at 142 registers 113; a copy
// reaches 4.8); 16 tokens 4.2 (7.0 with a token's heads in one workgroup, one pass after the other); a write of 5096 tokens of 28 + 2 x 4
// heads 21 us, of 64 tokens into e4m3 6.1 (8.1 in one workgroup a token).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "serve_launch.hpp"
#include "serve_rows.hpp"

namespace fa2 {

namespace {

// 16 bytes a lane, D / 8 lanes a row. A workgroup has a group of one batch row's tokens, which share their angles among the heads;
// a lane has the same heads of every token (a pass of 256 lanes over a token's, or over several tokens' where they are few), so
// that their places and weights are worked out once, and loads the next token's row while it turns this one's.
template <int DT, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(6))) void rotary_qk_kernel(const RotaryQkParams p) {
  constexpr int LPR = D / 8, RP = 256 / LPR;  // lanes per row, rows of a pass
  __shared__ alignas(16) float cs[kMaxTokensPerWg][kMaxHalf][2];
  __shared__ alignas(16) float weights[2][D];
  const int groups = (p.n + p.tokens_per_wg - 1) / p.tokens_per_wg;
  const int b = (int)blockIdx.x / groups, t0 = ((int)blockIdx.x - b * groups) * p.tokens_per_wg;
  const int tokens = min(p.tokens_per_wg, p.n - t0);
  const int chunk = threadIdx.x % LPR, row = threadIdx.x / LPR;
  const int heads = p.h_q + p.h_k;
  const int half = p.rot.half;
  const bool interleaved = p.rot.interleaved;
  const int step = max(RP / heads, 1);                // tokens of a pass
  const int sub = heads < RP ? row / heads : 0;       // this lane's
  int head = row - sub * heads + (int)blockIdx.y * RP, t;
  bool is_k = false;
  const uint16_t* src = nullptr;
  uint16_t* dst = nullptr;
  int64_t sn = 0, son = 0;
  Chunks next{};
  auto begin = [&]() {  // on to `head`: its places, and the first token's row on its way
    t = tokens;
    if (head >= heads) return;
    is_k = head >= p.h_q;
    const int h = is_k ? head - p.h_q : head;
    sn = is_k ? p.skn : p.sqn;
    son = is_k ? p.skon : p.sqon;
    src = (is_k ? p.k + b * p.skb + h * p.skh : p.q + b * p.sqb + h * p.sqh) + (t0 + sub) * sn;
    dst = (is_k ? p.k_out + b * p.skob + h * p.skoh : p.q_out + b * p.sqob + h * p.sqoh) + (t0 + sub) * son + 8 * chunk;
    if (sub < step) t = sub;
    if (t < tokens) next = load_chunks(src, chunk, half, interleaved);
    sn *= step;
    son *= step;
  };
  begin();
  fill_weights<D>(weights, p.turn);
  fill_axes(cs, p.rot, p.turn, tokens, [&](int x, int axis) -> int64_t {
    return position_at(p.turn, axis * p.turn.spa + b * p.turn.spb + (t0 + x) * p.turn.spn);
  });
  __syncthreads();
  for (;;) {
    for (; t < tokens; t += step) {
      const Chunks in = next;
      src += sn;
      if (t + step < tokens) next = load_chunks(src, chunk, half, interleaved);
      float y[8];
      turned8<DT, D, float>(p.turn, is_k, in, chunk, half, interleaved, cs[t], weights, y);
      *(u32x4*)dst = pack8<DT>(y);
      dst += son;
    }
    head += RP * (int)gridDim.y;
    if (head >= heads) break;
    begin();
  }
}

// Workgroups below which each pass over a token's heads is one of its own, of rotations and of writes: few tokens wait for one pass after
// the other. Measured on MI355X, one workgroup a token and one a pass: 32 + 8 heads of 128, 3 passes, 16 tokens 6.4 and 4.6 us, 256 6.8 and
// 5.5, 384 7.6 and 6.7, 512 7.8 and 7.4, 700 8.7 and 9.8; written into e4m3 (32 + 2 x 8) 16 7.5 and 6.2, 256 8.3 and 7.2, 320 9.3 and 8.4,
// 384 9.5 and 10.4, 511 9.8 and 12.1; into 16 bits 256 6.8 and 6.2, 320 7.5 and 6.8, 384 7.5 and 7.5, 511 8.0 and 9.7.
constexpr unsigned kTurnFewWgs = 512, kWriteFewWgs = 352;
template <int DT, int D>
int launch_write_d(bool e4m3, const CacheTurnParams& p, unsigned grid, hipStream_t s) {
  const int rows = 256 / (D / 8);
  const int64_t each = (2 * (int64_t)p.h_kv + p.h_q) * p.tokens_per_wg;
  const unsigned passes = grid < kWriteFewWgs && each > rows ? (unsigned)std::min<int64_t>((each + rows - 1) / rows, 64) : 1u;
  if (e4m3)
    hipLaunchKernelGGL((cache_write_kernel<DT, D, true, CacheTurnParams>), dim3(grid, passes), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((cache_write_kernel<DT, D, false, CacheTurnParams>), dim3(grid, passes), dim3(256), 0, s, p);
  return (int)hipGetLastError();
}

template <int DT, int D>
int launch_qk_d(const RotaryQkParams& p, unsigned grid, hipStream_t s) {
  const int rows = 256 / (D / 8), heads = p.h_q + p.h_k;
  const unsigned passes = grid < kTurnFewWgs && heads > rows ? (unsigned)((heads + rows - 1) / rows) : 1u;
  hipLaunchKernelGGL((rotary_qk_kernel<DT, D>), dim3(grid, passes), dim3(256), 0, s, p);
  return (int)hipGetLastError();
}

}  // namespace

int launch_rotary_qk(int dtype, int head_dim, const RotaryQkParams& p, unsigned grid, hipStream_t s) {
  switch (dtype * 4 + (head_dim == 16 ? 0 : head_dim == 32 ? 1 : head_dim == 64 ? 2 : 3)) {
    case 0: return launch_qk_d<0, 16>(p, grid, s);
    case 1: return launch_qk_d<0, 32>(p, grid, s);
    case 2: return launch_qk_d<0, 64>(p, grid, s);
    case 3: return launch_qk_d<0, 128>(p, grid, s);
    case 4: return launch_qk_d<1, 16>(p, grid, s);
    case 5: return launch_qk_d<1, 32>(p, grid, s);
    case 6: return launch_qk_d<1, 64>(p, grid, s);
    default: return launch_qk_d<1, 128>(p, grid, s);
  }
}

int launch_cache_write_turn(int dtype, int head_dim, bool e4m3, const CacheTurnParams& p, unsigned grid, hipStream_t s) {
  switch (dtype * 4 + (head_dim == 16 ? 0 : head_dim == 32 ? 1 : head_dim == 64 ? 2 : 3)) {
    case 0: return launch_write_d<0, 16>(e4m3, p, grid, s);
    case 1: return launch_write_d<0, 32>(e4m3, p, grid, s);
    case 2: return launch_write_d<0, 64>(e4m3, p, grid, s);
    case 3: return launch_write_d<0, 128>(e4m3, p, grid, s);
    case 4: return launch_write_d<1, 16>(e4m3, p, grid, s);
    case 5: return launch_write_d<1, 32>(e4m3, p, grid, s);
    case 6: return launch_write_d<1, 64>(e4m3, p, grid, s);
    default: return launch_write_d<1, 128>(e4m3, p, grid, s);
  }
}

}  // namespace fa2
