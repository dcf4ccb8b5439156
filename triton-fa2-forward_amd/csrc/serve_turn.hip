// serve_turn.hip - queries and keys of a layer made ready for attention in one pass: every head divided by its root
// mean square, then rotated, by one position a token or by the positions of several axes (images, video).
//
//   x_hat = x / sqrt(mean_d x_d^2 + eps) * weight_d
//   (a, b) of pair i -> scale * (a cos t - b sin t, b cos t + a sin t),  t = freqs[i] * position[axes[i]]
//
// Squares and their sum are formed in float64 (a bf16 value's square is past float's range from 1.8e19 on), the
// root's inverse too; products in float, or in float64 for keys on their way into an e4m3 cache, and rounded once.
// Angles as in serve_cache.hip, in float64, once per token for all heads.
#include <hip/hip_runtime.h>

#include "serve_launch.hpp"
#include "serve_rows.hpp"

namespace fa2 {

namespace {

// 16 bytes a lane, D / 8 lanes a row; rows of q and k of a group of tokens, which share the tokens' angles.
template <int DT, int D>
__global__ __launch_bounds__(256) void rotary_qk_kernel(const RotaryQkParams p) {
  constexpr int LPR = D / 8, ROWS = kRowsAtOnce;
  __shared__ float cs[kMaxTokensPerWg][kMaxHalf][2];
  __shared__ float weights[2][D];
  const int64_t total = (int64_t)p.batch * p.n;
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens_per_wg;
  const int tokens = (int)min((int64_t)p.tokens_per_wg, total - t0);
  const int chunk = threadIdx.x % LPR;
  const int heads = p.h_q + p.h_k, rows = tokens * heads;
  const int half = p.rot.half;
  const bool interleaved = p.rot.interleaved;
  for (int base = 0; base < rows; base += ROWS * (256 / LPR)) {
    Chunks in[ROWS];
    uint16_t* dst[ROWS];
    int token[ROWS];  // -1: nothing to do
    bool is_k[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const int r = base + u * (256 / LPR) + (int)threadIdx.x / LPR;
      token[u] = -1;
      if (r >= rows) continue;
      const int t = r / heads, x = r - t * heads;
      const int64_t b = (t0 + t) / p.n, i = (t0 + t) - b * p.n;
      token[u] = t;
      is_k[u] = x >= p.h_q;
      const uint16_t* src = is_k[u] ? p.k + b * p.skb + (x - p.h_q) * p.skh + i * p.skn : p.q + b * p.sqb + x * p.sqh + i * p.sqn;
      dst[u] = is_k[u] ? p.k_out + b * p.skob + (x - p.h_q) * p.skoh + i * p.skon
                       : p.q_out + b * p.sqob + x * p.sqoh + i * p.sqon;
      in[u] = load_chunks(src, chunk, half, interleaved);
    }
    if (base == 0) {  // while the first rows are on their way
      fill_weights<D>(weights, p.turn);
      fill_axes(cs, p.rot, p.turn, tokens, [&](int t, int axis) -> int64_t {
        const int64_t b = (t0 + t) / p.n, i = (t0 + t) - b * p.n;
        return position_at(p.turn, axis * p.turn.spa + b * p.turn.spb + i * p.turn.spn);
      });
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      if (token[u] < 0) continue;
      float y[8];
      turned8<DT, D, float>(p.turn, is_k[u], in[u], chunk, half, interleaved, cs[token[u]], weights, y);
      *(u32x4*)(dst[u] + 8 * chunk) = pack8<DT>(y);
    }
  }
}

template <int DT, int D>
int launch_write_d(bool e4m3, const CacheTurnParams& p, unsigned grid, hipStream_t s) {
  if (e4m3)
    hipLaunchKernelGGL((cache_write_kernel<DT, D, true, CacheTurnParams>), dim3(grid), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((cache_write_kernel<DT, D, false, CacheTurnParams>), dim3(grid), dim3(256), 0, s, p);
  return (int)hipGetLastError();
}

template <int DT, int D>
int launch_qk_d(const RotaryQkParams& p, unsigned grid, hipStream_t s) {
  hipLaunchKernelGGL((rotary_qk_kernel<DT, D>), dim3(grid), dim3(256), 0, s, p);
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
