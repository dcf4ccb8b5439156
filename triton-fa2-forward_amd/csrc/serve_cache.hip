// serve_cache.hip - rotary positions, and the paged K/V cache written and read.
//
// Rotary: with p a token's position and w_i the pair's frequency,
//   (a, b) -> scale * (a cos(w_i p) - b sin(w_i p), b cos(w_i p) + a sin(w_i p)).
// The angle is formed in float64: at position 10^6 a float32 angle is off by 0.06. A token's angles are the
// same for every head, so a workgroup computes them once per token, in LDS, and its heads share them.
//
// e4m3 rows: e is the least integer with max|x| <= 448 * 2^e (448: the largest e4m3 value), the row is
// stored as e4m3(x * 2^-e) beside the byte e + 127. A power of two makes the product and its inverse
// exact, so a value is rounded once, when it is written; reading it back gives a bf16 or fp16 value
// exactly. What a row cannot hold: NaN and infinities are stored as NaN (e4m3 has no infinity; the scale
// is that of the row's finite values), and at the largest exponent of the row's type the largest
// magnitude is 240 instead of 448, so that no stored value is past the type's own range.
//
// Rotating and reading are bound by HBM, and small calls by the chain of lookups (sequence, length, page), which a group of
// tokens makes together: 16 bytes per lane and load, a row's D / 8 lanes side by side. Writes wait for that chain and the
// angles with few waves in flight, and for a last pass over the rows that may hold few of them (4 tokens of 36 rows: 128 and
// 16). Measured on MI355X (kernel alone): rotary of 16384 x 32 heads of 128 40 us, 6.7 TB/s, of 16 tokens 3.8; a write of 5096
// tokens of 28 + 2 x 4 heads of 64 with their rotation 16 us, 3.0 TB/s (1.5 waves a SIMD on average), of 64 tokens into
// e4m3 5.9, of 16000 tokens of 2 x 8 heads of 128 into e4m3 52 us, 1.9 TB/s (2.7 waves a SIMD; LDS busy 15% of the cycles, bank
// conflicts of the float64 angles 8%); a read of 57071 tokens of 2 x 8 e4m3 heads of 128 71 us, 5 TB/s.
#include <hip/hip_runtime.h>

#include "serve_launch.hpp"
#include "serve_rows.hpp"

namespace fa2 {

namespace {

// ---- rotary ----------------------------------------------------------------------------------

template <int DT, int D>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
  constexpr int LPR = D / 8;  // lanes per row
  __shared__ float cs[kMaxTokensPerWg][kMaxHalf][2];
  const int64_t total = (int64_t)p.batch * p.n;
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens_per_wg;
  const int tokens = (int)min((int64_t)p.tokens_per_wg, total - t0);
  fill_angles(cs, p.rot, tokens, [&](int t) -> int64_t {
    const int64_t b = (t0 + t) / p.n, i = (t0 + t) - b * p.n;
    const int64_t at = b * p.spb + i * p.spn;
    return p.positions64 ? ((const int64_t*)p.positions)[at] : (int64_t)((const int32_t*)p.positions)[at];
  });
  __syncthreads();
  const int chunk = threadIdx.x % LPR;
  const int rows = tokens * p.heads;
  for (int r = threadIdx.x / LPR; r < rows; r += 256 / LPR) {
    const int t = r / p.heads, h = r - t * p.heads;
    const int64_t b = (t0 + t) / p.n, i = (t0 + t) - b * p.n;
    float y[8];
    rotated8<DT, float>(load_chunks(p.x + b * p.sxb + h * p.sxh + i * p.sxn, chunk, p.rot.half, p.rot.interleaved), chunk,
                 p.rot.half, p.rot.interleaved, cs[t], y);
    *(u32x4*)(p.out + b * p.sob + h * p.soh + i * p.son + 8 * chunk) = pack8<DT>(y);
  }
}

// ---- the cache -------------------------------------------------------------------------------

// 16 bytes of the cache a lane: 8 values, or 16 of e4m3
template <int DT, int D, bool E4M3>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheParams p) {
  constexpr int LPR = D / (E4M3 ? 16 : 8), STEP = 256 / LPR, ROWS = 8;
  __shared__ Place places[kMaxTokensPerWg];
  const int t0 = (int)blockIdx.x * p.tokens_per_wg;
  const int tokens = min(p.tokens_per_wg, p.seq.n_tokens - t0);
  if (threadIdx.x < 64) {
    const LanePlace place = find_positions(p.seq, t0, tokens, (int)threadIdx.x);
    const int page = find_page(p.seq, place);
    if ((int)threadIdx.x < tokens) places[threadIdx.x] = Place{place.pos, page};
  }
  __syncthreads();
  const int chunk = threadIdx.x % LPR;
  const int per_token = 2 * p.h_kv;
  const int rows = tokens * per_token;
  for (int r0 = threadIdx.x / LPR; r0 < rows; r0 += ROWS * STEP) {
    u32x4 w[ROWS];
    uint32_t scale[ROWS];
    uint16_t* dst[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const int r = r0 + u * STEP;
      dst[u] = nullptr;
      w[u] = u32x4{0u, 0u, 0u, 0u};
      scale[u] = 0u;
      if (r >= rows) continue;
      const int t = r / per_token, x = r - t * per_token;
      const Place at = places[t];
      if (at.pos < 0) continue;
      const int64_t tok = t0 + t;
      const bool is_v = x >= p.h_kv;
      const int h = is_v ? x - p.h_kv : x;
      dst[u] = is_v ? p.v + tok * p.svt + h * p.svh : p.k + tok * p.skt + h * p.skh;
      if (at.page < 0) continue;
      w[u] = *(const u32x4*)(cache_row(p, is_v, at, h, E4M3 ? 1 : 2) + 16 * chunk);
      if constexpr (E4M3) scale[u] = *scale_row(p, is_v, at, h);
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      if (!dst[u]) continue;
      if constexpr (E4M3) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u32x2 lo = e4m3_to_16<DT>(w[u][2 * i], scale[u]), hi = e4m3_to_16<DT>(w[u][2 * i + 1], scale[u]);
          *(u32x4*)(dst[u] + 16 * chunk + 8 * i) = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      } else {
        *(u32x4*)(dst[u] + 8 * chunk) = w[u];
      }
    }
  }
}

template <int DT, int D>
int launch_rotary_d(const RotaryParams& p, unsigned grid, hipStream_t s) {
  hipLaunchKernelGGL((rotary_kernel<DT, D>), dim3(grid), dim3(256), 0, s, p);
  return (int)hipGetLastError();
}

template <int DT, int D>
int launch_cache_d(bool write, bool e4m3, const CacheParams& p, unsigned grid, hipStream_t s) {
  if (write && e4m3)
    hipLaunchKernelGGL((cache_write_kernel<DT, D, true, CacheParams>), dim3(grid), dim3(256), 0, s, p);
  else if (write)
    hipLaunchKernelGGL((cache_write_kernel<DT, D, false, CacheParams>), dim3(grid), dim3(256), 0, s, p);
  else if (e4m3)
    hipLaunchKernelGGL((cache_read_kernel<DT, D, true>), dim3(grid), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((cache_read_kernel<DT, D, false>), dim3(grid), dim3(256), 0, s, p);
  return (int)hipGetLastError();
}

}  // namespace

int serve_tokens_per_wg(int lanes_per_token, int64_t tokens, int64_t least_wgs) {
  int n = 1;
  while (n < kMaxTokensPerWg && (2 * n * lanes_per_token <= 256 || tokens >= 2 * n * least_wgs)) n *= 2;
  return n;
}

int launch_rotary(int dtype, int head_dim, const RotaryParams& p, unsigned grid, hipStream_t s) {
  switch (dtype * 4 + (head_dim == 16 ? 0 : head_dim == 32 ? 1 : head_dim == 64 ? 2 : 3)) {
    case 0: return launch_rotary_d<0, 16>(p, grid, s);
    case 1: return launch_rotary_d<0, 32>(p, grid, s);
    case 2: return launch_rotary_d<0, 64>(p, grid, s);
    case 3: return launch_rotary_d<0, 128>(p, grid, s);
    case 4: return launch_rotary_d<1, 16>(p, grid, s);
    case 5: return launch_rotary_d<1, 32>(p, grid, s);
    case 6: return launch_rotary_d<1, 64>(p, grid, s);
    default: return launch_rotary_d<1, 128>(p, grid, s);
  }
}

int launch_cache(bool write, int dtype, int head_dim, bool e4m3, const CacheParams& p, unsigned grid,
                 hipStream_t s) {
  switch (dtype * 4 + (head_dim == 16 ? 0 : head_dim == 32 ? 1 : head_dim == 64 ? 2 : 3)) {
    case 0: return launch_cache_d<0, 16>(write, e4m3, p, grid, s);
    case 1: return launch_cache_d<0, 32>(write, e4m3, p, grid, s);
    case 2: return launch_cache_d<0, 64>(write, e4m3, p, grid, s);
    case 3: return launch_cache_d<0, 128>(write, e4m3, p, grid, s);
    case 4: return launch_cache_d<1, 16>(write, e4m3, p, grid, s);
    case 5: return launch_cache_d<1, 32>(write, e4m3, p, grid, s);
    case 6: return launch_cache_d<1, 64>(write, e4m3, p, grid, s);
    default: return launch_cache_d<1, 128>(write, e4m3, p, grid, s);
  }
}

}  // namespace fa2
