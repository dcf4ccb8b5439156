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
// All of it is bound by HBM: 16 bytes per lane and load, a row's D / 8 lanes side by side.
#include <hip/hip_runtime.h>

#include "serve_common.hpp"
#include "serve_launch.hpp"

namespace fa2 {

namespace {

constexpr int kMaxTokensPerWg = 8;
constexpr int kMaxHalf = 64;  // head_dim 128, all of it rotated

// cos and sin of 2 pi x for |x| <= 1/2 turns
__device__ __forceinline__ void sincos_turns(double x, double* s, double* c) { sincospi(2.0 * x, s, c); }

// cos and sin (times scale) of every pair's angle at the workgroup's tokens, into cs[token][pair][2]
template <class Position>
__device__ __forceinline__ void fill_angles(double (*cs)[kMaxHalf][2], const RotaryPlan& rot, int tokens,
                                            Position&& position) {
  const int n = tokens * rot.half;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int t = i / rot.half, f = i - t * rot.half;
    const double turns = (double)position(t) * rot.freqs[f] * 0.15915494309189533577;  // 1 / (2 pi)
    double s, c;
    sincos_turns(turns - rint(turns), &s, &c);
    cs[t][f][0] = c * rot.scale;
    cs[t][f][1] = s * rot.scale;
  }
}

// The 8 values x[8 chunk ..] of a row, rotated (T: the type the products are formed in)
template <int DT, class T>
__device__ __forceinline__ void rotated8(const uint16_t* row, int chunk, const RotaryPlan& rot,
                                         const double (*cs)[2], T (&y)[8]) {
  const u32x4 own = *(const u32x4*)(row + 8 * chunk);
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = to_f32<DT>((uint16_t)own[i]);
    x[2 * i + 1] = to_f32<DT>((uint16_t)(own[i] >> 16));
  }
  const int d0 = 8 * chunk;
  if (d0 >= 2 * rot.half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
  } else if (rot.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T c = (T)cs[d0 / 2 + i][0], s = (T)cs[d0 / 2 + i][1];
      y[2 * i] = (T)x[2 * i] * c - (T)x[2 * i + 1] * s;
      y[2 * i + 1] = (T)x[2 * i + 1] * c + (T)x[2 * i] * s;
    }
  } else {
    const bool second = d0 >= rot.half;
    const int f0 = second ? d0 - rot.half : d0;
    const u32x4 other = *(const u32x4*)(row + (second ? f0 : d0 + rot.half));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T c = (T)cs[f0 + i][0], s = (T)cs[f0 + i][1];
      const T o = (T)to_f32<DT>((uint16_t)(other[i / 2] >> (16 * (i & 1))));
      y[i] = (T)x[i] * c + (second ? o * s : -(o * s));
    }
  }
}

template <int DT, class T>
__device__ __forceinline__ u32x4 pack8(const T (&y)[8]) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = Elem<DT>::pack2((float)y[2 * i], (float)y[2 * i + 1]);
  return r;
}

// ---- rotary ----------------------------------------------------------------------------------

template <int DT, int D>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
  constexpr int LPR = D / 8;  // lanes per row
  __shared__ double cs[kMaxTokensPerWg][kMaxHalf][2];
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
    rotated8<DT>(p.x + b * p.sxb + h * p.sxh + i * p.sxn, chunk, p.rot, cs[t], y);
    *(u32x4*)(p.out + b * p.sob + h * p.soh + i * p.son + 8 * chunk) = pack8<DT>(y);
  }
}

// ---- the cache -------------------------------------------------------------------------------

__device__ __forceinline__ char* cache_row(const CacheTensor& c, const Place& p, int head, int page_shift,
                                           int bytes) {
  const int64_t at = p.page * c.page + head * c.head + (int64_t)(p.pos & ((1 << page_shift) - 1)) * c.token;
  return c.data + at * bytes;
}
__device__ __forceinline__ uint8_t* scale_row(const CacheTensor& c, const Place& p, int head, int page_shift) {
  return c.scale + p.page * c.scale_page + head * c.scale_head +
         (int64_t)(p.pos & ((1 << page_shift) - 1)) * c.scale_token;
}

// One row's 8 values of this lane as e4m3, with the row's scale byte (D / 8 lanes hold a row).
template <int DT, int D, class T>
__device__ __forceinline__ u32x2 quantise8(const T (&y)[8], uint32_t* scale_byte) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf((float)y[i]);
    top = a < INFINITY ? fmaxf(top, a) : top;  // finite values only (false for NaN)
  }
#pragma unroll
  for (int off = D / 16; off >= 1; off /= 2) top = fmaxf(top, __shfl_xor(top, off, 64));
  // top = m 2^(k - 1), 1 <= m < 2; 448 = 1.75 * 2^8
  const uint32_t bits = __float_as_uint(top);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  constexpr int kLargest = DT == 0 ? 8 : 120;  // 240 * 2^e is the type's largest power-of-two multiple
  e = min(max(e, -126), kLargest);
  const float limit = e == kLargest ? 240.f : 448.f;
  *scale_byte = (uint32_t)(e + 127);
  const T inv = (T)__uint_as_float((uint32_t)(127 - e) << 23);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = (float)(y[4 * h + i] * inv);
      z[i] = fabsf(x) < INFINITY ? fminf(fmaxf(x, -limit), limit) : __uint_as_float(0x7fc00000u);
    }
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], r, true);
  }
  return u32x2{w[0], w[1]};
}

// The places of the workgroup's tokens, a wave per token in turn
__device__ __forceinline__ void fill_places(Place* places, const Sequences& q, int t0, int tokens) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int t = wave; t < tokens; t += 4) {
    const Place p = find_place(q, t0 + t, lane);
    if (lane == 0) places[t] = p;
  }
}

// Rows per token: K heads, V heads, then (q) query heads. K is rotated in float64: a rotated value next to
// a border between two e4m3 values goes to the one that its exact value goes to.
template <int DT, int D, bool E4M3>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheParams p) {
  constexpr int LPR = D / 8;
  __shared__ double cs[kMaxTokensPerWg][kMaxHalf][2];
  __shared__ Place places[kMaxTokensPerWg];
  const int t0 = (int)blockIdx.x * p.tokens_per_wg;
  const int tokens = min(p.tokens_per_wg, p.seq.n_tokens - t0);
  fill_places(places, p.seq, t0, tokens);
  __syncthreads();
  if (p.rot.half) {
    fill_angles(cs, p.rot, tokens, [&](int t) -> int64_t { return places[t].pos; });
    __syncthreads();
  }
  const int chunk = threadIdx.x % LPR;
  const int per_token = 2 * p.h_kv + (p.q ? p.h_q : 0);
  const int rows = tokens * per_token;
  RotaryPlan none = p.rot;
  none.half = 0;
  for (int r = threadIdx.x / LPR; r < rows; r += 256 / LPR) {
    const int t = r / per_token, x = r - t * per_token;
    const Place at = places[t];
    if (at.seq < 0) continue;
    const int64_t tok = t0 + t;
    if (x >= 2 * p.h_kv) {
      const int h = x - 2 * p.h_kv;
      float y[8];
      rotated8<DT>(p.q + tok * p.sqt + h * p.sqh, chunk, p.rot, cs[t], y);
      *(u32x4*)(p.q_out + tok * p.sot + h * p.soh + 8 * chunk) = pack8<DT>(y);
      continue;
    }
    if (at.page < 0) continue;
    const bool is_v = x >= p.h_kv;
    const int h = is_v ? x - p.h_kv : x;
    const uint16_t* src = is_v ? p.v + tok * p.svt + h * p.svh : p.k + tok * p.skt + h * p.skh;
    const CacheTensor& c = is_v ? p.vc : p.kc;
    char* dst = cache_row(c, at, h, p.seq.page_shift, E4M3 ? 1 : 2);
    if constexpr (E4M3) {
      double y[8];
      rotated8<DT>(src, chunk, is_v ? none : p.rot, cs[t], y);
      uint32_t byte;
      const u32x2 w = quantise8<DT, D>(y, &byte);
      *(u32x2*)(dst + 8 * chunk) = w;
      if (chunk == 0) *scale_row(c, at, h, p.seq.page_shift) = (uint8_t)byte;
    } else {
      float y[8];
      rotated8<DT>(src, chunk, is_v ? none : p.rot, cs[t], y);
      *(u32x4*)(dst + 16 * chunk) = pack8<DT>(y);
    }
  }
}

template <int DT, int D, bool E4M3>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheParams p) {
  constexpr int LPR = D / 8;
  __shared__ Place places[kMaxTokensPerWg];
  const int t0 = (int)blockIdx.x * p.tokens_per_wg;
  const int tokens = min(p.tokens_per_wg, p.seq.n_tokens - t0);
  fill_places(places, p.seq, t0, tokens);
  __syncthreads();
  const int chunk = threadIdx.x % LPR;
  const int rows = tokens * 2 * p.h_kv;
  for (int r = threadIdx.x / LPR; r < rows; r += 256 / LPR) {
    const int t = r / (2 * p.h_kv), x = r - t * 2 * p.h_kv;
    const Place at = places[t];
    if (at.seq < 0) continue;
    const int64_t tok = t0 + t;
    const bool is_v = x >= p.h_kv;
    const int h = is_v ? x - p.h_kv : x;
    const CacheTensor& c = is_v ? p.vc : p.kc;
    u32x4 w = {0u, 0u, 0u, 0u};
    if (at.page >= 0) {
      const char* src = cache_row(c, at, h, p.seq.page_shift, E4M3 ? 1 : 2);
      if constexpr (E4M3) {
        const u32x2 b = *(const u32x2*)(src + 8 * chunk);
        const uint32_t scale = *scale_row(c, at, h, p.seq.page_shift);
        const u32x2 lo = e4m3_to_16<DT>(b[0], scale), hi = e4m3_to_16<DT>(b[1], scale);
        w = u32x4{lo[0], lo[1], hi[0], hi[1]};
      } else {
        w = *(const u32x4*)(src + 16 * chunk);
      }
    }
    uint16_t* dst = is_v ? p.v + tok * p.svt + h * p.svh : p.k + tok * p.skt + h * p.skh;
    *(u32x4*)(dst + 8 * chunk) = w;
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
    hipLaunchKernelGGL((cache_write_kernel<DT, D, true>), dim3(grid), dim3(256), 0, s, p);
  else if (write)
    hipLaunchKernelGGL((cache_write_kernel<DT, D, false>), dim3(grid), dim3(256), 0, s, p);
  else if (e4m3)
    hipLaunchKernelGGL((cache_read_kernel<DT, D, true>), dim3(grid), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((cache_read_kernel<DT, D, false>), dim3(grid), dim3(256), 0, s, p);
  return (int)hipGetLastError();
}

}  // namespace

int serve_tokens_per_wg(int lanes_per_token) {
  int n = 1;
  while (n < kMaxTokensPerWg && 2 * n * lanes_per_token <= 256) n *= 2;
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
