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

#include <type_traits>

#include "serve_common.hpp"
#include "serve_launch.hpp"

namespace fa2 {

namespace {

constexpr int kMaxTokensPerWg = 16;
constexpr int kRowsAtOnce = 4;  // rows of a lane whose loads are in flight together
// Scale bytes that a workgroup of several tokens keeps until its end, to store those of a head and page side by side.
// Measured on MI355X: 16000 tokens of 2 x 8 heads of 128, keys rotated: 56 us a byte a store, 48 gathered.
constexpr int kScalesAtOnce = 1024;
constexpr int kMaxHalf = 64;  // head_dim 128, all of it rotated

// cos and sin of 2 pi x for |x| <= 1/2 turns
__device__ __forceinline__ void sincos_turns(double x, double* s, double* c) { sincospi(2.0 * x, s, c); }

// cos and sin (times scale) of every pair's angle at the workgroup's tokens, formed in float64, into cs[token][pair][2] of
// type A: float, rounded once, or double where the products are formed in float64.
template <class A, class Position>
__device__ __forceinline__ void fill_angles(A (*cs)[kMaxHalf][2], const RotaryPlan& rot, int tokens, Position&& position) {
  const int n = tokens * rot.half;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int t = i / rot.half, f = i - t * rot.half;
    const double turns = (double)position(t) * rot.freqs[f] * 0.15915494309189533577;  // 1 / (2 pi)
    double s, c;
    sincos_turns(turns - rint(turns), &s, &c);
    cs[t][f][0] = (A)(c * rot.scale);
    cs[t][f][1] = (A)(s * rot.scale);
  }
}

// This lane's 8 values x[8 chunk ..] of a row, and with them the 8 that they are paired with where those lie in
// another chunk of the row
struct Chunks {
  u32x4 own, other;
};
__device__ __forceinline__ Chunks load_chunks(const uint16_t* row, int chunk, int half, bool interleaved) {
  Chunks x;
  x.own = *(const u32x4*)(row + 8 * chunk);
  x.other = u32x4{0u, 0u, 0u, 0u};
  const int d0 = 8 * chunk;
  if (d0 < 2 * half && !interleaved) x.other = *(const u32x4*)(row + (d0 >= half ? d0 - half : d0 + half));
  return x;
}

// ... rotated (T: the type the products and sums are formed in, rounded to float once)
template <int DT, class T, class A>
__device__ __forceinline__ void rotated8(const Chunks& in, int chunk, int half, bool interleaved,
                                         const A (*cs)[2], float (&y)[8]) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = to_f32<DT>((uint16_t)in.own[i]);
    x[2 * i + 1] = to_f32<DT>((uint16_t)(in.own[i] >> 16));
  }
  const int d0 = 8 * chunk;
  if (d0 >= 2 * half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
  } else if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T c = (T)cs[d0 / 2 + i][0], s = (T)cs[d0 / 2 + i][1];
      y[2 * i] = (float)((T)x[2 * i] * c - (T)x[2 * i + 1] * s);
      y[2 * i + 1] = (float)((T)x[2 * i + 1] * c + (T)x[2 * i] * s);
    }
  } else {
    const bool second = d0 >= half;
    const int f0 = second ? d0 - half : d0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T c = (T)cs[f0 + i][0], s = (T)cs[f0 + i][1];
      const T o = (T)to_f32<DT>((uint16_t)(in.other[i / 2] >> (16 * (i & 1))));
      y[i] = (float)((T)x[i] * c + (second ? o * s : -(o * s)));
    }
  }
}

template <int DT>
__device__ __forceinline__ u32x4 pack8(const float (&y)[8]) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = Elem<DT>::pack2(y[2 * i], y[2 * i + 1]);
  return r;
}

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

// Where a row of K (or V) lies in the cache, in elements, and its scale byte. Both tensors' strides are scalars and
// the choice between them is made value by value: a reference to one of them, chosen per lane, would
// have every lane load the strides from the kernel's arguments.
__device__ __forceinline__ int64_t pick(bool second, int64_t a, int64_t b) { return second ? b : a; }
__device__ __forceinline__ char* cache_row(const CacheParams& p, bool v, const Place& at, int head, int bytes) {
  const int64_t row = at.pos & ((1 << p.seq.page_shift) - 1);
  return (v ? p.vc.data : p.kc.data) + bytes * (at.page * pick(v, p.kc.page, p.vc.page) + head * pick(v, p.kc.head, p.vc.head) +
                                                row * pick(v, p.kc.token, p.vc.token));
}
__device__ __forceinline__ uint8_t* scale_row(const CacheParams& p, bool v, const Place& at, int head) {
  const int64_t row = at.pos & ((1 << p.seq.page_shift) - 1);
  return (v ? p.vc.scale : p.kc.scale) + at.page * pick(v, p.kc.scale_page, p.vc.scale_page) +
         head * pick(v, p.kc.scale_head, p.vc.scale_head) + row * pick(v, p.kc.scale_token, p.vc.scale_token);
}

// One row's 8 values of this lane as e4m3, with the row's scale byte (D / 8 lanes hold a row).
template <int DT, int D>
__device__ __forceinline__ u32x2 quantise8(const float (&y)[8], uint32_t* scale_byte) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(y[i]);
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
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = y[4 * h + i] * inv;
      z[i] = fabsf(x) < INFINITY ? fminf(fmaxf(x, -limit), limit) : __uint_as_float(0x7fc00000u);
    }
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], r, true);
  }
  return u32x2{w[0], w[1]};
}

// Rows per token: K heads, V heads, then (q) query heads. K of an e4m3 cache is rotated in float64 and rounded to float
// once: products in float would take more of the values next to a border between two e4m3 values across it.
// Scaling by a power of two adds no rounding. (V and what is not rotated in float: rows in float64 throughout took
// 136 us where 125 are enough, 16000 tokens of 32 + 2 x 8 heads of 128.)
template <int DT, int D, bool E4M3>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheParams p) {
  constexpr int LPR = D / 8;
  using Angle = std::conditional_t<E4M3, double, float>;
  __shared__ Angle cs[kMaxTokensPerWg][kMaxHalf][2];
  __shared__ Place places[kMaxTokensPerWg];
  __shared__ uint8_t scales[E4M3 ? kScalesAtOnce : 1];  // [K and V heads][tokens]
  const int t0 = (int)blockIdx.x * p.tokens_per_wg;
  const int tokens = min(p.tokens_per_wg, p.seq.n_tokens - t0);
  const bool gather = E4M3 && tokens > 1 && (int64_t)tokens * 2 * p.h_kv <= kScalesAtOnce;
  const int chunk = threadIdx.x % LPR;
  const int per_token = 2 * p.h_kv + (p.q ? p.h_q : 0);
  const int rows = tokens * per_token;
  const int half = p.rot.half;
  const bool interleaved = p.rot.interleaved;
  for (int base = 0; base < rows; base += kRowsAtOnce * (256 / LPR)) {
    Chunks in[kRowsAtOnce];
    int token[kRowsAtOnce], which[kRowsAtOnce];  // row `which` of the token's; -1: nothing to do
#pragma unroll
    for (int u = 0; u < kRowsAtOnce; ++u) {
      const int r = base + u * (256 / LPR) + (int)threadIdx.x / LPR;
      token[u] = r / per_token;
      which[u] = r < rows ? r - token[u] * per_token : -1;
      if (r >= rows) continue;
      const int x = which[u];
      const int64_t tok = t0 + token[u];
      const bool is_q = x >= 2 * p.h_kv, is_v = !is_q && x >= p.h_kv;
      const uint16_t* src = is_q ? p.q : is_v ? p.v : p.k;
      const int64_t at = tok * (is_q ? p.sqt : is_v ? p.svt : p.skt) +
                         (is_q ? x - 2 * p.h_kv : is_v ? x - p.h_kv : x) * (is_q ? p.sqh : is_v ? p.svh : p.skh);
      in[u] = load_chunks(src + at, chunk, is_v ? 0 : half, interleaved);
    }
    if (base == 0) {  // while the first rows are on their way
      LanePlace place;
      int page = -1;
      const bool looks_up = threadIdx.x < 64;
      if (looks_up) {
        place = find_positions(p.seq, t0, tokens, (int)threadIdx.x);
        if ((int)threadIdx.x < tokens) places[threadIdx.x].pos = place.pos;
        page = find_page(p.seq, place);  // on its way while the angles are computed
      }
      __syncthreads();
      if (p.rot.half) fill_angles(cs, p.rot, tokens, [&](int t) -> int64_t { return places[t].pos; });
      if (looks_up && (int)threadIdx.x < tokens) places[threadIdx.x].page = page;
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kRowsAtOnce; ++u) {
      const int x = which[u];
      if (x < 0) continue;
      const Place at = places[token[u]];
      if (at.pos < 0) continue;
      const Angle(*angles)[2] = cs[token[u]];
      if (x >= 2 * p.h_kv) {
        float y[8];
        rotated8<DT, float>(in[u], chunk, half, interleaved, angles, y);
        *(u32x4*)(p.q_out + (int64_t)(t0 + token[u]) * p.sot + (x - 2 * p.h_kv) * p.soh + 8 * chunk) = pack8<DT>(y);
        continue;
      }
      if (at.page < 0) continue;
      const bool is_v = x >= p.h_kv;
      const int h = is_v ? x - p.h_kv : x;
      char* dst = cache_row(p, is_v, at, h, E4M3 ? 1 : 2);
      if constexpr (E4M3) {
        float y[8];
        if (is_v || half == 0)
          rotated8<DT, float>(in[u], chunk, 0, interleaved, angles, y);
        else
          rotated8<DT, double>(in[u], chunk, half, interleaved, angles, y);
        uint32_t byte;
        const u32x2 w = quantise8<DT, D>(y, &byte);
        *(u32x2*)(dst + 8 * chunk) = w;
        if (chunk == 0) {
          if (gather)
            scales[x * tokens + token[u]] = (uint8_t)byte;
          else
            *scale_row(p, is_v, at, h) = (uint8_t)byte;
        }
      } else {
        float y[8];
        rotated8<DT, float>(in[u], chunk, is_v ? 0 : half, interleaved, angles, y);
        *(u32x4*)(dst + 16 * chunk) = pack8<DT>(y);
      }
    }
  }
  if constexpr (E4M3) {
    if (!gather) return;
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * 2 * p.h_kv; i += 256) {
      const int x = i / tokens;
      const Place at = places[i - x * tokens];
      const bool is_v = x >= p.h_kv;
      if (at.pos >= 0 && at.page >= 0) *scale_row(p, is_v, at, is_v ? x - p.h_kv : x) = scales[i];
    }
  }
}

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
