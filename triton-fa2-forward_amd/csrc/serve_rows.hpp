// serve_rows.hpp - device code that the rotary and cache kernels share: a token's angles, a lane's eight values of a row
// rotated, a row's place in the cache, and its rounding to e4m3.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "serve_common.hpp"

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

// 1 / sqrt(m), m > 0: the instruction's estimate and Newton's steps (m = inf, of an infinite value: 0)
template <int STEPS>
__device__ __forceinline__ double inverse_root(double m) {
  double r = __builtin_amdgcn_rsq(m);
  const double half = 0.5 * m;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const double e = __builtin_fma(-half * r, r, 0.5);
    r = m < __builtin_inf() ? __builtin_fma(r, e, r) : r;
  }
  return r;
}

// A value on its way to e4m3: float64 rounded to float to odd (to the neighbour whose last bit is set, where it is not a
// float), so that rounding that again, to fewer bits, is as rounding the float64 value.
__device__ __forceinline__ float rounded(float x) { return x; }
__device__ __forceinline__ float rounded(double x) {
  const float f = (float)x;
  const uint32_t bits = __float_as_uint(f);
  const double off = fabs(x) - (double)fabsf(f);
  return (bits & 1u) || !(off != 0.0) || !(fabsf(f) < INFINITY) ? f : __uint_as_float(off > 0.0 ? bits + 1u : bits - 1u);
}

// The sum over the 2, 4, 8 or 16 neighbouring lanes that hold a row
template <int LANES>
__device__ __forceinline__ float row_sum(float x) {
  auto with = [&](auto ctrl) {
    constexpr int c = decltype(ctrl)::value;
    x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), c, 0xf, 0xf, true));
  };
  with(std::integral_constant<int, 0xb1>{});                           // neighbours
  if constexpr (LANES >= 4) with(std::integral_constant<int, 0x4e>{});  // pairs of a quad
  if constexpr (LANES >= 8) with(std::integral_constant<int, 0x141>{});  // quads of 8
  if constexpr (LANES >= 16) with(std::integral_constant<int, 0x140>{});
  return x;
}
// Two bf16 values times 2^k: exact, but where a product leaves bf16's normal numbers at their lower end
__device__ __forceinline__ uint32_t scaled(uint32_t pair, int k) {
  const float lo = __builtin_amdgcn_ldexpf(__uint_as_float(pair << 16), k);
  const float hi = __builtin_amdgcn_ldexpf(__uint_as_float(pair & 0xffff0000u), k);
  return (__float_as_uint(lo) >> 16) | (__float_as_uint(hi) & 0xffff0000u);
}

// 1 / sqrt(mean x^2 + eps) of the row, in float64, or in float where the squares' sum and eps are well inside its range. As a float it
// may be past its range: above for rows of zeros, whatever it is, and for bf16 rows below 2^-126, whose values take 2^16 of it; below for
// the largest bf16 rows and for an eps from 2^240 on, where bf16 values take as much of it as leaves it at 2^-64 (values that are
// no normal numbers then are results below 2^-189; of fp16 all results are below 2^-104).
template <int DT, int D, class T>
__device__ __forceinline__ T inverse_rms(Chunks& in, double eps) {
  if constexpr (sizeof(T) == 4) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = Elem<DT>::sumsq2(in.own[i], sum);
    sum = row_sum<D / 8>(sum);
    if (sum > 1e-30f && sum < 1e30f && eps < 1e30) return __builtin_amdgcn_rsqf(__builtin_fmaf(sum, 1.0f / D, (float)eps));
  }
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double x = (double)to_f32<DT>((uint16_t)(in.own[i / 2] >> (16 * (i & 1))));
    sum = __builtin_fma(x, x, sum);
  }
#pragma unroll
  for (int off = D / 16; off >= 1; off /= 2) sum += __shfl_xor(sum, off, 64);
  double r = inverse_root<sizeof(T) == 8 ? 3 : 1>(sum * (1.0 / D) + eps);
  if constexpr (sizeof(T) == 4) {
    const bool above = r > 0x1p126, below = r > 0.0 && r < 0x1p-120;  // (0: of an infinite value)
    if (DT == 1 && (above || below)) {
      const int k = above ? 16 : 64 + __builtin_amdgcn_frexp_exp(r);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        in.own[i] = scaled(in.own[i], k);
        in.other[i] = scaled(in.other[i], k);
      }
      r = __builtin_amdgcn_ldexp(r, -k);
    }
    if (above) r = fmin(r, 0x1p126);
  }
  return (T)r;
}

// Where pair f's angle and dim d's weight lie in LDS: in units of 16 bytes, the i-th units of all chunks side by side, so that
// the lanes of a row read neighbouring units. Measured on MI355X, 16384 tokens of 40 heads of 128: in their own order, four
// lanes to a bank, 121 us, LDS busy 55% of the cycles.
template <class A>
__device__ __forceinline__ int angle_slot(int chunk, int i) {  // f = 8 chunk + i
  constexpr int PER = 8 / sizeof(A);                           // pairs of a unit
  return (i / PER * (kMaxHalf / 8) + chunk) * PER + i % PER;
}
template <int D>
__device__ __forceinline__ int weight_slot(int chunk, int i) {
  return (i / 4 * (D / 8) + chunk) * 4 + i % 4;
}

// This lane's 8 values of a row (D / 8 lanes hold it) normalised (NORM) and rotated: rotated8 of
// x / sqrt(mean x^2 + eps) * weight
template <int DT, int D, class T, bool NORM, class A>
__device__ __forceinline__ void normed_rotated8(Chunks in, int chunk, int half, bool interleaved, const A (*cs)[2],
                                                const float* weight, double eps, float (&y)[8]) {
  T r = 1;
  if constexpr (NORM) r = inverse_rms<DT, D, T>(in, eps);
  auto value = [&](uint32_t pair, int i) { return (T)to_f32<DT>((uint16_t)(pair >> (16 * (i & 1)))); };
  const int d0 = 8 * chunk;
  T a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = NORM ? value(in.own[i / 2], i) * r * (T)weight[weight_slot<D>(chunk, i)] : value(in.own[i / 2], i);
  if (d0 >= 2 * half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = rounded(a[i]);
  } else if (interleaved) {  // four pairs, the first or the last of an angles' chunk
    cs += angle_slot<A>(chunk / 2, 0) + (chunk & 1) * angle_slot<A>(0, 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const A* angle = cs[angle_slot<A>(0, i)];
      const T c = (T)angle[0], s = (T)angle[1];
      y[2 * i] = rounded(a[2 * i] * c - a[2 * i + 1] * s);
      y[2 * i + 1] = rounded(a[2 * i + 1] * c + a[2 * i] * s);
    }
  } else {
    const bool second = d0 >= half;
    const int first = second ? chunk - half / 8 : chunk, other = second ? first : chunk + half / 8;
    cs += angle_slot<A>(first, 0);
    const T sign = second ? r : -r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const A* angle = cs[angle_slot<A>(0, i)];
      const T c = (T)angle[0], s = (T)angle[1];
      const T o = NORM ? value(in.other[i / 2], i) * sign * (T)weight[weight_slot<D>(other, i)] : value(in.other[i / 2], i);
      y[i] = rounded(a[i] * c + (NORM || second ? o * s : -(o * s)));
    }
  }
}

// fill_angles with a position per axis, into angle_slot's places
template <class A, class Position>
__device__ __forceinline__ void fill_axes(A (*cs)[kMaxHalf][2], const RotaryPlan& rot, const TurnParams& turn, int tokens,
                                          Position&& position) {
  const int n = tokens * rot.half;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int t = i / rot.half, f = i - t * rot.half;
    const int axis = turn.axes ? min(max(turn.axes[f], 0), turn.n_axes - 1) : 0;
    const double turns = (double)position(t, axis) * rot.freqs[f] * 0.15915494309189533577;  // 1 / (2 pi)
    double s, c;
    sincos_turns(turns - rint(turns), &s, &c);
    A(&at)[2] = cs[t][angle_slot<A>(f / 8, f % 8)];
    at[0] = (A)(c * rot.scale);
    at[1] = (A)(s * rot.scale);
  }
}
__device__ __forceinline__ int64_t position_at(const TurnParams& t, int64_t at) {
  return t.positions64 ? ((const int64_t*)t.positions)[at] : (int64_t)((const int32_t*)t.positions)[at];
}

// The weights of both tensors in LDS: lanes read those of their chunk, and of the chunk that it is paired with
template <int D>
__device__ __forceinline__ void fill_weights(float (&weights)[2][D], const TurnParams& turn) {
  for (int i = threadIdx.x; i < 2 * D; i += 256) {
    const float* w = i < D ? turn.q_weight : turn.k_weight;
    if (w) weights[i / D][weight_slot<D>(i % D / 8, i % 8)] = w[i % D];
  }
}

template <int DT, int D, class T, class A, class Weights>
__device__ __forceinline__ void turned8(const TurnParams& t, bool is_k, const Chunks& in, int chunk, int half, bool interleaved,
                                        const A (*cs)[2], const Weights& weights, float (&y)[8]) {
  if (is_k ? t.k_weight != nullptr : t.q_weight != nullptr)
    normed_rotated8<DT, D, T, true>(in, chunk, half, interleaved, cs, weights[is_k], is_k ? t.k_eps : t.q_eps, y);
  else
    normed_rotated8<DT, D, T, false>(in, chunk, half, interleaved, cs, weights[is_k], 0.0, y);
}

// Rows per token: K heads, V heads, then (q) query heads. K of an e4m3 cache is rotated in float64 and rounded to float
// once: products in float would take more of the values next to a border between two e4m3 values across it.
// Scaling by a power of two adds no rounding. (V and what is not rotated in float: rows in float64 throughout took
// 136 us where 125 are enough, 16000 tokens of 32 + 2 x 8 heads of 128.)
// Params: CacheParams, or CacheTurnParams (rows of q and k normalised and rotated by their own positions, turned8).
template <int DT, int D, bool E4M3, class Params>
__global__ __launch_bounds__(256) void cache_write_kernel(const Params p) {
  constexpr bool kTurn = std::is_same_v<Params, CacheTurnParams>;
  constexpr int LPR = D / 8;
  using Angle = std::conditional_t<E4M3, double, float>;
  __shared__ alignas(16) Angle cs[kMaxTokensPerWg][kMaxHalf][2];
  __shared__ Place places[kMaxTokensPerWg];
  __shared__ alignas(16) float weights[kTurn ? 2 : 1][kTurn ? D : 1];
  __shared__ uint8_t scales[E4M3 ? kScalesAtOnce : 1];  // [K and V heads][tokens]
  const int t0 = (int)blockIdx.x * p.tokens_per_wg;
  const int tokens = min(p.tokens_per_wg, p.seq.n_tokens - t0);
  const bool gather = E4M3 && tokens > 1 && (!kTurn || gridDim.y == 1) && (int64_t)tokens * 2 * p.h_kv <= kScalesAtOnce;
  const int chunk = threadIdx.x % LPR;
  const int per_token = 2 * p.h_kv + (p.q ? p.h_q : 0);
  const int rows = tokens * per_token;
  const int half = p.rot.half;
  const bool interleaved = p.rot.interleaved;
  auto look_up = [&]() {
    LanePlace place;
    int page = -1;
    const bool looks_up = threadIdx.x < 64;
    if (looks_up) {
      place = find_positions(p.seq, t0, tokens, (int)threadIdx.x);
      if ((int)threadIdx.x < tokens) places[threadIdx.x].pos = place.pos;
      page = find_page(p.seq, place);  // on its way while the angles are computed
    }
    __syncthreads();
    if constexpr (kTurn) {
      fill_weights<D>(weights, p.turn);
      fill_axes(cs, p.rot, p.turn, tokens, [&](int t, int axis) -> int64_t {
        return p.turn.positions ? position_at(p.turn, axis * p.turn.spa + (t0 + t) * p.turn.spn) : (int64_t)places[t].pos;
      });
    } else {
      if (p.rot.half) fill_angles(cs, p.rot, tokens, [&](int t) -> int64_t { return places[t].pos; });
    }
    if (looks_up && (int)threadIdx.x < tokens) places[threadIdx.x].page = page;
    __syncthreads();
  };
  // Turned rows: the places and angles first, so that what they need does not stay in registers; few tokens' rows are dealt out to
  // several workgroups, which each work those out.
  const int share = kTurn ? (rows + (256 / LPR) * (int)gridDim.y - 1) / ((256 / LPR) * (int)gridDim.y) * (256 / LPR) : rows;
  const int row0 = kTurn ? (int)blockIdx.y * share : 0, row_end = kTurn ? min(row0 + share, rows) : rows;
  if constexpr (kTurn) look_up();
  for (int base = row0; base < row_end; base += kRowsAtOnce * (256 / LPR)) {
    Chunks in[kRowsAtOnce];
    int token[kRowsAtOnce], which[kRowsAtOnce];  // row `which` of the token's; -1: nothing to do
#pragma unroll
    for (int u = 0; u < kRowsAtOnce; ++u) {
      const int r = base + u * (256 / LPR) + (int)threadIdx.x / LPR;
      token[u] = r / per_token;
      which[u] = r < row_end ? r - token[u] * per_token : -1;
      if (r >= row_end) continue;
      const int x = which[u];
      const int64_t tok = t0 + token[u];
      const bool is_q = x >= 2 * p.h_kv, is_v = !is_q && x >= p.h_kv;
      const uint16_t* src = is_q ? p.q : is_v ? p.v : p.k;
      const int64_t at = tok * (is_q ? p.sqt : is_v ? p.svt : p.skt) +
                         (is_q ? x - 2 * p.h_kv : is_v ? x - p.h_kv : x) * (is_q ? p.sqh : is_v ? p.svh : p.skh);
      in[u] = load_chunks(src + at, chunk, is_v ? 0 : half, interleaved);
    }
    if constexpr (!kTurn) {
      if (base == 0) look_up();  // while the first rows are on their way
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
        if constexpr (kTurn)
          turned8<DT, D, float>(p.turn, false, in[u], chunk, half, interleaved, angles, weights, y);
        else
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
        else if constexpr (kTurn)
          turned8<DT, D, double>(p.turn, true, in[u], chunk, half, interleaved, angles, weights, y);
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
        if constexpr (kTurn) {
          if (is_v)
            rotated8<DT, float>(in[u], chunk, 0, interleaved, angles, y);
          else
            turned8<DT, D, float>(p.turn, true, in[u], chunk, half, interleaved, angles, weights, y);
        } else {
          rotated8<DT, float>(in[u], chunk, is_v ? 0 : half, interleaved, angles, y);
        }
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

}  // namespace

}  // namespace fa2
