// serve_common.hpp - device helpers of the serving kernels: which sequence a packed row belongs to,
// where a token lies in the cache, and the conversion between 16-bit rows and e4m3 rows.
#pragma once

#include "attn_fwd_common.hpp"
#include "serve_params.hpp"

namespace fa2 {

template <int DT>
__device__ __forceinline__ float to_f32(uint16_t x) {
  if constexpr (DT == 0) return (float)__builtin_bit_cast(_Float16, x);
  return __uint_as_float((uint32_t)x << 16);
}

// cu[i], held to [0, n_tokens]: no row outside the tensors is ever addressed, whatever cu holds.
__device__ __forceinline__ int row_bound(const int32_t* cu, int i, int n_tokens) {
  return min(max(cu[i], 0), n_tokens);
}

// The largest s in [0, n_seq) with cu[s] <= t, for ascending cu (some s in [0, n_seq) otherwise). All 64
// lanes of a wave ask for one t; each round tests 64 sequences at once, so a call of up to 64
// sequences waits for one load, up to 4096 for two.
__device__ __forceinline__ int find_sequence(const int32_t* cu, int n_seq, int t, int lane) {
  int lo = 0, n = n_seq;  // the answer lies in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int i = lane * step;
    const uint64_t below = __builtin_amdgcn_ballot_w64(i < n && cu[lo + (i < n ? i : 0)] <= t);
    const int c = max(__builtin_popcountll(below) - 1, 0);
    lo += c * step;
    n = min(step, n - c * step);
  }
  return lo;
}

// A packed row's position in its sequence and the page of the cache that holds it. pos < 0: the row belongs to no
// sequence, or its place is before the sequence's start (more rows than tokens). page < 0: past the table, or not a
// page of the cache.
struct Place {
  int pos;
  int page;
};

// The sequences and positions of rows t0 .. t0 + tokens - 1 (at most 64), a lane each, by one wave: the ends of 64
// sequences are loaded at once (past 64 sequences, of those from the first row's on, which is looked up) and
// compared with every row, and the lengths of all rows are loaded together: two loads in a row for a group of rows.
struct LanePlace {
  int seq, pos;  // pos < 0: none
};
__device__ __forceinline__ LanePlace find_positions(const Sequences& q, int t0, int tokens, int lane) {
  const int first = q.n_seq <= 64 ? 0 : find_sequence(q.cu, q.n_seq, t0, lane);
  const int end = first + lane < q.n_seq ? q.cu[first + lane + 1] : 0x7fffffff;
  int seq = first;
  for (int i = 0; i < tokens; ++i) {  // (scalar: a ballot per row)
    const uint64_t before = __builtin_amdgcn_ballot_w64(end <= t0 + i);
    int s = first + __builtin_popcountll(before);
    // 64 sequences that end before the row: it lies past them all
    if (s - first == 64 && q.n_seq > 64) s = find_sequence(q.cu, q.n_seq, t0 + i, lane);
    if (lane == i) seq = s;
  }
  LanePlace p = {seq, -1};
  const int t = t0 + lane;
  if (lane >= tokens || seq >= q.n_seq) return p;
  const int length = max(q.lens[seq], 0);
  const int upto = row_bound(q.cu, seq + 1, q.n_tokens);
  if (t < row_bound(q.cu, seq, q.n_tokens) || t >= upto) return p;
  const int64_t pos = (int64_t)length - (upto - t);
  if (pos >= 0) p.pos = (int)pos;
  return p;
}
// The page of a lane's position, as Place's
__device__ __forceinline__ int find_page(const Sequences& q, const LanePlace& p) {
  const int slot = p.pos >> q.page_shift;
  if (p.pos < 0 || slot >= q.max_pages) return -1;
  const int page = q.table[p.seq * q.table_stride + slot];
  return (unsigned)page < (unsigned)q.n_pages ? page : -1;
}

// load_lds16 (attn_fwd_common.hpp) behind five wait states. A vector instruction may have written the
// resource's SGPRs right before (a readfirstlane, or the reload of a spilled SGPR), and a scalar one M0; the
// hardware needs 5 and 1 wait states before a buffer load reads them, and the compiler, which inserts
// those before its own loads, does not look into inline asm. Without them a load of a tile in several pages
// ran with the resource of the load before it.
__device__ __forceinline__ void load_lds16_settled(u32x4 desc, uint32_t voffset, uint32_t lds_base) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(voffset), "s"(desc), "{m0}"(lds_base)
               : "memory");
}

// A buffer resource over [data, data + bytes) (wave-uniform), and loads through it: past it they give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const char* data, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(data);
  auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
  const uint64_t base = (uint64_t)uniform((uint32_t)(a >> 32)) << 32 | uniform((uint32_t)a);
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base), 0, (int)uniform(bytes), 0x00020000);
}
__device__ __forceinline__ u32x4 load_buffer16(__amdgpu_buffer_rsrc_t rsrc, uint32_t offset) {
  return __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)offset, 0, 0);
}
__device__ __forceinline__ uint32_t load_buffer1(__amdgpu_buffer_rsrc_t rsrc, uint32_t offset) {
  return __builtin_amdgcn_raw_buffer_load_b8(rsrc, (int)offset, 0, 0);
}

// 2^(byte - 127) of an e8m0 scale byte (255: NaN)
__device__ __forceinline__ float e8m0_to_f32(uint32_t b) {
  return __uint_as_float(b == 0 ? 0x00400000u : b == 255u ? 0x7fc00000u : b << 23);
}

// 4 e4m3 values of a word times 2^(byte - 127), rounded to the 16-bit type (exactly, but where the product
// leaves the type's range): two packed pairs. The instruction takes its scale from a float's exponent bits.
template <int DT>
__device__ __forceinline__ u32x2 e4m3_to_16(uint32_t w, uint32_t scale_byte) {
  const float scale = __uint_as_float(scale_byte << 23);
  if constexpr (DT == 0)
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true))};
  else
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))};
}

}  // namespace fa2
