// serve_step_host.hpp - host side of the entry points of include/fa2_fwd.h that serve a step beyond serve_host.hpp's:
// windows and common prefixes in attention, normalised rotations of several axes, a step's pages. Included by fa2_fwd.hip
// after serve_host.hpp, whose checks it shares; everything here has internal linkage.
#pragma once

#include "serve_host.hpp"

namespace {

int check_turn(const fa2_turn* turn, int32_t head_dim, const void* positions, int32_t position_bytes, const int64_t* p_stride,
               int n_strides, fa2::RotaryPlan* rot, fa2::TurnParams* out) {
  *out = fa2::TurnParams{};
  if (!turn) return fail(FA2_EINVAL, "null turn");
  if (const int rc = check_rotation(&turn->rotation, head_dim, rot)) return rc;
  if (turn->n_axes < 1 || (!turn->axes && turn->n_axes != 1))
    return fail(FA2_EINVAL, "n_axes must be at least 1, and 1 without axes, got %d", turn->n_axes);
  if (reinterpret_cast<uintptr_t>(turn->axes) & 3u) return fail(FA2_EALIGN, "axes must be 4-byte aligned");
  for (const float* w : {turn->q_weight, turn->k_weight})
    if (reinterpret_cast<uintptr_t>(w) & 3u) return fail(FA2_EALIGN, "a norm's weight must be 4-byte aligned");
  if ((turn->q_weight && !(turn->q_eps > 0 && std::isfinite(turn->q_eps))) ||
      (turn->k_weight && !(turn->k_eps > 0 && std::isfinite(turn->k_eps))))
    return fail(FA2_EINVAL, "a norm's eps must be positive and finite, got %g and %g", turn->q_eps, turn->k_eps);
  if (positions) {
    if (position_bytes != 4 && position_bytes != 8)
      return fail(FA2_EINVAL, "positions are int32 or int64, got %d bytes each", position_bytes);
    if (reinterpret_cast<uintptr_t>(positions) % (unsigned)position_bytes)
      return fail(FA2_EALIGN, "positions must be aligned to their size");
    if (!p_stride) return fail(FA2_EINVAL, "null stride array: positions");
  }
  out->axes = turn->axes;
  out->n_axes = turn->n_axes;
  out->positions64 = position_bytes == 8;
  out->positions = positions;
  if (positions) {
    out->spa = p_stride[0];
    out->spb = n_strides == 3 ? p_stride[1] : 0;
    out->spn = p_stride[n_strides - 1];
  }
  out->q_weight = turn->q_weight;
  out->k_weight = turn->k_weight;
  out->q_eps = turn->q_eps;
  out->k_eps = turn->k_eps;
  return FA2_OK;
}

// Workgroups that are left at least where rotary_qk gathers tokens, and angles a workgroup forms from which on it gathers no more. Measured on
// MI355X, 32 + 8 heads of 128, three axes: 2048 tokens, one / two / four a workgroup 17.1 / 14.3 / 16.1 us, 4096 27.1 / 22.5 / 20.8 (and 26.1 of
// eight); 16384, one / four / eight / sixteen 127 / 79.4 / 78.7 / 81.5. 16 + 4 heads of 64: 16384 tokens, one / eight / sixteen 47.1 / 23.1 /
// 22.2.
constexpr int64_t kTurnWgs = 1024, kTurnAngles = 512;

// The keys that a row sees of n_kv at most, as the choice of a form counts them.
int64_t window_keys(int64_t n_kv, int32_t window, int32_t sinks) { return std::min<int64_t>(n_kv, (int64_t)window + sinks + 128); }

int check_window(int32_t causal, int32_t window, int32_t sinks) {
  if (!causal) return fail(FA2_EINVAL, "a window needs the causal mask");
  if (window < 1 || sinks < 0) return fail(FA2_EINVAL, "window must be positive and sinks not negative, got %d and %d", window, sinks);
  return FA2_OK;
}

// The form of attention behind a common prefix: 128-row workgroups for the prefix where the batch has more rows of a KV head than one
// wave takes, and for the keys behind it by the rows of a sequence, as ragged_plan chooses them; `shares` workgroups per
// head, which the kernel deals to the two. Workspace: every row's results of both, then the pieces of cut row tiles.
struct SharedPlan {
  int prefix_waves = 4, own_waves = 4, shares = 0;
  size_t rows = 0, workspace = 0;
};
SharedPlan shared_plan(int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t n_tokens, int32_t n_seq, int cus) {
  SharedPlan pl;
  const int64_t rows = (int64_t)n_tokens * (h_q / h_kv);
  pl.prefix_waves = rows <= 32 ? 1 : 4;
  pl.own_waves = rows <= (int64_t)32 * n_seq ? 1 : 4;
  pl.shares = std::max(2, fa2::kSharedWaves * cus / h_kv);
  const size_t row = (size_t)(head_dim + 4) * sizeof(float);
  pl.rows = (2 * (size_t)n_tokens * h_q * row + 255) & ~(size_t)255;
  pl.workspace = pl.rows + (size_t)h_kv * pl.shares * 2 * 32 * pl.prefix_waves * row;
  return pl;
}

// Every workgroup of the pages' kernels goes through the lengths, or counts, of all sequences before its own, 256 or 64 at a time.
constexpr int32_t kMostStepSequences = 1 << 20;
int check_step_sequences(int32_t n_seq) {
  if (n_seq > kMostStepSequences) return fail(FA2_EINVAL, "at most 2^20 sequences, got %d", n_seq);
  return FA2_OK;
}

}  // namespace

extern "C" {

int fa2_rotary_qk(const void* q, const void* k, void* q_out, void* k_out, const int64_t q_stride[3], const int64_t k_stride[3],
                  const int64_t qo_stride[3], const int64_t ko_stride[3], const void* positions, int32_t position_bytes,
                  const int64_t p_stride[3], const fa2_turn* turn, int32_t batch, int32_t h_q, int32_t h_k, int32_t n,
                  int32_t head_dim, int32_t dtype, void* stream) {
  g_err[0] = '\0';
  fa2::RotaryQkParams p{};
  if (const int rc = check_type(head_dim, dtype)) return rc;
  if (!positions) return fail(FA2_EINVAL, "null pointer: positions");
  if (const int rc = check_turn(turn, head_dim, positions, position_bytes, p_stride, 3, &p.rot, &p.turn)) return rc;
  if (batch < 0 || h_q < 0 || h_k < 0 || n < 0)
    return fail(FA2_EINVAL, "bad sizes: batch=%d h_q=%d h_k=%d n=%d", batch, h_q, h_k, n);
  if (h_q > (1 << 18) || h_k > (1 << 18)) return fail(FA2_EINVAL, "at most 2^18 heads");  // (passes are the grid's second dimension)
  if (batch == 0 || n == 0 || h_q + h_k == 0) return FA2_OK;
  if (h_q) {
    if (const int rc = check_rows("q", q, q_stride, 3, 8)) return rc;
    if (const int rc = check_rows("q_out", q_out, qo_stride, 3, 8)) return rc;
    if (const int rc = check_written("q_out", {{batch, qo_stride[0]}, {h_q, qo_stride[1]}, {n, qo_stride[2]}})) return rc;
    p.q = static_cast<const uint16_t*>(q);
    p.q_out = static_cast<uint16_t*>(q_out);
    p.sqb = q_stride[0]; p.sqh = q_stride[1]; p.sqn = q_stride[2];
    p.sqob = qo_stride[0]; p.sqoh = qo_stride[1]; p.sqon = qo_stride[2];
  }
  if (h_k) {
    if (const int rc = check_rows("k", k, k_stride, 3, 8)) return rc;
    if (const int rc = check_rows("k_out", k_out, ko_stride, 3, 8)) return rc;
    if (const int rc = check_written("k_out", {{batch, ko_stride[0]}, {h_k, ko_stride[1]}, {n, ko_stride[2]}})) return rc;
    p.k = static_cast<const uint16_t*>(k);
    p.k_out = static_cast<uint16_t*>(k_out);
    p.skb = k_stride[0]; p.skh = k_stride[1]; p.skn = k_stride[2];
    p.skob = ko_stride[0]; p.skoh = ko_stride[1]; p.skon = ko_stride[2];
  }
  p.batch = batch; p.h_q = h_q; p.h_k = h_k; p.n = n;
  // as many tokens as fill the lanes with rows, and, where workgroups are left for the CUs, with angles
  p.tokens_per_wg = fa2::serve_tokens_per_wg((int)std::min<int64_t>(((int64_t)h_q + h_k) * (head_dim / 8), 256), n, kRotaryWgs);
  while (p.tokens_per_wg < 16 && p.tokens_per_wg * p.rot.half < kTurnAngles && (int64_t)batch * n >= 2 * p.tokens_per_wg * kTurnWgs)
    p.tokens_per_wg *= 2;
  const int64_t grid = (int64_t)batch * (((int64_t)n + p.tokens_per_wg - 1) / p.tokens_per_wg);
  if (const int rc = check_grid(grid)) return rc;
  return launched(fa2::launch_rotary_qk(dtype, head_dim, p, (unsigned)grid, static_cast<hipStream_t>(stream)), "rotary");
}

int fa2_cache_write_turned(const fa2_cache* cache, const fa2_sequences* seq, const void* k, const void* v,
                           const int64_t k_stride[2], const int64_t v_stride[2], const void* q, void* q_out,
                           const int64_t q_stride[2], const int64_t qo_stride[2], int32_t h_q, const void* positions,
                           int32_t position_bytes, const int64_t p_stride[2], const fa2_turn* turn, int32_t dtype,
                           void* stream) {
  g_err[0] = '\0';
  fa2::CacheTurnParams p{};
  if (const int rc = write_params(cache, seq, k, v, k_stride, v_stride, q, q_out, q_stride, qo_stride, h_q,
                                  turn ? &turn->rotation : nullptr, dtype, &p))
    return rc;
  if (const int rc = check_turn(turn, cache->head_dim, positions, position_bytes, p_stride, 2, &p.rot, &p.turn)) return rc;
  if (!positions && turn->n_axes != 1) return fail(FA2_EINVAL, "a rotation by %d axes needs positions", turn->n_axes);
  if (p.seq.n_seq == 0 || p.seq.n_tokens == 0) return FA2_OK;
  const int64_t grid = cache_grid(&p, 2 * (int64_t)p.h_kv + p.h_q, cache->head_dim, kWriteWgs);
  if (const int rc = check_grid(grid)) return rc;
  return launched(fa2::launch_cache_write_turn(dtype, cache->head_dim, cache->cache_dtype == FA2_DTYPE_E4M3, p, (unsigned)grid,
                                               static_cast<hipStream_t>(stream)),
                  "cache write");
}

int fa2_attn_packed_window(const void* q, const void* k, const void* v, void* out, const int64_t q_stride[2],
                           const int64_t k_stride[2], const int64_t v_stride[2], const int64_t o_stride[2],
                           const int32_t* cu, const int32_t* cu_kv, int32_t n_seq, int32_t n_tokens, int32_t kv_tokens,
                           int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t dtype, int32_t window, int32_t sinks,
                           float qk_scale, float* lse, void* stream) {
  g_err[0] = '\0';
  fa2::RaggedParams p{};
  if (const int rc = packed_params(q, k, v, out, q_stride, k_stride, v_stride, o_stride, cu, cu_kv, n_seq, n_tokens,
                                   kv_tokens, h_q, h_kv, head_dim, dtype, 1, qk_scale, lse, &p))
    return rc;
  if (const int rc = check_window(1, window, sinks)) return rc;
  if (n_seq == 0 || n_tokens == 0) return FA2_OK;
  p.window = window;
  p.sinks = sinks;
  const int64_t keys = std::min<int64_t>(kv_tokens, n_seq * window_keys(kv_tokens, window, sinks));
  return launch_ragged<fa2::kModeWindow>(dtype, head_dim, h_q, p, fa2::kSourcePacked, keys, nullptr, 0, stream);
}

int fa2_attn_paged_window(const void* q, void* out, const int64_t q_stride[2], const int64_t o_stride[2],
                          const fa2_cache* cache, const fa2_sequences* seq, int32_t h_q, int32_t dtype, int32_t window,
                          int32_t sinks, float qk_scale, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = '\0';
  fa2::RaggedParams p{};
  if (const int rc = paged_params(q, out, q_stride, o_stride, cache, seq, h_q, dtype, 1, qk_scale, lse, &p)) return rc;
  if (const int rc = check_window(1, window, sinks)) return rc;
  if (p.seq.n_seq == 0 || p.seq.n_tokens == 0) return FA2_OK;
  p.window = window;
  p.sinks = sinks;
  const int64_t keys = window_keys((int64_t)p.seq.max_pages << p.seq.page_shift, window, sinks);
  return launch_ragged<fa2::kModeWindow>(dtype, cache->head_dim, h_q, p, source_of(cache->cache_dtype), keys, workspace,
                                         workspace_bytes, stream);
}

size_t fa2_paged_window_workspace_bytes(int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t cache_dtype, int32_t n_tokens,
                                        int32_t n_seq, int64_t max_keys, int32_t window, int32_t sinks, int32_t num_cus) {
  if (window < 1 || sinks < 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv || dim_index(head_dim) < 0 || n_tokens <= 0 || n_seq <= 0 ||
      num_cus <= 0)
    return 0;
  return window_plan(source_of(cache_dtype), h_q, h_kv, head_dim, n_tokens, n_seq, window_keys(max_keys, window, sinks), num_cus)
      .workspace;
}

int fa2_attn_paged_shared(const void* q, void* out, const int64_t q_stride[2], const int64_t o_stride[2],
                          const fa2_cache* cache, const fa2_sequences* seq, const int32_t* shared, int32_t h_q, int32_t dtype,
                          int32_t causal, float qk_scale, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = '\0';
  fa2::RaggedParams p{};
  if (const int rc = paged_params(q, out, q_stride, o_stride, cache, seq, h_q, dtype, causal, qk_scale, lse, &p)) return rc;
  if (p.seq.n_seq == 0 || p.seq.n_tokens == 0) return FA2_OK;
  if (!shared) return fail(FA2_EINVAL, "null pointer: shared");
  if (reinterpret_cast<uintptr_t>(shared) & 3u) return fail(FA2_EALIGN, "shared must be 4-byte aligned");
  const int source = source_of(cache->cache_dtype);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const Topology topo = device_topology(stream_device(st));
  const SharedPlan pl = shared_plan(h_q, p.h_kv, cache->head_dim, p.seq.n_tokens, p.seq.n_seq, topo.cus);
  p.group = h_q / p.h_kv;
  const int64_t grid = (int64_t)p.h_kv * pl.shares;
  for (const auto& [wgs, threads] : {std::pair<int64_t, int>{grid, 256}, {fa2::shared_join_grid(p), 1024}})
    if (const int rc = check_grid(wgs, threads)) return rc;
  if (!workspace || workspace_bytes < pl.workspace)
    return fail(FA2_EINVAL, "the call needs a workspace of %zu bytes, got %zu", pl.workspace,
                workspace ? workspace_bytes : (size_t)0);
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return fail(FA2_EALIGN, "the workspace must be 256-byte aligned");
  p.shared = shared;
  p.xcd_shift = topo.xcd_shift;
  p.shares = pl.shares;
  p.rows = static_cast<float*>(workspace);
  p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.rows);
  p.part_rows = 32 * pl.prefix_waves;
  const unsigned g = (unsigned)grid;
  int e;
  switch (dtype * 4 + dim_index(cache->head_dim)) {
    case 0: e = fa2::launch_shared<0, 16>(p, source, pl.prefix_waves, pl.own_waves, g, st); break;
    case 1: e = fa2::launch_shared<0, 32>(p, source, pl.prefix_waves, pl.own_waves, g, st); break;
    case 2: e = fa2::launch_shared<0, 64>(p, source, pl.prefix_waves, pl.own_waves, g, st); break;
    case 3: e = fa2::launch_shared<0, 128>(p, source, pl.prefix_waves, pl.own_waves, g, st); break;
    case 4: e = fa2::launch_shared<1, 16>(p, source, pl.prefix_waves, pl.own_waves, g, st); break;
    case 5: e = fa2::launch_shared<1, 32>(p, source, pl.prefix_waves, pl.own_waves, g, st); break;
    case 6: e = fa2::launch_shared<1, 64>(p, source, pl.prefix_waves, pl.own_waves, g, st); break;
    default: e = fa2::launch_shared<1, 128>(p, source, pl.prefix_waves, pl.own_waves, g, st);
  }
  return launched(e, "attention");
}

size_t fa2_paged_shared_workspace_bytes(int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t n_tokens, int32_t n_seq,
                                        int32_t num_cus) {
  if (h_q <= 0 || h_kv <= 0 || h_q % h_kv || dim_index(head_dim) < 0 || n_tokens <= 0 || n_seq <= 0 || num_cus <= 0) return 0;
  return shared_plan(h_q, h_kv, head_dim, n_tokens, n_seq, num_cus).workspace;
}

int fa2_pages_extend(const int32_t* free_pages, int32_t n_pages, const int32_t* count, int32_t* count_out, int32_t* table,
                     int64_t table_stride, int32_t n_seq, int32_t max_pages, int32_t page_size, const int32_t* lens,
                     const int32_t* new_tokens, int32_t* lens_out, int32_t* cu_out, int32_t* positions, int64_t* slots,
                     int32_t n_tokens, void* stream) {
  g_err[0] = '\0';
  if (n_pages < 0 || n_seq < 1 || max_pages < 0 || n_tokens < 0 || table_stride < 0)
    return fail(FA2_EINVAL, "bad sizes: n_pages=%d n_seq=%d max_pages=%d n_tokens=%d table_stride=%lld", n_pages, n_seq,
                max_pages, n_tokens, (long long)table_stride);
  if (const int rc = check_step_sequences(n_seq)) return rc;
  if (!power_of_two(page_size) || page_size > (1 << 20))
    return fail(FA2_EINVAL, "page_size must be a power of two up to 2^20, got %d", page_size);
  if (!count || !count_out || !lens || !new_tokens || !lens_out || !cu_out || (n_pages > 0 && !free_pages) ||
      (max_pages > 0 && !table) || (n_tokens > 0 && (!positions || !slots)))
    return fail(FA2_EINVAL, "null pointer");
  for (const void* x : {(const void*)free_pages, (const void*)count, (const void*)count_out, (const void*)table,
                        (const void*)lens, (const void*)new_tokens, (const void*)lens_out, (const void*)cu_out,
                        (const void*)positions})
    if (reinterpret_cast<uintptr_t>(x) & 3u) return fail(FA2_EALIGN, "int32 arrays must be 4-byte aligned");
  if (reinterpret_cast<uintptr_t>(slots) & 7u) return fail(FA2_EALIGN, "slots must be 8-byte aligned");
  if (max_pages > 0)
    if (const int rc = check_written("the table", {{n_seq, table_stride}})) return rc;
  fa2::PagesParams p{};
  p.free_pages = free_pages; p.count = count; p.table = table; p.lens = lens; p.fresh = new_tokens;
  p.table_stride = table_stride;
  p.n_pages = n_pages; p.n_seq = n_seq; p.max_pages = max_pages; p.n_tokens = n_tokens;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.count_out = count_out; p.lens_out = lens_out; p.cu_out = cu_out; p.positions = positions; p.slots = slots;
  // 256 sequences a block, and stripes of about 1024 rows (entries are fewer than rows and sequences together)
  const unsigned blocks = (unsigned)(((int64_t)n_seq + 255) / 256);
  const unsigned stripes = (unsigned)std::min<int64_t>(((int64_t)n_tokens / blocks + 1023) / 1024 + (n_tokens == 0), 1024);
  return launched(fa2::launch_pages_extend(p, blocks, std::max(stripes, 1u), static_cast<hipStream_t>(stream)), "pages");
}

int fa2_pages_release(int32_t* free_pages, int32_t n_pages, const int32_t* count, int32_t* count_out, const int32_t* table,
                      int64_t table_stride, int32_t n_seq, int32_t max_pages, const int32_t* first, const int32_t* last,
                      int32_t* workspace, void* stream) {
  g_err[0] = '\0';
  if (n_pages < 0 || n_seq < 1 || max_pages < 0 || table_stride < 0)
    return fail(FA2_EINVAL, "bad sizes: n_pages=%d n_seq=%d max_pages=%d table_stride=%lld", n_pages, n_seq, max_pages,
                (long long)table_stride);
  if (const int rc = check_step_sequences(n_seq)) return rc;
  if (!count || !count_out || !first || !last || !workspace || (n_pages > 0 && !free_pages) || (max_pages > 0 && !table))
    return fail(FA2_EINVAL, "null pointer");
  for (const void* x : {(const void*)free_pages, (const void*)count, (const void*)count_out, (const void*)table,
                        (const void*)first, (const void*)last, (const void*)workspace})
    if (reinterpret_cast<uintptr_t>(x) & 3u) return fail(FA2_EALIGN, "int32 arrays must be 4-byte aligned");
  fa2::ReleaseParams p{};
  p.free_pages = free_pages; p.count = count; p.table = table; p.first = first; p.last = last;
  p.table_stride = table_stride;
  p.n_pages = n_pages; p.n_seq = n_seq; p.max_pages = max_pages;
  p.count_out = count_out;
  p.counts = workspace;
  return launched(fa2::launch_pages_release(p, static_cast<hipStream_t>(stream)), "pages");
}

}  // extern "C"
