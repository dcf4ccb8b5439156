// serve_host.hpp - host side of the serving entry points (include/fa2_fwd.h): argument checks, the grid and
// the launch. Included by fa2_fwd.hip after attn_fwd_host.hpp, whose error string and device topology it
// shares; everything here has internal linkage.
#pragma once

#include <initializer_list>
#include <utility>

#include "attn_fwd_host.hpp"
#include "serve_launch.hpp"

namespace {

bool power_of_two(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }

// Longest sequence and most rows: positions stay 32-bit in the kernels with two rounds of four 128-key tiles of
// headroom.
constexpr int32_t kMaxKeys = 0x7fffffff - 2048;

// `n` strides of a 16-bit tensor (or of e4m3 bytes: multiples of 16) and its pointer
int check_rows(const char* what, const void* p, const int64_t* stride, int n, int multiple) {
  if (!p) return fail(FA2_EINVAL, "null pointer: %s", what);
  if (!stride) return fail(FA2_EINVAL, "null stride array: %s", what);
  if (!aligned16(p)) return fail(FA2_EALIGN, "%s must be 16-byte aligned", what);
  for (int i = 0; i < n; ++i)
    if (stride[i] < 0 || stride[i] % multiple)
      return fail(FA2_EALIGN, "strides of %s must be non-negative multiples of %d elements (%lld)", what,
                  multiple, (long long)stride[i]);
  return FA2_OK;
}

// What is written has a place of its own for every row: no stride of zero over several
int check_written(const char* what, std::initializer_list<std::pair<int64_t, int64_t>> count_and_stride) {
  for (const auto& [count, stride] : count_and_stride)
    if (count > 1 && stride == 0) return fail(FA2_EINVAL, "%s is written: it cannot have a stride of 0", what);
  return FA2_OK;
}

int check_type(int32_t head_dim, int32_t dtype) {
  if (dim_index(head_dim) < 0)
    return fail(FA2_EINVAL, "head_dim must be a power of two in [16, 128], got %d", head_dim);
  if (dtype != FA2_DTYPE_F16 && dtype != FA2_DTYPE_BF16)
    return fail(FA2_EINVAL, "dtype must be FA2_DTYPE_F16 or FA2_DTYPE_BF16, got %d", dtype);
  return FA2_OK;
}

int check_rotation(const fa2_rotation* r, int32_t head_dim, fa2::RotaryPlan* out) {
  *out = fa2::RotaryPlan{nullptr, 0, 0, 1.0};
  if (!r) return FA2_OK;
  if (r->half < 8 || r->half % 8 || r->half > head_dim / 2)
    return fail(FA2_EINVAL, "a rotation covers 16, 32, ... up to head_dim (%d) values, got %lld", head_dim,
                2 * (long long)r->half);
  if (!r->freqs || (reinterpret_cast<uintptr_t>(r->freqs) & 7u))
    return fail(FA2_EALIGN, "the rotation's frequencies must be an 8-byte aligned float64 array");
  if (!std::isfinite(r->scale)) return fail(FA2_EINVAL, "the rotation's scale must be finite");
  *out = fa2::RotaryPlan{r->freqs, r->half, r->interleaved != 0, r->scale};
  return FA2_OK;
}

// The kernels count sequences in 32 bits, 64 at a time.
int check_sequences(int32_t n_seq) {
  if (n_seq > kMaxKeys) return fail(FA2_EINVAL, "n_seq must be at most %d", kMaxKeys);
  return FA2_OK;
}

// The cache and the sequences over it, checked, as the kernels take them.
int check_cache(const fa2_cache* c, const fa2_sequences* q, int32_t dtype, fa2::CacheTensor* kc,
                fa2::CacheTensor* vc, fa2::Sequences* seq) {
  if (!c || !q) return fail(FA2_EINVAL, "null cache or sequences");
  if (const int rc = check_type(c->head_dim, dtype)) return rc;
  const bool e4m3 = c->cache_dtype == FA2_DTYPE_E4M3;
  if (!e4m3 && c->cache_dtype != dtype)
    return fail(FA2_EINVAL, "a 16-bit cache must be of the rows' own type (%d), got %d", dtype, c->cache_dtype);
  if (c->n_pages < 1 || c->h_kv < 1)
    return fail(FA2_EINVAL, "bad sizes: n_pages=%d h_kv=%d", c->n_pages, c->h_kv);
  const int64_t page_bytes = (int64_t)c->page_size * c->head_dim * (e4m3 ? 1 : 2);
  if (!power_of_two(c->page_size) || c->page_size < 16 || c->page_size > (1 << 20) || page_bytes < 1024)
    return fail(FA2_EINVAL,
                "page_size must be a power of two in [16, 2^20] with at least 1024 bytes of a head's rows, got %d "
                "(%lld bytes)",
                c->page_size, (long long)page_bytes);
  const int multiple = e4m3 ? 16 : 8;
  if (const int rc = check_rows("the cache's k", c->k, c->k_stride, 3, multiple)) return rc;
  if (const int rc = check_rows("the cache's v", c->v, c->v_stride, 3, multiple)) return rc;
  if (c->k_stride[2] > kMaxRowStride || c->v_stride[2] > kMaxRowStride)
    return fail(FA2_EINVAL, "a cache's token stride above %lld elements is not supported", (long long)kMaxRowStride);
  // the kernels add a page's bytes and a token's in 32 bits to a 64-bit base
  const int64_t most = 0x7fffffffLL / (e4m3 ? 1 : 2);
  for (const int64_t* s : {c->k_stride, c->v_stride})
    if (s[0] > most || s[2] * c->page_size > most)
      return fail(FA2_EINVAL, "a cache's pages must lie, and extend, less than 2^31 bytes apart");
  if (e4m3) {
    if (!c->k_scale || !c->v_scale) return fail(FA2_EINVAL, "an e4m3 cache needs k_scale and v_scale");
    for (int i = 0; i < 3; ++i)
      if (c->k_scale_stride[i] < 0 || c->v_scale_stride[i] < 0)
        return fail(FA2_EINVAL, "strides of the cache's scales must not be negative");
    if (c->k_scale_stride[2] > kMaxRowStride || c->v_scale_stride[2] > kMaxRowStride)
      return fail(FA2_EINVAL, "a scale's token stride above %lld is not supported", (long long)kMaxRowStride);
    for (const int64_t* s : {c->k_scale_stride, c->v_scale_stride})
      if (s[0] > most || s[2] * c->page_size > most)
        return fail(FA2_EINVAL, "the scales of a cache's pages must lie, and extend, less than 2^31 bytes apart");
  }
  if (q->n_seq < 0 || q->n_tokens < 0 || q->max_pages < 0 || q->table_stride < 0)
    return fail(FA2_EINVAL, "bad sizes: n_seq=%d n_tokens=%d max_pages=%d table_stride=%lld", q->n_seq, q->n_tokens,
                q->max_pages, (long long)q->table_stride);
  if (q->n_tokens > kMaxKeys) return fail(FA2_EINVAL, "n_tokens must be at most %d", kMaxKeys);
  if (const int rc = check_sequences(q->n_seq)) return rc;
  if ((int64_t)q->max_pages * c->page_size > kMaxKeys)
    return fail(FA2_EINVAL, "max_pages * page_size must be at most %d (32-bit key positions), got %lld", kMaxKeys,
                (long long)q->max_pages * c->page_size);
  if (q->n_seq > 0 && q->n_tokens > 0 && (!q->cu || !q->lens || (q->max_pages > 0 && !q->table)))
    return fail(FA2_EINVAL, "null pointer: cu, lens or table");
  auto tensor = [](const void* p, const void* s, const int64_t* st, const int64_t* ss) {
    return fa2::CacheTensor{static_cast<char*>(const_cast<void*>(p)),
                            static_cast<uint8_t*>(const_cast<void*>(s)), st[0], st[1], st[2],
                            s ? ss[0] : 0, s ? ss[1] : 0, s ? ss[2] : 0};
  };
  *kc = tensor(c->k, e4m3 ? c->k_scale : nullptr, c->k_stride, c->k_scale_stride);
  *vc = tensor(c->v, e4m3 ? c->v_scale : nullptr, c->v_stride, c->v_scale_stride);
  int shift = 0;
  while ((1 << shift) < c->page_size) ++shift;
  *seq = fa2::Sequences{q->cu, q->lens, q->table, q->table_stride, q->n_seq, q->n_tokens, q->max_pages, c->n_pages, shift};
  return FA2_OK;
}

// A launch holds fewer than 2^32 threads. (So rows, and the kernels' counts of their groups, stay far inside 32 bits.)
int check_grid(int64_t wgs, int threads = 256) {
  if (wgs > 0xffffffffLL / threads) return fail(FA2_EINVAL, "a grid of %lld workgroups is too large", (long long)wgs);
  return FA2_OK;
}

int launched(int e, const char* what) {
  return e == hipSuccess ? FA2_OK : fail(FA2_ELAUNCH, "%s launch failed: %s", what, hipGetErrorString((hipError_t)e));
}

// Workgroups that the tokens of a call are gathered into at least, as a group of tokens shares the lookup of their places
// (three loads in a row). Measured on MI355X (kernel alone): a write of 5096 tokens of 28 + 2 x 4 heads of 64 in 5096, 2548 and
// 1274 workgroups 20.0, 16.8 and 16.4 us; a read of 57071 tokens of 2 x 8 e4m3 heads of 128 in 57071, 7134 and
// 3567 112, 73 and 81 us. The rotary kernel has no such lookup, and takes as few tokens as fill its lanes.
constexpr int64_t kWriteWgs = 1024, kReadWgs = 4096, kRotaryWgs = int64_t(1) << 40;
int64_t cache_grid(fa2::CacheParams* p, int64_t rows_per_token, int32_t head_dim, int64_t least_wgs) {
  p->tokens_per_wg = fa2::serve_tokens_per_wg((int)std::min<int64_t>(rows_per_token * (head_dim / 8), 256),
                                              p->seq.n_tokens, least_wgs);
  return ((int64_t)p->seq.n_tokens + p->tokens_per_wg - 1) / p->tokens_per_wg;
}

// The form of a ragged attention call (attn_ragged.hpp, ragged_work.hpp), from what the host knows of it: the
// rows, the sequences and a bound on their keys, not the lengths. Measured on MI355X, us:
//   * packed rows: 32-row workgroups up to two tiles a CU, of sequences long enough that four waves have keys to take in
//     turn. 16 heads of 64, one sequence, 32 and 128 rows: 120 keys 7.0 and 6.5, 250 7.3 and 8.2, 1000 (512
//     tiles) 12.1 and 18.1, 4000 (2000 tiles) 78 and 63; 4 x 250 of 32 / 8 heads of 128 (1024 tiles) 21.5 and 11.8.
//   * pages: 32-row workgroups for up to 32 rows a sequence on average. 16 sequences behind 4k, 32 / 8 heads of 128, rows a
//     sequence: 16 50 and 66, 32 55 and 69, 64 60 and 71 - but 24 steps beside a chunk of 700 rows (35 on average)
//     75 and 66, and beside one of 3500 153 and 117.
//   * shares, or a workgroup a row tile: a tile each above 8 a CU, as then they even out (4 prompts of 4000, 500 and 611),
//     and where no sequence can have more keys than a share saves: 4 prompts of 500 21 and 41, of 1000 46 and 71; of 2000 148 and 164; steps of 8
//     sequences of 300 10 and 17, of 1000 16 and 19, of 2000 24 and 23; uneven ones of up to 1000, 64 and 256 of
//     them, 33 and 33, 102 and 99.
constexpr int64_t kShortKeys = 1536;
struct RaggedPlan {
  int row_waves = 4;  // 32-row workgroups (1) or 128-row ones (4)
  bool mixed = false;  // (of a window) 128-row workgroups' shares, and a 32-row one for each sequence of few rows
  int shares = 0;     // workgroups per KV head that share its work; 0: one per row tile
  int64_t grid = 0;
  size_t parts = 0, workspace = 0;  // bytes of the partial results, and with what their merge needs to know
};
// keys: of packed rows, all of them; of pages, the most that a sequence can have
RaggedPlan ragged_plan(int source, int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t n_tokens, int32_t n_seq,
                       int64_t keys, int cus) {
  RaggedPlan pl;
  const bool paged = source != fa2::kSourcePacked;
  const int64_t rows = (int64_t)n_tokens * (h_q / h_kv);
  auto tiles = [&](int64_t block_m) { return (rows + (int64_t)n_seq * (block_m - 1)) / block_m; };  // at most
  if (paged)
    pl.row_waves = rows <= (int64_t)32 * n_seq ? 1 : 4;
  else
    pl.row_waves = tiles(32) * h_kv <= 2 * (int64_t)cus && keys >= (int64_t)192 * n_seq ? 1 : 4;
  const int64_t n = tiles(32 * pl.row_waves);
  if (paged && n * h_kv < 8 * (int64_t)cus && keys > kShortKeys) {
    pl.shares = std::max(1, fa2::ragged_waves(head_dim, source, pl.row_waves) * cus / h_kv);
    // (a multiple of 256)
    pl.parts = (size_t)h_kv * pl.shares * 2 * 32 * pl.row_waves * (head_dim + 4) * sizeof(float);
    pl.workspace = pl.parts + (size_t)h_kv * pl.shares * fa2::kMergeBytes;
  }
  pl.grid = (pl.shares ? pl.shares : n) * h_kv;
  return pl;
}
// ... of a window over pages: mixed where sequences of few rows stand beside chunks whose row tiles give every CU one at least.
// Measured on MI355X, window 2048, a chunk beside single tokens behind 6000, 128-row tiles alone and mixed, us: heads of 16, 32 / 8, a
// chunk of 1024 beside 24 51 and 40, of 2048 64 and 52, of 4096 beside 64 124 and 99; of 64, 28 / 4, of 2048 beside 24 71 and 60, of 3000
// 76 and 91; e4m3 of 128, 28 / 4, of 1024 beside 24 86 and 71, of 2048 115 and 94, of 4096 186 and 184, 32 / 8 220 and 184.
// 16-bit heads of 128, where a single token's workgroup takes longest, only where the few would take the row tiles past one round of the
// workgroups, which then share all of them and merge the pieces, while the chunk's alone are a tile a workgroup (ragged_work.hpp's
// whole_tiles), and where the few are no more than the CUs:
//   * so: 28 / 4 heads, a chunk of 2048 (112 tiles on 128 workgroups a head) beside 24 97 and 86, 40 105 and 104; 32 / 8, 2048 (64 on
//     64) beside 24 119 and 112.
//   * all of them in one round: 28 / 4, 1500 (82 tiles) beside 24 70 and 90; 32 / 8, 1200 (37) 70 and 111.
//   * the chunk past a round: 28 / 4, 2500 (136) beside 24 116 and 123, 4096 159 and 170; 32 / 8, 3000 (93) 151 and 181.
//   * more of the few: 28 / 4, 2048 beside 64 121 and 153, 100 144 and 192; 32 / 8 beside 40 134 and 153.
RaggedPlan window_plan(int source, int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t n_tokens, int32_t n_seq, int64_t keys,
                       int cus) {
  RaggedPlan pl = ragged_plan(source, h_q, h_kv, head_dim, n_tokens, n_seq, keys, cus);
  const int64_t tiles = (int64_t)n_tokens * (h_q / h_kv) / 128, shares = std::max(1, fa2::kSharedWaves * cus / h_kv);
  if (source == fa2::kSourcePacked || pl.row_waves == 1 || !pl.shares || n_seq == 1 || tiles * h_kv < cus) return pl;
  if (head_dim == 128 && source == fa2::kSourcePages) {
    const bool whole = tiles <= shares && (keys + fa2::kTileCost<128>) * (shares - tiles) <= fa2::kShareCost * shares;
    if (!whole || tiles + n_seq <= pl.shares || (int64_t)n_seq * h_kv > cus) return pl;
  }
  pl.mixed = true;
  pl.shares = (int)shares;
  pl.parts = (size_t)h_kv * pl.shares * 2 * 128 * (head_dim + 4) * sizeof(float);
  pl.workspace = pl.parts + (size_t)h_kv * pl.shares * fa2::kMergeBytes;
  pl.grid = ((int64_t)pl.shares + n_seq) * h_kv;
  return pl;
}

// The heads and scale of a ragged attention call.
int check_heads(int32_t h_q, int32_t h_kv, int32_t n_tokens, float qk_scale, const float* lse) {
  if (h_q <= 0 || h_kv <= 0) return fail(FA2_EINVAL, "bad sizes: h_q=%d h_kv=%d", h_q, h_kv);
  if (h_q % h_kv) return fail(FA2_EINVAL, "GQA needs H_q divisible by H_kv (%d %% %d)", h_q, h_kv);
  if (!(qk_scale > 0.f) || !std::isfinite(qk_scale))
    return fail(FA2_EINVAL, "qk_scale (sm_scale * log2 e) must be positive and finite, got %g", (double)qk_scale);
  if (reinterpret_cast<uintptr_t>(lse) & 3u) return fail(FA2_EALIGN, "lse must be 4-byte aligned");
  const int64_t rows = (int64_t)n_tokens * (h_q / h_kv);
  if (rows > kMaxKeys) return fail(FA2_EINVAL, "n_tokens * (h_q / h_kv) must be at most %d, got %lld", kMaxKeys, (long long)rows);
  return FA2_OK;
}

int source_of(int32_t cache_dtype) { return cache_dtype == FA2_DTYPE_E4M3 ? fa2::kSourceE4m3 : fa2::kSourcePages; }

// A call's arguments, checked, as the kernels take them.
int packed_params(const void* q, const void* k, const void* v, void* out, const int64_t q_stride[2],
                  const int64_t k_stride[2], const int64_t v_stride[2], const int64_t o_stride[2], const int32_t* cu,
                  const int32_t* cu_kv, int32_t n_seq, int32_t n_tokens, int32_t kv_tokens, int32_t h_q, int32_t h_kv,
                  int32_t head_dim, int32_t dtype, int32_t causal, float qk_scale, float* lse, fa2::RaggedParams* p) {
  if (const int rc = check_type(head_dim, dtype)) return rc;
  if (n_seq < 0 || n_tokens < 0 || kv_tokens < 0 || kv_tokens > kMaxKeys)
    return fail(FA2_EINVAL, "bad sizes: n_seq=%d n_tokens=%d kv_tokens=%d", n_seq, n_tokens, kv_tokens);
  if (const int rc = check_sequences(n_seq)) return rc;
  if (!cu_kv && kv_tokens != n_tokens)
    return fail(FA2_EINVAL, "k and v of %d rows for q of %d need their own cu_kv", kv_tokens, n_tokens);
  if (const int rc = check_heads(h_q, h_kv, n_tokens, qk_scale, lse)) return rc;
  if (n_seq == 0 || n_tokens == 0) return FA2_OK;  // (nothing to launch)
  if (!cu) return fail(FA2_EINVAL, "null pointer: cu");
  if (const int rc = check_rows("q", q, q_stride, 2, 8)) return rc;
  if (const int rc = check_rows("out", out, o_stride, 2, 8)) return rc;
  if (const int rc = check_written("out", {{n_tokens, o_stride[0]}, {h_q, o_stride[1]}})) return rc;
  if (kv_tokens > 0) {  // (tensors of no rows may have no memory, and nothing of them is read)
    if (const int rc = check_rows("k", k, k_stride, 2, 8)) return rc;
    if (const int rc = check_rows("v", v, v_stride, 2, 8)) return rc;
    if (k_stride[0] > kMaxRowStride || v_stride[0] > kMaxRowStride)
      return fail(FA2_EINVAL, "a k/v row stride above %lld elements is not supported", (long long)kMaxRowStride);
    p->kc.data = static_cast<char*>(const_cast<void*>(k));
    p->kc.token = k_stride[0]; p->kc.head = k_stride[1];
    p->vc.data = static_cast<char*>(const_cast<void*>(v));
    p->vc.token = v_stride[0]; p->vc.head = v_stride[1];
  }
  p->q = static_cast<const uint16_t*>(q);
  p->o = static_cast<uint16_t*>(out);
  p->lse = lse;
  p->sqt = q_stride[0]; p->sqh = q_stride[1];
  p->sot = o_stride[0]; p->soh = o_stride[1];
  p->seq.cu = cu;
  p->seq.n_seq = n_seq;
  p->seq.n_tokens = n_tokens;
  p->cu_kv = cu_kv ? cu_kv : cu;
  p->kv_tokens = kv_tokens;
  p->h_kv = h_kv;
  p->causal = causal != 0;
  p->qk_scale = qk_scale;
  return FA2_OK;
}
int paged_params(const void* q, void* out, const int64_t q_stride[2], const int64_t o_stride[2], const fa2_cache* cache,
                 const fa2_sequences* seq, int32_t h_q, int32_t dtype, int32_t causal, float qk_scale, float* lse,
                 fa2::RaggedParams* p) {
  if (const int rc = check_cache(cache, seq, dtype, &p->kc, &p->vc, &p->seq)) return rc;
  if (const int rc = check_heads(h_q, cache->h_kv, seq->n_tokens, qk_scale, lse)) return rc;
  if (p->seq.n_seq == 0 || p->seq.n_tokens == 0) return FA2_OK;  // (nothing to launch)
  if (const int rc = check_rows("q", q, q_stride, 2, 8)) return rc;
  if (const int rc = check_rows("out", out, o_stride, 2, 8)) return rc;
  if (const int rc = check_written("out", {{p->seq.n_tokens, o_stride[0]}, {h_q, o_stride[1]}})) return rc;
  p->q = static_cast<const uint16_t*>(q);
  p->o = static_cast<uint16_t*>(out);
  p->lse = lse;
  p->sqt = q_stride[0]; p->sqh = q_stride[1];
  p->sot = o_stride[0]; p->soh = o_stride[1];
  p->h_kv = cache->h_kv;
  p->causal = causal != 0;
  p->qk_scale = qk_scale;
  return FA2_OK;
}

template <int DT, int D, int MODE>
int launch_form(const fa2::RaggedParams& p, int source, const RaggedPlan& pl, unsigned grid, hipStream_t s) {
  if (MODE == fa2::kModeWindow && pl.mixed) return fa2::launch_window_mixed<DT, D>(p, source, grid, s);
  return fa2::launch_ragged<DT, D, MODE>(p, source, pl.row_waves, grid, s);
}

// Launches a checked call whose heads, tensors and sequences are in p. keys: see ragged_plan.
template <int MODE = fa2::kModeAll>
int launch_ragged(int32_t dtype, int32_t head_dim, int32_t h_q, fa2::RaggedParams& p, int source, int64_t keys, void* workspace,
                  size_t workspace_bytes, void* stream) {
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const Topology topo = device_topology(stream_device(s));
  const RaggedPlan pl = (MODE == fa2::kModeWindow ? window_plan : ragged_plan)(source, h_q, p.h_kv, head_dim, p.seq.n_tokens,
                                                                               p.seq.n_seq, keys, topo.cus);
  if (const int rc = check_grid(pl.grid)) return rc;
  if (pl.workspace) {
    if (!workspace || workspace_bytes < pl.workspace)
      return fail(FA2_EINVAL, "the call needs a workspace of %zu bytes, got %zu", pl.workspace,
                  workspace ? workspace_bytes : (size_t)0);
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return fail(FA2_EALIGN, "the workspace must be 256-byte aligned");
  }
  p.group = h_q / p.h_kv;
  p.xcd_shift = topo.xcd_shift;
  p.shares = pl.shares;
  p.per_share = pl.shares ? 1.0 / pl.shares : 0.0;
  p.parts = static_cast<float*>(workspace);
  p.merges = static_cast<char*>(workspace) + pl.parts;
  const unsigned g = (unsigned)pl.grid;
  int e;
  switch (dtype * 4 + dim_index(head_dim)) {
    case 0: e = launch_form<0, 16, MODE>(p, source, pl, g, s); break;
    case 1: e = launch_form<0, 32, MODE>(p, source, pl, g, s); break;
    case 2: e = launch_form<0, 64, MODE>(p, source, pl, g, s); break;
    case 3: e = launch_form<0, 128, MODE>(p, source, pl, g, s); break;
    case 4: e = launch_form<1, 16, MODE>(p, source, pl, g, s); break;
    case 5: e = launch_form<1, 32, MODE>(p, source, pl, g, s); break;
    case 6: e = launch_form<1, 64, MODE>(p, source, pl, g, s); break;
    default: e = launch_form<1, 128, MODE>(p, source, pl, g, s);
  }
  return launched(e, "attention");
}

int write_params(const fa2_cache* cache, const fa2_sequences* seq, const void* k, const void* v, const int64_t k_stride[2],
                 const int64_t v_stride[2], const void* q, void* q_out, const int64_t q_stride[2], const int64_t qo_stride[2],
                 int32_t h_q, const fa2_rotation* rotation, int32_t dtype, fa2::CacheParams* p) {
  if (const int rc = check_cache(cache, seq, dtype, &p->kc, &p->vc, &p->seq)) return rc;
  if (const int rc = check_rotation(rotation, cache->head_dim, &p->rot)) return rc;
  if (q && !rotation) return fail(FA2_EINVAL, "q is taken to be rotated: it needs a rotation");
  if (q && h_q < 1) return fail(FA2_EINVAL, "bad sizes: h_q=%d", h_q);
  if (cache->h_kv > (1 << 24) || h_q > (1 << 24)) return fail(FA2_EINVAL, "at most 2^24 heads");
  if (p->seq.n_seq == 0 || p->seq.n_tokens == 0) return FA2_OK;  // (nothing to launch)
  for (const int64_t* s : {cache->k_stride, cache->v_stride, p->kc.scale ? cache->k_scale_stride : cache->k_stride,
                           p->kc.scale ? cache->v_scale_stride : cache->v_stride})
    if (const int rc = check_written("the cache", {{cache->n_pages, s[0]}, {cache->h_kv, s[1]}, {cache->page_size, s[2]}}))
      return rc;
  if (const int rc = check_rows("k", k, k_stride, 2, 8)) return rc;
  if (const int rc = check_rows("v", v, v_stride, 2, 8)) return rc;
  if (q) {
    if (const int rc = check_rows("q", q, q_stride, 2, 8)) return rc;
    if (const int rc = check_rows("q_out", q_out, qo_stride, 2, 8)) return rc;
    if (const int rc = check_written("q_out", {{p->seq.n_tokens, qo_stride[0]}, {h_q, qo_stride[1]}})) return rc;
    p->q = static_cast<const uint16_t*>(q);
    p->q_out = static_cast<uint16_t*>(q_out);
    p->sqt = q_stride[0]; p->sqh = q_stride[1];
    p->sot = qo_stride[0]; p->soh = qo_stride[1];
    p->h_q = h_q;
  }
  p->k = static_cast<uint16_t*>(const_cast<void*>(k));
  p->v = static_cast<uint16_t*>(const_cast<void*>(v));
  p->skt = k_stride[0]; p->skh = k_stride[1];
  p->svt = v_stride[0]; p->svh = v_stride[1];
  p->h_kv = cache->h_kv;
  return FA2_OK;
}

}  // namespace

extern "C" {

int fa2_rotary(const void* x, void* out, const int64_t x_stride[3], const int64_t o_stride[3],
               const void* positions, int32_t position_bytes, const int64_t p_stride[2],
               const fa2_rotation* rotation, int32_t batch, int32_t heads, int32_t n, int32_t head_dim,
               int32_t dtype, void* stream) {
  g_err[0] = '\0';
  fa2::RotaryParams p{};
  if (const int rc = check_type(head_dim, dtype)) return rc;
  if (!rotation) return fail(FA2_EINVAL, "null rotation");
  if (const int rc = check_rotation(rotation, head_dim, &p.rot)) return rc;
  if (batch < 0 || heads < 0 || n < 0) return fail(FA2_EINVAL, "bad sizes: batch=%d heads=%d n=%d", batch, heads, n);
  if (position_bytes != 4 && position_bytes != 8)
    return fail(FA2_EINVAL, "positions are int32 or int64, got %d bytes each", position_bytes);
  if (batch == 0 || heads == 0 || n == 0) return FA2_OK;
  if (const int rc = check_rows("x", x, x_stride, 3, 8)) return rc;
  if (const int rc = check_rows("out", out, o_stride, 3, 8)) return rc;
  if (const int rc = check_written("out", {{batch, o_stride[0]}, {heads, o_stride[1]}, {n, o_stride[2]}})) return rc;
  if (!positions || !p_stride) return fail(FA2_EINVAL, "null pointer: positions");
  if (reinterpret_cast<uintptr_t>(positions) % (unsigned)position_bytes)
    return fail(FA2_EALIGN, "positions must be aligned to their size");
  p.x = static_cast<const uint16_t*>(x);
  p.out = static_cast<uint16_t*>(out);
  p.sxb = x_stride[0]; p.sxh = x_stride[1]; p.sxn = x_stride[2];
  p.sob = o_stride[0]; p.soh = o_stride[1]; p.son = o_stride[2];
  p.positions = positions;
  p.positions64 = position_bytes == 8;
  p.spb = p_stride[0]; p.spn = p_stride[1];
  p.batch = batch; p.heads = heads; p.n = n;
  if (heads > (1 << 24)) return fail(FA2_EINVAL, "at most 2^24 heads, got %d", heads);
  p.tokens_per_wg = fa2::serve_tokens_per_wg((int)std::min<int64_t>((int64_t)heads * (head_dim / 8), 256),
                                             (int64_t)batch * n, kRotaryWgs);
  const int64_t grid = ((int64_t)batch * n + p.tokens_per_wg - 1) / p.tokens_per_wg;
  if (const int rc = check_grid(grid)) return rc;
  return launched(fa2::launch_rotary(dtype, head_dim, p, (unsigned)grid, static_cast<hipStream_t>(stream)), "rotary");
}

int fa2_cache_write(const fa2_cache* cache, const fa2_sequences* seq, const void* k, const void* v,
                    const int64_t k_stride[2], const int64_t v_stride[2], const void* q, void* q_out,
                    const int64_t q_stride[2], const int64_t qo_stride[2], int32_t h_q,
                    const fa2_rotation* rotation, int32_t dtype, void* stream) {
  g_err[0] = '\0';
  fa2::CacheParams p{};
  if (const int rc = write_params(cache, seq, k, v, k_stride, v_stride, q, q_out, q_stride, qo_stride, h_q, rotation, dtype, &p))
    return rc;
  if (p.seq.n_seq == 0 || p.seq.n_tokens == 0) return FA2_OK;
  const int64_t grid = cache_grid(&p, 2 * (int64_t)p.h_kv + p.h_q, cache->head_dim, kWriteWgs);
  if (const int rc = check_grid(grid)) return rc;
  return launched(fa2::launch_cache(true, dtype, cache->head_dim, cache->cache_dtype == FA2_DTYPE_E4M3, p, (unsigned)grid,
                                    static_cast<hipStream_t>(stream)),
                  "cache write");
}

int fa2_cache_read(const fa2_cache* cache, const fa2_sequences* seq, void* k, void* v, const int64_t k_stride[2],
                   const int64_t v_stride[2], int32_t dtype, void* stream) {
  g_err[0] = '\0';
  fa2::CacheParams p{};
  if (const int rc = check_cache(cache, seq, dtype, &p.kc, &p.vc, &p.seq)) return rc;
  if (cache->h_kv > (1 << 24)) return fail(FA2_EINVAL, "at most 2^24 heads");
  if (p.seq.n_seq == 0 || p.seq.n_tokens == 0) return FA2_OK;
  if (const int rc = check_rows("k", k, k_stride, 2, 8)) return rc;
  if (const int rc = check_rows("v", v, v_stride, 2, 8)) return rc;
  for (const int64_t* s : {k_stride, v_stride})
    if (const int rc = check_written("k and v", {{p.seq.n_tokens, s[0]}, {cache->h_kv, s[1]}})) return rc;
  p.k = static_cast<uint16_t*>(k);
  p.v = static_cast<uint16_t*>(v);
  p.skt = k_stride[0]; p.skh = k_stride[1];
  p.svt = v_stride[0]; p.svh = v_stride[1];
  p.h_kv = cache->h_kv;
  const int64_t grid = cache_grid(&p, 2 * (int64_t)p.h_kv, cache->head_dim, kReadWgs);
  if (const int rc = check_grid(grid)) return rc;
  return launched(fa2::launch_cache(false, dtype, cache->head_dim, cache->cache_dtype == FA2_DTYPE_E4M3, p, (unsigned)grid,
                                    static_cast<hipStream_t>(stream)),
                  "cache read");
}

int fa2_attn_packed(const void* q, const void* k, const void* v, void* out, const int64_t q_stride[2],
                    const int64_t k_stride[2], const int64_t v_stride[2], const int64_t o_stride[2],
                    const int32_t* cu, const int32_t* cu_kv, int32_t n_seq, int32_t n_tokens, int32_t kv_tokens,
                    int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t dtype, int32_t causal, float qk_scale,
                    float* lse, void* stream) {
  g_err[0] = '\0';
  fa2::RaggedParams p{};
  if (const int rc = packed_params(q, k, v, out, q_stride, k_stride, v_stride, o_stride, cu, cu_kv, n_seq, n_tokens,
                                   kv_tokens, h_q, h_kv, head_dim, dtype, causal, qk_scale, lse, &p))
    return rc;
  if (n_seq == 0 || n_tokens == 0) return FA2_OK;
  return launch_ragged(dtype, head_dim, h_q, p, fa2::kSourcePacked, kv_tokens, nullptr, 0, stream);
}

int fa2_attn_paged(const void* q, void* out, const int64_t q_stride[2], const int64_t o_stride[2],
                   const fa2_cache* cache, const fa2_sequences* seq, int32_t h_q, int32_t dtype, int32_t causal,
                   float qk_scale, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = '\0';
  fa2::RaggedParams p{};
  if (const int rc = paged_params(q, out, q_stride, o_stride, cache, seq, h_q, dtype, causal, qk_scale, lse, &p)) return rc;
  if (p.seq.n_seq == 0 || p.seq.n_tokens == 0) return FA2_OK;
  return launch_ragged(dtype, cache->head_dim, h_q, p, source_of(cache->cache_dtype),
                       (int64_t)p.seq.max_pages << p.seq.page_shift, workspace, workspace_bytes, stream);
}

size_t fa2_paged_workspace_bytes(int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t cache_dtype, int32_t n_tokens,
                                 int32_t n_seq, int64_t max_keys, int32_t num_cus) {
  const int source = source_of(cache_dtype);
  if (h_q <= 0 || h_kv <= 0 || h_q % h_kv || dim_index(head_dim) < 0 || n_tokens <= 0 || n_seq <= 0 || num_cus <= 0) return 0;
  return ragged_plan(source, h_q, h_kv, head_dim, n_tokens, n_seq, max_keys, num_cus).workspace;
}

}  // extern "C"
