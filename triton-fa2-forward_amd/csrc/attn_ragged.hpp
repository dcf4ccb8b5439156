// attn_ragged.hpp - attention of packed rows: sequences of different lengths back to back, with K and V
// in packed rows as well (source 0), in pages of 16-bit elements (1) or in pages of e4m3 (2).
//
//   O[r] = sum_n softmax_n(q_r . k_n * sm_scale) v_n over the keys n <= last(r) of the row's sequence,
//   last(r) = n_kv - 1, or with the causal mask n_kv - n_q + (the row's position): the last row sees the
//   last key. Of a window, n > last(r) - window or n < sinks: the key tiles between the sinks' and the window's are left
//   out of the count of tiles. A row that sees no key gets O = 0 and a log-sum-exp of -inf.
//
// All query heads of a KV head share a workgroup's rows: row r of a sequence is position r / group, head
// r % group. Which rows and keys a workgroup takes: ragged_work.hpp.
//
// The tile arithmetic is attn_fwd_kernel.hpp's: S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_32x32x16, P
// in registers, online softmax in base 2 with a lazily moved reference. Two forms:
//   * GW = 4: 128 rows, 32 a wave, which walk tiles of 64 keys together (attn_fwd_kernel.hpp's one-tile
//     loop: one barrier per tile, K two tiles and V one tile ahead). For prompts and chunks of them.
//   * GW = 1: 32 rows, whose key tiles the four waves take in turn, each through LDS buffers of its own without
//     a barrier, and merge once in LDS (attn_fwd_wavesplit.hpp). For single tokens and small grids.
// K and V rows of 16 bits go from HBM to LDS directly; the rows of one load instruction lie in one page (the
// host's rule on page sizes), so a load has one scalar resource, and the pages of the next 64 loads' worth of tiles
// sit in a register, a lane each. e4m3 rows go through registers, converted to the 16-bit type on
// their way into LDS (once per workgroup or wave, not once per operand read): from there on the sources are alike.
//
// What bounds it, and what it measured on MI355X (kernel alone, its merge apart):
//   * prompts: the instructions of a tile, one wave's products beside another's softmax. 8 packed sequences of up to 2048,
//     32 / 8 heads of 128, bf16 causal: 114 us, 850 TFLOP/s, matrix cores 40% busy, 7.5 vector instructions a
//     product; 4 of up to 8192, 16 heads of 64, fp16, with the log-sum-exp: 232 us, 790 TFLOP/s, 12.9.
//   * chunks: the same, at 2 workgroups a CU by their registers, which e4m3 at head_dim 128 does not get by with (18 or 19
//     spilled, 7 of them with 32 rows). 2 e4m3 chunks of up to 2048 behind 12k and 32k: 1218 us, 930 TFLOP/s, and 17 of merge.
//     One of 500 beside 24 steps of up to 8k: 88 us and 12 of merge.
//   * windows: the same, and the tiles at both ends, of which a row tile sees parts: 4 packed prompts of up to 8192, window 1024 and 4 sinks, 32 / 8
//     heads of 128, bf16, with the log-sum-exp: 267 to 294 us (the least and the median of 60 in a row, up to 357 as the clock gives), 745 to
//     820 TFLOP/s of the pairs that are seen, matrix cores 42% busy.
//   * steps: reading K and V. 16 of up to 4095 tokens, 32 / 8 heads of 128, bf16, pages of 16: 28 us, 4.7 TB/s, and 4.5 of
//     merge; 64 of up to 16000, e4m3: 198 us, 5.3 TB/s.
// Tried and dropped: writing e4m3's converted pairs in an order without bank conflicts (10% of the cycles have one; the
// selects cost more: 1060 -> 1105 us); sequences of few rows as a line of shares apart (114 -> 122 us), and weighted
// 1/2 or 2 in the one line (121 -> 140, 125).
#pragma once

#include <type_traits>

#include "attn_fwd_wavesplit.hpp"
#include "ragged_work.hpp"

namespace fa2 {

// Keys per tile
constexpr int ragged_block_n(int head_dim, int row_waves) {
  return row_waves == 4 ? (head_dim == 16 ? 128 : 64) : head_dim == 128 ? 32 : 64;
}

// A row's results over a common prefix, or over its own keys behind it: O, then m, l, exact l and a word that says more: bit 1, the row
// sees no key; bit 0, they lie in pieces, and the words before it are the first and the last of the shares that have
// one, and the row's place there.
template <int D, int MODE>
__device__ __forceinline__ float* row_results(ParamsRef p, int64_t token, int head) {
  const int64_t h_q = p.h_kv * p.group;
  return p.rows + ((MODE == kModeOwn ? p.seq.n_tokens * h_q : 0) + token * h_q + head) * (D + 4);
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A workgroup's LDS: K and V, and where four waves take a row's keys in turn, what they merge
template <int D, int GW>
struct RaggedLds {
  u32x4 kv[2 * 2 * ragged_block_n(D, 4) * (D / 8)];
};
template <int D>
struct RaggedLds<D, 1> {
  static constexpr int kKvChunks = 4 * 2 * ragged_block_n(D, 1) * (D / 8), kMergeChunks = 32 * 4 * (D / 4);
  u32x4 kv[kKvChunks > kMergeChunks ? kKvChunks : kMergeChunks];
  float sm[4][32][3];  // m, l, exact l of every group's rows
  int odd[32];         // rows whose sums are not finite
};

// LSE: with 128 rows, whether p.lse is set: known to the compiler, the sums it needs mix with the rest of the tile's
// instructions, and cost nothing where they are not asked for.
template <int DT, int D, int SRC, int GW, bool LSE, int MODE>
__device__ __forceinline__ void ragged_rows(RaggedLds<D, GW>& mem, int hkv, int rank, Cursor cur) {
  using E = Elem<DT>;
  ParamsRef p = params_here();
  constexpr bool kE4m3 = SRC == kSourceE4m3;
  constexpr bool kPages = SRC != kSourcePacked;
  constexpr bool kWindow = MODE == kModeWindow, kPrefix = MODE == kModePrefix, kOwn = MODE == kModeOwn;
  constexpr bool kJoined = kPrefix || kOwn;  // results are kept in float, for attn_shared_join_kernel
  constexpr int EB = kE4m3 ? 1 : 2;      // bytes of a cached element
  constexpr int BN = ragged_block_n(D, GW);
  constexpr int BM = 32 * GW;            // rows per workgroup
  constexpr int KG = 4 / GW;             // key groups of GW waves
  constexpr int BUFS = GW == 1 ? 1 : 2;  // K (and V) tiles in LDS per group
  constexpr int KS = D / 16;             // 16-dim k-steps of S^T = K Q^T
  constexpr int DB = (D + 31) / 32;      // 32-dim row blocks of O^T
  constexpr int NB = BN / 32;            // 32-key row blocks of S^T
  constexpr int NT = BN / 16;            // 16-key k-steps of O^T
  constexpr int CPR = D / 8;             // 16-byte chunks per K / V row in LDS
  constexpr int TCH = BN * CPR;          // chunks per K (or V) tile
  constexpr int NI = TCH / 64 * EB / 2;  // 1 KiB loads per tile
  constexpr int JW = (NI + GW - 1) / GW; // ... per wave
  constexpr int RPI = BN / NI;           // rows of one load
  // rows of a page at least (one load's rows lie in one page: the host's rule on page sizes), and the loads of them
  constexpr int SEG = RPI > 16 ? RPI : 16, LPS = SEG / RPI;
  constexpr int LPR = 64 / RPI;          // lanes per row of a load
  static_assert(NI >= 1 && BN % NI == 0, "a tile must be whole 1 KiB loads");
  constexpr int QPR = D / 4;             // 16-byte pieces of an fp32 output row

  auto& lds = mem.kv;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int c = lane & 31;
  const int g = lane >> 5;
  const int grp = wave / GW, gwave = wave % GW;

  // ---- LDS operand reads, as in attn_fwd_kernel.hpp
  const FA2_LDS char* gbuf = (const FA2_LDS char*)(lds + grp * BUFS * 2 * TCH);
  auto kbuf = [&](int i) { return gbuf + (BUFS == 1 ? 0 : (i & 1) * TCH * 16); };
  auto vbuf = [&](int i) { return kbuf(i) + BUFS * TCH * 16; };
  const int kk = k_key<D>(c & 15);
  const int vj = (lane & 15) >> 2;
  const int vq = lane & 3;
  const int vsig = ((vq & 1) << 1) | ((vq & 2) >> 1);
  const int vdh = (D == 16) ? 0 : ((lane >> 4) & 1);
  uint32_t koffs[KS], voffs[2][DB];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koffs[ks] = (uint32_t)((pi_row(c) * CPR + ((2 * ks + g) ^ kk)) * 16);
  if constexpr (GW > 1) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(koffs[ks]));  // (kept whole: attn_fwd_kernel.hpp)
  }
#pragma unroll
  for (int rr = 0; rr < 2; ++rr)
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int row = 8 * g + 4 * rr + vj;
      const int chunk = (4 * db + 2 * vdh + (vsig >> 1)) ^ v_key<D>(row);
      voffs[rr][db] = (uint32_t)(row * (D * 2) + chunk * 16 + (vsig & 1) * 8);
    }
  auto k_operand = [&](int i, int ks, int nb) {
    return *(const u32x4 FA2_LDS*)(kbuf(i) + koffs[ks] + nb * 32 * CPR * 16);
  };
  auto v_operand = [&](int i, int t, int db) {
    const u32x2 lo = lds_read_tr(vbuf(i) + voffs[0][db] + t * 16 * D * 2);
    const u32x2 hi = lds_read_tr(vbuf(i) + voffs[1][db] + t * 16 * D * 2);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };

  // ---- this head's K and V: where they start, the bytes between pages and between tokens (below 2^31: the
  // host's limits), and this lane's offset from a segment's first row in load u of the segment
  const int page_shift = p.seq.page_shift;
  struct Source {
    const char* data;
    uint32_t page, token;
  };
  const Source ks = {p.kc.data + hkv * p.kc.head * EB, (uint32_t)p.kc.page * EB, (uint32_t)p.kc.token * EB};
  const Source vs = {p.vc.data + hkv * p.vc.head * EB, (uint32_t)p.vc.page * EB, (uint32_t)p.vc.token * EB};
  const Source kscale = {(const char*)p.kc.scale + hkv * p.kc.scale_head, (uint32_t)p.kc.scale_page, (uint32_t)p.kc.scale_token};
  const Source vscale = {(const char*)p.vc.scale + hkv * p.vc.scale_head, (uint32_t)p.vc.scale_page, (uint32_t)p.vc.scale_token};
  uint32_t koff[LPS], voff[LPS], kscale_off[LPS], vscale_off[LPS];
#pragma unroll
  for (int u = 0; u < LPS; ++u) {
    const int row = u * RPI + lane / LPR, x = lane % LPR;  // (the swizzle keys repeat every 16 rows)
    if constexpr (kE4m3) {
      koff[u] = (uint32_t)row * ks.token + x * 16;
      voff[u] = (uint32_t)row * vs.token + x * 16;
      kscale_off[u] = (uint32_t)row * kscale.token;
      vscale_off[u] = (uint32_t)row * vscale.token;
    } else {
      koff[u] = (uint32_t)row * ks.token + (x ^ k_key<D>(pi_row(row & 31) & 15)) * 16;
      voff[u] = (uint32_t)row * vs.token + (x ^ v_key<D>(row & 15)) * 16;
    }
  }

  const float qk_scale = p.qk_scale;
  const bool want_exact = GW == 1 ? p.lse != nullptr : LSE, causal = !kPrefix && p.causal != 0,
             shared = kJoined || (kPages && p.shares > 0 && !cur.by_tile);

  // ---- the workgroup's work: the pieces of its share, or its one tile
  Share share = {0, 0, 0, 0};
  if (shared) {
    share = find_share<BM, kPages, MODE>(p, rank, lane, &cur);
    if (share.x >= share.end) {
      if constexpr (!kJoined) {
        if (tid == 0) merge_of(p, hkv, rank)->first = -1;
      }
      return;
    }
  } else if (!find_tile<BM, kPages, MODE>(p, rank, lane, &cur)) {
    return;
  }
  bool fresh = true;  // LDS has not been used yet
  for (bool first_piece = true, more = true; more; first_piece = false) {
    ParamsRef p = params_here();
    const LaneSequence sq = sequence_at(cur.lanes, cur.l);
    const int seq = kPrefix ? cur.prefix.row : cur.s0 + cur.l, n_kv = sq.n_kv;
    const int rows = sq.n_q * p.group;
    const int row0 = cur.tile * BM;       // this workgroup's rows [row0, row_end)
    const int row_end = min(row0 + BM, rows);
    const int shift = n_kv - sq.n_q;      // causal: position i sees keys up to i + shift
    // the last key of a position, the end of the keys that some row sees, and of those that every row sees
    auto last_of = [&](int i) { return causal ? min(i + shift, n_kv - 1) : n_kv - 1; };
    const int see_end = max(last_of((row_end - 1) / p.group) + 1, 0);
    const int full_end = max(last_of(row0 / p.group) + 1, 0);
    // A window: the first key of a position (beside the sinks), the least and the largest of the tile's, and the key
    // tiles between the sinks' and the window's, which are skipped. Key tiles are counted without those.
    // (compared first: a window up to 2^31 - 1 less a negative last key, of a row that sees none, is no int)
    auto first_of = [&](int i) { return kWindow && last_of(i) >= p.window ? last_of(i) - p.window + 1 : 0; };
    const int sinks = kWindow ? p.sinks : 0;
    const int see_begin = first_of(row0 / p.group), first_end = first_of((row_end - 1) / p.group);
    const int sink_tiles = kWindow ? (min(sinks, see_end) + BN - 1) / BN : 0;
    const int skip = kWindow ? max(see_begin / BN - sink_tiles, 0) : 0;
    auto tile_key = [&](int t) { return (kWindow && t >= sink_tiles ? t + skip : t) * BN; };
    const int all_tiles = (see_end + BN - 1) / BN - skip;

    int t_begin = 0, t_end = all_tiles;
    float* part = nullptr;  // where the piece's partial results go, if it is not the whole tile
    if (shared) {
      const int64_t length = lengths_of<BM, MODE>(p, sq.n_q, n_kv).of(cur.tile);
      const int64_t out = min(length, share.in + (share.end - share.x));
      if (share.in > 0) t_begin = cut_at(share.in, length, all_tiles);
      if (out < length) t_end = cut_at(out, length, all_tiles);
      // nothing between the cuts (a tile that sees no key at all belongs to the share that it starts in)
      const bool empty = all_tiles == 0 ? share.in > 0 : t_begin == t_end;
      const bool whole = t_begin == 0 && t_end == all_tiles;
      if constexpr (kJoined) {
        if (!whole) part = joined_part<D>(p, hkv, cur.first_share + rank, share.in == 0);
        if (!whole && !empty && t_begin == 0 && tid < row_end - row0) {  // the first piece says where they all are
          const int64_t start = share.x - share.in;
          const int i = (row0 + tid) / p.group, head = hkv * p.group + (row0 + tid - i * p.group);
          *(i32x4*)(row_results<D, MODE>(p, sq.first + i, head) + D) =
              i32x4{cur.first_share + (int)(start / share.size), cur.first_share + (int)((start + length - 1) / share.size), tid,
                    1 + (last_of(i) < 0 ? 2 : 0)};
        }
      } else if (!whole) {
        part = part_of<BM, D>(p, hkv, rank, share.in == 0);
      }
      if (!kJoined && first_piece && tid == 0) {  // what the merge of a tile that ends here needs to know
        Merge m = {-1, row0, row_end - row0, sq.first, n_kv, shift};
        if (!empty && !whole && t_end == all_tiles) m.first = (int)((share.x - share.in) / share.size);
        *merge_of(p, hkv, rank) = m;
      }
      const bool null_part = empty && !whole && tid < row_end - row0;
      share.x += out - share.in;
      share.in = 0;
      if (empty) {
        if (null_part) *(f32x4*)(part + part_sums<BM, D>(tid)) = f32x4{-INFINITY, 0.f, 0.f, 0.f};
        more = share.x < share.end && next_tile<BM, kPages, MODE>(p, lane, &cur);
        continue;
      }
    }
    const int kv_begin = tile_key(t_begin), kv_end = min(kWindow ? tile_key(t_end - 1) + BN : t_end * BN, see_end);
    if (!fresh) __syncthreads();  // the last piece's merge has left LDS
    fresh = false;

    // ---- this lane's row; rows past the last repeat it and are never stored
    const int wr = gwave * 32 + c;  // the row inside the workgroup
    const int r = min(row0 + wr, rows - 1);
    const int pos = r / p.group;
    const int last_key = last_of(pos), first_key = first_of(pos);
    u32x4 qreg[KS];
    {
      const int head = hkv * p.group + (r - pos * p.group);
      const uint16_t* qrow = p.q + (int64_t)(sq.first + pos) * p.sqt + head * p.sqh + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qreg[ks] = *(const u32x4*)(qrow + 16 * ks);
    }

    // ---- this group's key tiles: grp, grp + KG, ... of the piece
    const int n_tiles = t_end - t_begin;
    const int count = (n_tiles - grp + KG - 1) / KG;
    auto key_of = [&](int i) {  // first key of tile i
      if constexpr (kWindow) return tile_key(t_begin + grp + i * KG);
      return kv_begin + (grp + i * KG) * BN;
    };
    // whether no row sees any of `keys` keys from n on, those up to kv_end all being seen but for the window
    auto hidden = [&](int n, int keys) { return kWindow && n >= sinks && n + keys <= see_begin; };

    // ---- pages: lane x of `pages` holds the page of tile x / per_tile of the current block of 64 / per_tile
    // tiles, its page x % per_tile; `pages_next` those of the next block, on their way. An entry that
    // is no page of the cache reads page 0 and makes the rows NaN.
    constexpr int kLog2Bn = BN == 32 ? 5 : BN == 64 ? 6 : 7;
    const int tile_shift = kPages ? max(0, kLog2Bn - page_shift) : 0;  // log2 pages per tile
    const int block = 64 >> tile_shift;  // tiles of a block
    const int64_t first_token = kOwn ? sq.kv_first : 0;  // (whole pages)
    int pages = 0, pages_next = 0, bad = 0;
    auto load_pages = [&](int i0) {
      ParamsRef p = params_here();
      const int i = i0 + (lane >> tile_shift);
      int64_t n;
      if constexpr (kWindow)
        n = tile_key(t_begin + grp + min(i, count) * KG);
      else
        n = kv_begin + (int64_t)(grp + (int64_t)i * KG) * BN;
      n += (int64_t)(lane & ((1 << tile_shift) - 1)) << page_shift;
      int e = 0;
      // (a page that no row sees may be none of the cache any more: its entry is not looked at, and nothing of it loaded)
      if (i < count && n < kv_end && !hidden((int)(n >> page_shift << page_shift), 1 << page_shift))
        e = p.seq.table[seq * p.seq.table_stride + ((n + first_token) >> page_shift)];
      return e;
    };
    auto checked_pages = [&](int e) {
      if ((unsigned)e >= (unsigned)params_here().seq.n_pages) {
        bad = 1;
        e = 0;
      }
      return e;
    };
    // Moves on to the block that holds tile i, when i is its first (i > 0, in order). The wait for the loads of
    // the entries is here and nowhere else: the compiler does not count the asm loads around it.
    auto turn_pages = [&](int i) {
      if (kPages && (i & (block - 1)) == 0) {
        asm volatile("" : "+v"(pages_next));
        pages = checked_pages(pages_next);
        pages_next = load_pages(i + block);
      }
    };
    // the page of tile i's row x (wave-uniform)
    auto page_of = [&](int i, int x) {
      return __builtin_amdgcn_readlane(pages, ((i << tile_shift) & 63) + (x >> page_shift));
    };

    // ---- a wave loads JW KiB of consecutive rows of a tile, from row gwave * JW * RPI on: segments of SEG rows, each in
    // one page, with a buffer resource each. Rows from kv_end on read as zeros.
    constexpr int NS = JW / LPS;
    static_assert(JW % LPS == 0, "a wave loads whole segments");
    const bool loads = NI % GW == 0 || gwave < NI;  // (tiles of fewer KiB than waves)
    auto segment_row = [&](int s) { return gwave * JW * RPI + s * SEG; };
    auto segment_data = [&](const Source& x, int i, int s) {
      const int n = key_of(i) + segment_row(s);
      if constexpr (kPages)
        return x.data + (uint64_t)(uint32_t)page_of(i, segment_row(s)) * x.page +
               (uint64_t)(uint32_t)(n & ((1 << page_shift) - 1)) * x.token;
      else
        return x.data + (uint64_t)(uint32_t)(sq.kv_first + n) * x.token;
    };
    auto segment_bytes = [&](const Source& x, int i, int s, int row_bytes) {
      const int n = key_of(i) + segment_row(s);
      const int valid = hidden(n, SEG) ? 0 : max(min(kv_end - n, SEG), 0);
      return (uint32_t)max(valid * (int)x.token - ((int)x.token - row_bytes), 0);
    };
    auto issue = [&](const Source& x, const uint32_t (&off)[LPS], const FA2_LDS char* buf, int i) {
      if (!loads) return;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const u32x4 rsrc = make_desc(segment_data(x, i, s), segment_bytes(x, i, s, D * 2));
#pragma unroll
        for (int u = 0; u < LPS; ++u)
          load_lds16_settled(rsrc, off[u], lds_addr(buf + (gwave * JW + s * LPS + u) * 1024));
      }
    };
    auto issue_k = [&](int i) { issue(ks, koff, kbuf(i), i); };
    auto issue_v = [&](int i) { issue(vs, voff, vbuf(i), i); };

    // ---- e4m3: 16 values of one row a lane, and the row's scale byte
    struct Raw {
      u32x4 w[JW];
      uint32_t scale[JW];
    };
    auto fetch = [&](const Source& x, const Source& xs, const uint32_t (&off)[LPS], const uint32_t (&scale_off)[LPS], int i,
                     Raw& raw) {
      if (!loads) return;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const auto rsrc = buffer_of(segment_data(x, i, s), segment_bytes(x, i, s, D));
        const auto scales = buffer_of(segment_data(xs, i, s), segment_bytes(xs, i, s, 1));
#pragma unroll
        for (int u = 0; u < LPS; ++u) {
          raw.w[s * LPS + u] = load_buffer16(rsrc, off[u]);
          raw.scale[s * LPS + u] = load_buffer1(scales, scale_off[u]);
        }
      }
    };
    auto fetch_k = [&](int i, Raw& raw) { fetch(ks, kscale, koff, kscale_off, i, raw); };
    auto fetch_v = [&](int i, Raw& raw) { fetch(vs, vscale, voff, vscale_off, i, raw); };
    auto store = [&](bool is_v, const FA2_LDS char* to, Raw& raw) {
      FA2_LDS char* buf = (FA2_LDS char*)to;
      if (!loads) return;
#pragma unroll
      for (int jj = 0; jj < JW; ++jj) {
        // nothing that uses what was loaded moves up across this point, and with it the wait for it
        asm volatile("" : "+v"(raw.w[jj]), "+v"(raw.scale[jj]));
        const int row = (gwave * JW + jj) * RPI + lane / LPR, chunk = lane % LPR * 2;
        const int key = is_v ? v_key<D>(row & 15) : k_key<D>(pi_row(row & 31) & 15);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x2 lo = e4m3_to_16<DT>(raw.w[jj][2 * h], raw.scale[jj]);
          const u32x2 hi = e4m3_to_16<DT>(raw.w[jj][2 * h + 1], raw.scale[jj]);
          *(u32x4 FA2_LDS*)(buf + (row * CPR + ((chunk + h) ^ key)) * 16) = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      }
    };

    // ---- the online softmax of one tile, base 2, with a lazily moved reference (attn_fwd_wavesplit.hpp). The weights are
    // rounded to the 16-bit type, as the matrix instruction takes them, and the sum that the row is divided by is of the
    // rounded ones, so that a row's weights still add up to one; the log-sum-exp is of the sum in float. Against weights in float
    // the error of a row grows by 1.1 to 1.4 times (it is rounded to the same type at the end).
    float m_i = -INFINITY, l_i = 0.f, l_exact = 0.f;
    f32x16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
    auto softmax = [&](f32x16 (&s)[NB], u32x4 (&pb)[NT], int n0) {
      if (n0 + BN > full_end) {
        const int lim = last_key - n0 - 8 * g;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (nb * 32 + 16 * (x / 8) + (x % 8) > lim) s[nb][x] = -INFINITY;
      }
      if (kWindow && n0 < first_end && n0 + BN > sinks) {
        const int lim = first_key - n0 - 8 * g, open = sinks - n0 - 8 * g;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int n = nb * 32 + 16 * (x / 8) + (x % 8);
            if (n < lim && n >= open) s[nb][x] = -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 16; ++x) mx = fmaxf(mx, s[nb][x]);
      mx = pair_max(mx) * qk_scale;
      const bool grow = mx > m_i + kRescaleTau;
      if (__builtin_amdgcn_ballot_w64(grow)) {
        const float m_new = grow ? mx : m_i;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m_i - m_new) : 1.0f;
        l_i *= alpha;
        l_exact *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] *= alpha;
        m_i = m_new;
      }
      // a row that has seen no key in its tiles yet (reference -inf) gets weights 0, not NaN
      const float m_ref = m_i == -INFINITY ? 0.f : m_i;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 16; ++x)
          s[nb][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nb][x], qk_scale, -m_ref));
      if (want_exact) l_exact += lane_sum(s);
      float rs0 = 0.f, rs1 = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int nb = t >> 1, h = t & 1;
        pb[t] = u32x4{E::pack2(s[nb][8 * h + 0], s[nb][8 * h + 1]), E::pack2(s[nb][8 * h + 2], s[nb][8 * h + 3]),
                      E::pack2(s[nb][8 * h + 4], s[nb][8 * h + 5]), E::pack2(s[nb][8 * h + 6], s[nb][8 * h + 7])};
        rs0 = E::sum2(pb[t][0], rs0);
        rs1 = E::sum2(pb[t][1], rs1);
        rs0 = E::sum2(pb[t][2], rs0);
        rs1 = E::sum2(pb[t][3], rs1);
      }
      l_i += rs0 + rs1;
    };

    if constexpr (kPages) {
      pages = checked_pages(load_pages(0));
      pages_next = load_pages(block);
    }
    Raw kraw, vraw;
    if constexpr (GW == 1) {
      if constexpr (kE4m3) {
        fetch_k(0, kraw);
        fetch_v(0, vraw);
      } else {
        if (count > 0) {
          issue_k(0);
          issue_v(0);
        }
        // Q is waited for here: the compiler does not count the asm loads, so its own wait for Q is for
        // everything in flight, and inside the loop it would come every time
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qreg[ks]));
      }
      for (int i = 0; i < count; ++i) {
        if constexpr (kE4m3) store(false, kbuf(i), kraw);
        else wait_vm_fence<NI>();  // K_i has landed; V_i may be in flight
        u32x4 kop[KS][NB];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) kop[ks][nb] = k_operand(i, ks, nb);
        turn_pages(i + 1);
        if constexpr (kE4m3) {
          fetch_k(i + 1, kraw);
        } else {
          wait_lds_fence();  // the operands have left the buffer: refill it
          if (i + 1 < count) issue_k(i + 1);
        }
        f32x16 s[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[nb] = f32x16{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) s[nb] = E::mma(kop[ks][nb], qreg[ks], s[nb]);
        u32x4 pb[NT];
        softmax(s, pb, key_of(i));
        if constexpr (kE4m3) store(true, vbuf(i), vraw);
        else if (i + 1 < count) wait_vm_fence<NI>();  // V_i has landed; K_{i+1} may be in flight
        else wait_vm_fence<0>();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int db = 0; db < DB; ++db) acc[db] = E::mma(v_operand(i, t, db), pb[t], acc[db]);
        if constexpr (kE4m3) {
          fetch_v(i + 1, vraw);
        } else {
          wait_lds_fence();
          if (i + 1 < count) issue_v(i + 1);
        }
      }
    } else {
      // attn_fwd_kernel.hpp's one-tile loop. 16-bit sources: K_{j+2} and V_{j+1} are issued after tile j's barrier
      // and land before tile j + 1's. e4m3: K_{j+1} and V_j, fetched into registers one tile earlier, are
      // converted and written before tile j's barrier; the next ones are fetched right after.
      constexpr int LA_S = KS < 4 ? KS : 4;
      constexpr int NPV = NT * DB;
      constexpr int kLaV = D == 128 ? 2 : 4;
      constexpr int LA_V = NPV < kLaV ? NPV : kLaV;
      constexpr int NKP = LA_S * NB;
      u32x4 kop[LA_S][NB];
      if (n_tiles > 0) {
        if constexpr (kE4m3) {
          fetch_k(0, kraw);
          store(false, kbuf(0), kraw);
          fetch_k(1, kraw);
          fetch_v(0, vraw);
        } else {
          issue_k(0);
          issue_v(0);
          if (n_tiles > 1) issue_k(1);
          // K_0 has landed; V_0 and K_1 may be in flight (where every wave issues as many loads)
          if (NI % GW != 0) wait_vm_fence<0>();
          else if (n_tiles > 1) wait_vm_fence<2 * JW>();
          else wait_vm_fence<JW>();
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < LA_S; ++ks)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            kop[ks][nb] = *(const volatile u32x4 FA2_LDS*)(kbuf(0) + koffs[ks] + nb * 32 * CPR * 16);
      }
      // Q is waited for here, on every path: the compiler does not count the asm loads (see above)
#pragma unroll
      for (int x = 0; x < KS; ++x) asm volatile("" : "+v"(qreg[x]));
      // tiles that start past every row of the wave add exact zeros: their products are skipped
      const int wave_last = __builtin_amdgcn_readlane(last_key, 31);  // rows grow with the lane
      int n_active = 0;
      if constexpr (kWindow) {
        const int upto = wave_last < 0 ? 0 : wave_last / BN + 1;  // key tiles that start up to wave_last
        if (row0 + gwave * 32 < row_end)
          n_active = min(n_tiles, max((upto > sink_tiles ? max(upto - skip, sink_tiles) : upto) - t_begin, 0));
      } else if (!(row0 + gwave * 32 >= row_end || wave_last < kv_begin)) {
        n_active = min(n_tiles, (wave_last - kv_begin) / BN + 1);
      }
      auto turn_tile = [&](int j) {  // before tile j's barrier and after it: all that keeps the loads going
        if constexpr (kE4m3) {
          store(false, kbuf(j + 1), kraw);
          store(true, vbuf(j), vraw);
          fetch_v(j + 1, vraw);  // (j + 1's block of pages: K's have not moved on yet)
          turn_pages(j + 2);
          fetch_k(j + 2, kraw);
          __syncthreads();
        } else {
          wait_vm_fence<0>();  // this wave's loads of V_j and K_{j+1} have landed
          __syncthreads();     // ... every wave's; and every wave is done with K_j
          if (j + 1 < n_tiles) issue_v(j + 1);  // (as above)
          turn_pages(j + 2);
          if (j + 2 < n_tiles) issue_k(j + 2);
        }
      };
      for (int j = 0; j < n_active; ++j) {
        __builtin_amdgcn_s_setprio(1);
        f32x16 s[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[nb] = f32x16{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int slot = ks % LA_S;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) s[nb] = E::mma(kop[slot][nb], qreg[ks], s[nb]);
          if (ks + LA_S < KS) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) kop[slot][nb] = k_operand(j, ks + LA_S, nb);
          }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          __builtin_amdgcn_sched_group_barrier(0x008, NB, 0);
          if (ks + LA_S < KS) __builtin_amdgcn_sched_group_barrier(0x100, NB, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        turn_tile(j);
        u32x4 va[LA_V], pb[NT];
#pragma unroll
        for (int x = 0; x < LA_V; ++x) va[x] = v_operand(j, x / DB, x % DB);
        softmax(s, pb, key_of(j));
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < NPV; ++x) {
          acc[x % DB] = E::mma(va[x % LA_V], pb[x / DB], acc[x % DB]);
          if (x + LA_V < NPV) va[x % LA_V] = v_operand(j, (x + LA_V) / DB, (x + LA_V) % DB);
          // K_{j+1}'s first operands (a harmless stale read after the last tile)
#pragma unroll
          for (int y = x * NKP / NPV; y < (x + 1) * NKP / NPV; ++y)
            kop[y / NB][y % NB] = k_operand(j + 1, y / NB, y % NB);
        }
#pragma unroll
        for (int x = 0; x < NPV; ++x) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          const int nreads = (x + LA_V < NPV ? 2 : 0) + ((x + 1) * NKP / NPV - x * NKP / NPV);
#pragma unroll
          for (int y = 0; y < nreads; ++y) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      for (int j = n_active; j < n_tiles; ++j) turn_tile(j);
    }

    // ---- the piece's results. A weight of zero times an infinite or NaN value is NaN, and such a value may
    // lie in a key of a tile that the row does not see: rows whose sums are not finite are computed again, over the
    // keys that they see alone.
    if (__builtin_amdgcn_ballot_w64(bad != 0)) m_i = __uint_as_float(0x7fc00000u);
    const float l = pair_sum(l_i);
    const float lx = want_exact ? pair_sum(l_exact) : l;
    float test = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int x = 0; x < 16; ++x) test = __builtin_fmaf(acc[db][x], 0.f, test);
    // row x of the workgroup: its place in out, q and lse
    ParamsRef pe = params_here();
    const int group = pe.group;
    struct RowPlace {
      int64_t token;
      int head, pos;
    };
    auto place = [&](int x) {
      const int i = (row0 + x) / group;
      return RowPlace{(int64_t)(sq.first + i), hkv * group + (row0 + x - i * group), i};
    };
    // m, l and exact l of row x, by one lane
    auto put_sums = [&](int x, float m, float sum, float exact) {
      if (part) {
        *(f32x4*)(part + part_sums<BM, D>(x)) = f32x4{m, sum, exact, 0.f};
      } else if (kJoined) {
        const RowPlace at = place(x);
        *(f32x4*)(row_results<D, MODE>(pe, at.token, at.head) + D) = f32x4{m, sum, exact, __int_as_float(last_of(at.pos) < 0 ? 2 : 0)};
      } else if (pe.lse) {
        const RowPlace at = place(x);
        pe.lse[(int64_t)at.head * pe.seq.n_tokens + at.token] = (m + log2f(exact)) * kLn2;
      }
    };
    // One row again, by a wave: 64 keys at a time, one a lane; only keys that the row sees are read.
    auto again = [&](int x, bool nan) {
      const RowPlace at = place(x);
      const int end = nan ? kv_begin : min(last_of(at.pos) + 1, kv_end);
      const uint16_t* qrow = pe.q + at.token * pe.sqt + at.head * pe.sqh;
      int page = 0;
      auto row_at = [&](const auto& y, int n) {
        if constexpr (kPages) {
          page = pe.seq.table[seq * pe.seq.table_stride + ((n + first_token) >> page_shift)];
          if ((unsigned)page >= (unsigned)pe.seq.n_pages) page = 0;
          return y.data + (page * y.page + hkv * y.head + (int64_t)(n & ((1 << page_shift) - 1)) * y.token) * EB;
        } else {
          return y.data + ((int64_t)(sq.kv_first + n) * y.token + hkv * y.head) * EB;
        }
      };
      auto scale_at = [&](const auto& y, int n) {
        if constexpr (kE4m3)
          return e8m0_to_f32(y.scale[page * y.scale_page + hkv * y.scale_head +
                                     (int64_t)(n & ((1 << page_shift) - 1)) * y.scale_token]);
        else
          return 1.0f;
      };
      auto value = [&](const char* row, float scale, int d) {
        if constexpr (kE4m3) {
          const auto v = __builtin_amdgcn_cvt_pk_f32_fp8((int)(uint32_t)(uint8_t)row[d], false);
          return v[0] * scale;
        } else {
          return to_f32<DT>(((const uint16_t*)row)[d]);
        }
      };
      bool no_lse = nan;  // (an infinite score has one, though the row has no weights)
      float m = -INFINITY, sum = 0.f, o[(D + 63) / 64] = {};
      const int from = first_of(at.pos);
      auto sees = [&](int n) { return n < end && (!kWindow || n >= from || n < sinks); };
      for (int n0 = kv_begin; n0 < end; n0 += 64) {
        if (kWindow && n0 >= sinks && n0 + 64 <= from) n0 = from;
        const int n = n0 + lane;
        float s = -INFINITY;
        if (sees(n)) {
          const char* krow = row_at(pe.kc, n);
          const float scale = scale_at(pe.kc, n);
          s = 0.f;
          for (int d = 0; d < D; ++d) s = __builtin_fmaf(to_f32<DT>(qrow[d]), value(krow, scale, d), s);
          s *= qk_scale;
        }
        no_lse |= __builtin_amdgcn_ballot_w64(s != s) != 0;
        float m_new = s;  // fmaxf drops a NaN score here; its weight is NaN below
#pragma unroll
        for (int o2 = 32; o2 >= 1; o2 /= 2) m_new = fmaxf(m_new, __shfl_xor(m_new, o2, 64));
        m_new = fmaxf(m, m_new);
        const float m_ref = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_ref);
        const float w = sees(n) ? __builtin_amdgcn_exp2f(s - m_ref) : 0.f;
        m = m_new;
        sum = sum * alpha + w;
#pragma unroll
        for (int y = 0; y < (D + 63) / 64; ++y) o[y] *= alpha;
        for (int y = 0; y < min(end - n0, 64); ++y) {
          if constexpr (kWindow) {
            if (!sees(n0 + y)) continue;
          }
          const float wy = __shfl(w, y, 64);
          const char* vrow = row_at(pe.vc, n0 + y);
          const float scale = scale_at(pe.vc, n0 + y);
#pragma unroll
          for (int z = 0; z < (D + 63) / 64; ++z)
            if (lane + 64 * z < D) o[z] = __builtin_fmaf(wy, value(vrow, scale, lane + 64 * z), o[z]);
        }
      }
#pragma unroll
      for (int o2 = 32; o2 >= 1; o2 /= 2) sum += __shfl_xor(sum, o2, 64);
      if (no_lse) m = __uint_as_float(0x7fc00000u);
      const float inv = last_of(at.pos) < 0 ? 0.f : 1.0f / sum;
#pragma unroll
      for (int y = 0; y < (D + 63) / 64; ++y)
        if (lane + 64 * y < D) {
          const float v = nan ? m : o[y];
          if (part)
            part[part_index<GW, D>(x, lane + 64 * y)] = v;
          else if (kJoined)
            row_results<D, MODE>(pe, at.token, at.head)[lane + 64 * y] = v;
          else
            pe.o[at.token * pe.sot + at.head * pe.soh + lane + 64 * y] =
                (uint16_t)E::pack2(last_of(at.pos) < 0 ? 0.f : v * inv, 0.f);
        }
      // (an infinite score without a NaN one: the row's log-sum-exp is infinite too)
      if (lane == 0) put_sums(x, m, sum, m == INFINITY ? 1.0f : sum);
    };

    if constexpr (KG == 1) {
      const bool mine = row0 + wr < row_end;
      uint64_t again_rows = __builtin_amdgcn_ballot_w64(mine && test != 0.f);
      again_rows = (again_rows | (again_rows >> 32)) & 0xffffffffu;
      if (mine && !((again_rows >> c) & 1)) {
        const float inv = last_key < 0 ? 0.f : 1.0f / l;  // no key: 0
        const RowPlace at = place(wr);
        uint16_t* orow = pe.o + at.token * pe.sot + at.head * pe.soh;
        const float nan_or_0 = m_i != m_i ? m_i : 0.f;
        float* kept = kJoined ? row_results<D, MODE>(pe, at.token, at.head) : nullptr;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int d0 = 32 * db + 16 * h + 8 * g;
            if (d0 < D) {
              if (part || kJoined) {
                f32x4 lo, hi;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  lo[i] = acc[db][8 * h + i];
                  hi[i] = acc[db][8 * h + 4 + i];
                }
                *(f32x4*)(kJoined && !part ? kept + d0 : part + part_index<GW, D>(wr, d0)) = lo;
                *(f32x4*)(kJoined && !part ? kept + d0 + 4 : part + part_index<GW, D>(wr, d0 + 4)) = hi;
              } else {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(acc[db][8 * h + i], inv, nan_or_0);
                *(u32x4*)(orow + d0) = u32x4{E::pack2(y[0], y[1]), E::pack2(y[2], y[3]), E::pack2(y[4], y[5]),
                                             E::pack2(y[6], y[7])};
              }
            }
          }
        if (g == 0) put_sums(wr, m_i, l, lx);
      }
      for (uint64_t todo = again_rows; todo; todo &= todo - 1)
        again(gwave * 32 + __builtin_ctzll(todo), m_i != m_i);
    } else {
      auto& sm = mem.sm;
      auto& odd = mem.odd;
      // ---- merge the groups through LDS: O^T blocks as 16-byte pieces [group][row][4 dims], then
      // every thread folds the groups of its pieces
      if (tid < BM) odd[tid] = 0;
      if constexpr (!kE4m3) wait_vm_fence<0>();
      __syncthreads();  // every wave is done with every K/V buffer
      FA2_LDS f32x4* ob = (FA2_LDS f32x4*)lds;
      auto piece = [&](int group, int row, int q) {
        return (group * BM + row) * QPR + (q ^ (row & (QPR < 8 ? QPR - 1 : 7)));
      };
      if (row0 + wr < row_end) {
        if (test != 0.f) odd[wr] = 1;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int q = 8 * db + 4 * (h >> 1) + 2 * g + (h & 1);  // dims 4 q .. 4 q + 3
            if (q < QPR) {
              f32x4 x;
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = acc[db][4 * h + e];
              ob[piece(grp, wr, q)] = x;
            }
          }
        if (g == 0) {
          sm[grp][wr][0] = m_i;
          sm[grp][wr][1] = l;
          sm[grp][wr][2] = lx;
        }
      }
      __syncthreads();
      for (int t = tid; t < (row_end - row0) * QPR; t += 256) {
        const int x = t / QPR, q = t % QPR;
        if (odd[x]) continue;
        float m = -INFINITY, ls = 0.f, lxs = 0.f;
        bool nan = false;  // a group's reference: a bad page
#pragma unroll
        for (int y = 0; y < KG; ++y) {
          nan |= sm[y][x][0] != sm[y][x][0];
          m = fmaxf(m, sm[y][x][0]);
        }
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < KG; ++y) {
          const float mw = sm[y][x][0];
          const float w = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);  // (NaN stays NaN)
          ls = __builtin_fmaf(w, sm[y][x][1], ls);
          lxs = __builtin_fmaf(w, sm[y][x][2], lxs);
          const f32x4 v = ob[piece(y, x, q)];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(w, v[e], o[e]);
        }
        const RowPlace at = place(x);
        const float m_nan = nan ? __uint_as_float(0x7fc00000u) : m;
        if (part) {
          *(f32x4*)(part + part_index<GW, D>(x, 4 * q)) = o;
        } else if (kJoined) {
          *(f32x4*)(row_results<D, MODE>(pe, at.token, at.head) + 4 * q) = o;
        } else {
          const float inv = last_of(at.pos) < 0 ? 0.f : 1.0f / ls;  // no key: 0
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] *= inv;
          *(u32x2*)(pe.o + at.token * pe.sot + at.head * pe.soh + 4 * q) = u32x2{E::pack2(o[0], o[1]), E::pack2(o[2], o[3])};
        }
        // (fmaxf has dropped a NaN reference, and a piece whose groups all met bad pages would pass for one without keys)
        if (q == 0) put_sums(x, m_nan, ls, lxs);
      }
      for (int x = wave; x < row_end - row0; x += 4) {
        if (!odd[x]) continue;
        bool nan = false;
#pragma unroll
        for (int y = 0; y < KG; ++y) nan |= sm[y][x][0] != sm[y][x][0];
        again(x, nan);
      }
    }
    more = shared && share.x < share.end && next_tile<BM, kPages, MODE>(params_here(), lane, &cur);
  }
}

template <int DT, int D, int SRC, int GW, bool LSE, int MODE>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(ragged_waves(D, SRC, GW))))
void attn_ragged_kernel(const RaggedParams) {
  __shared__ RaggedLds<D, GW> mem;
  int hkv, rank;
  head_and_rank(params_here(), (int)blockIdx.x, &hkv, &rank);
  ragged_rows<DT, D, SRC, GW, LSE, MODE>(mem, hkv, rank, Cursor{});
}

// A window over chunks of prompts beside single tokens, where the chunks' rows fill the GPU: their 128-row tiles are shared out as
// ever, and each sequence of at most 32 rows has a 32-row workgroup of its own behind them. In 128-row tiles a token's row costs
// what a chunk's 128 do. Measured on MI355X, a chunk of 2048 beside 24 steps, window 2048, 28 / 4 heads of 128: 92 us and 17 of merge in
// 128-row tiles alone, 89 and 5 (no tile is cut) with both. When it is chosen, with other batches' times: serve_host.hpp, window_plan.
template <int DT, int D, int SRC, bool LSE>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(kSharedWaves)))
void attn_window_mixed_kernel(const RaggedParams) {
  __shared__ union {
    RaggedLds<D, 4> many;
    RaggedLds<D, 1> few;
  } mem;
  ParamsRef p = params_here();
  int hkv, rank;
  head_and_rank(p, (int)blockIdx.x, &hkv, &rank);
  Cursor cur{};
  cur.by_tile = rank >= p.shares;
  cur.rows_of = cur.by_tile ? kFewRows : kManyRows;
  if (cur.by_tile)
    ragged_rows<DT, D, SRC, 1, LSE, kModeWindow>(mem.few, hkv, rank - p.shares, cur);
  else
    ragged_rows<DT, D, SRC, 4, LSE, kModeWindow>(mem.many, hkv, rank, cur);
}

// Both passes of a batch with a common prefix in one launch: GWP row waves for the prefix's shares, whose rows are all of the
// batch's, GWO for the others. With M the larger of a row's two references m, O = sum 2^(m - M) O_pass / sum 2^(m - M) l_pass
// (attn_shared_join_kernel). K and V of the prefix are read once for 128 rows, where a step's own pass would read them for each
// sequence. Measured on MI355X, 32 steps behind 8192 shared tokens and up to 500 of their own, 32 / 8 heads of 128, bf16: 21.6 us and 7 of join
// (one launch after the other, each with its merge: 18 + 25 + 19 + 5; without sharing 63); bound by the chain of loads that finds a
// workgroup's work, its pages and its first keys (11 us with hardly a key). 16 drafts of up to 5 behind 32k, 28 / 4 heads, e4m3: 41 and 8; the
// loads of a tile, one ahead, and registers spilled at two workgroups a CU (34 of them; in e4m3 at head_dim 128 20 to 50; matrix
// cores 19% busy).
template <int DT, int D, int SRC, int GWP, int GWO, bool LSE>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(kSharedWaves)))
void attn_shared_kernel(const RaggedParams) {
  __shared__ union {
    RaggedLds<D, GWP> prefix;
    RaggedLds<D, GWO> own;
  } mem;
  ParamsRef p = params_here();
  int hkv, rank;
  head_and_rank(p, (int)blockIdx.x, &hkv, &rank);
  Cursor cur{};
  if (deal_shares<32 * GWP, 32 * GWO, SRC == kSourceE4m3>(p, rank, threadIdx.x & 63, &cur))
    ragged_rows<DT, D, SRC, GWP, LSE, kModePrefix>(mem.prefix, hkv, rank, cur);
  else
    ragged_rows<DT, D, SRC, GWO, LSE, kModeOwn>(mem.own, hkv, rank - cur.first_share, cur);
}

// Merges the pieces of the row tile that ends in share `rank` and starts in an earlier one: with M the largest of the
// pieces' references m_i, O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, in an order that the sizes alone decide. 32
// rows a workgroup, 4 dims a thread; bound by the latency of the pieces' loads, so a thread has one item and loads several
// pieces at once, and where a 32-row tile has few rows, up to 8 threads take an item's pieces in turn. Measured on MI355X, a
// step of one sequence of 30000, 32 / 8 heads of 128, 64 pieces a tile: 51 us with one thread an item, 35 with 8.
constexpr int combine_threads(int head_dim) { return head_dim <= 32 ? 256 : 8 * head_dim; }
struct Merged {
  float M, l, lx;
  f32x4 o;
  bool nan;
  __device__ void add(float m, float sum, float exact, const f32x4& v, bool is_nan) {
    const float M_new = fmaxf(M, m);
    const float a = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - M_new);
    const bool none = m == -INFINITY && !is_nan;  // (such a piece's values may be anything)
    const float w = is_nan ? __uint_as_float(0x7fc00000u) : none ? 0.f : __builtin_amdgcn_exp2f(m - M_new);
    nan |= is_nan;
    M = M_new;
    l = l * a + (none ? 0.f : w * sum);
    lx = lx * a + (none ? 0.f : w * exact);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * a + (none ? 0.f : w * v[e]);
  }
};
template <int DT, int D, int GW>
__global__ __launch_bounds__(combine_threads(D)) void attn_ragged_combine_kernel(const RaggedParams) {
  using E = Elem<DT>;
  ParamsRef p = params_here();
  constexpr int BM = 32 * GW, QPR = D / 4, STEP = 6, THREADS = combine_threads(D), WAYS = GW == 1 ? 8 : 1;
  static_assert(32 * QPR <= THREADS, "one item a thread");
  __shared__ f32x4 values[WAYS > 1 ? THREADS : 1], sums_of[WAYS > 1 ? THREADS : 1];
  const int rank = (int)blockIdx.x / GW % p.shares, hkv = (int)blockIdx.x / GW / p.shares;
  const Merge at = *merge_of(p, hkv, rank);
  if (at.first < 0) return;
  const int x0 = (int)blockIdx.x % GW * 32;
  const int n = (GW == 1 ? min(32, at.rows) : 32) * QPR;
  const int ways = WAYS == 1 ? 1 : min(min(WAYS, THREADS / n), rank - at.first + 1);
  const int way = (int)threadIdx.x / n, t = (int)threadIdx.x - way * n;
  // 4 dims of a row a thread, in the order that the partial results lie in
  const int x = x0 + (GW == 1 ? t / QPR : t & 31);
  const int q = GW == 1 ? t % QPR : t / 128 * 4 + (t / 32 & 1) * 2 + (t / 64 & 1);
  Merged r = {-INFINITY, 0.f, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}, false};
  if (way < ways && x < at.rows) {
    for (int i0 = at.first + way; i0 <= rank; i0 += STEP * ways) {
      f32x4 sums[STEP], v[STEP];
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        const int i = min(i0 + k * ways, rank);
        const float* part = part_of<BM, D>(p, hkv, i, i == at.first);
        sums[k] = *(const f32x4*)(part + part_sums<BM, D>(x));
        v[k] = *(const f32x4*)(part + part_index<GW, D>(x, 4 * q));
      }
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        if (i0 + k * ways > rank) break;
        r.add(sums[k][0], sums[k][1], sums[k][2], v[k], sums[k][0] != sums[k][0]);
      }
    }
  }
  if constexpr (WAYS > 1) {
    if (ways > 1) {
      values[threadIdx.x] = r.o;
      sums_of[threadIdx.x] = f32x4{r.M, r.l, r.lx, r.nan ? 1.f : 0.f};
      __syncthreads();
      if (way == 0)
        for (int y = 1; y < ways; ++y) {
          const f32x4 s = sums_of[y * n + t];
          r.add(s[0], s[1], s[2], values[y * n + t], s[3] != 0.f);
        }
    }
  }
  if (way > 0 || x >= at.rows) return;
  const int pos = (at.row0 + x) / p.group, head = hkv * p.group + (at.row0 + x - pos * p.group);
  const int64_t token = at.token + pos;
  const bool none = (p.causal ? min(pos + at.shift, at.n_kv - 1) : at.n_kv - 1) < 0;
  const float inv = none ? 0.f : 1.0f / r.l;
  *(u32x2*)(p.o + token * p.sot + head * p.soh + 4 * q) =
      u32x2{E::pack2(r.o[0] * inv, r.o[1] * inv), E::pack2(r.o[2] * inv, r.o[3] * inv)};
  if (p.lse && q == 0)  // (an infinite score has an infinite log-sum-exp, though the row has no weights)
    p.lse[(int64_t)head * p.seq.n_tokens + token] = !r.nan && r.M == INFINITY ? r.M : (r.M + log2f(r.lx)) * kLn2;
}

// Joins a row's results over a common prefix and over its own keys, each in one place or in pieces, as pieces are merged. 8
// neighbouring rows a workgroup (those of 32 rows' pieces lie side by side), 4 dims of a row a thread, and as many threads in
// turn for its pieces as 1024 have room for: bound by the latency of the pieces' loads.
template <int DT, int D, int GWP, int GWO>
__global__ __launch_bounds__(1024) void attn_shared_join_kernel(const RaggedParams) {
  using E = Elem<DT>;
  ParamsRef p = params_here();
  constexpr int ROWS = 8, Q = D / 4, WAYS = 1024 / (ROWS * Q), STEP = 4;
  __shared__ f32x4 values[1024], sums_of[1024];
  const int blocks = (int)(((int64_t)p.seq.n_tokens * p.group + ROWS - 1) / ROWS);
  const int hkv = (int)blockIdx.x / blocks, r = ((int)blockIdx.x - hkv * blocks) * ROWS + (int)(threadIdx.x % ROWS);
  const int q = (int)threadIdx.x / ROWS % Q, way = (int)threadIdx.x / (ROWS * Q);
  const int token = r / p.group, head = hkv * p.group + (r - token * p.group);
  const bool mine = token >= row_bound(p.seq.cu, 0, p.seq.n_tokens) && token < row_bound(p.seq.cu, p.seq.n_seq, p.seq.n_tokens);
  Merged m = {-INFINITY, 0.f, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}, false};
  bool no_key = false;
  auto take = [&](const f32x4& sums, const f32x4& value, auto gw) {
    constexpr int GW = decltype(gw)::value;
    if ((__float_as_int(sums[3]) & 1) == 0) {
      if (way == 0) m.add(sums[0], sums[1], sums[2], value, sums[0] != sums[0]);
      return;
    }
    // (held to the workspace, whatever lies there if the lengths changed under the launch)
    const int first = min(max(__float_as_int(sums[0]), 0), p.shares - 1), last = min(max(__float_as_int(sums[1]), 0), p.shares - 1);
    const int x = min(max(__float_as_int(sums[2]), 0), 32 * GW - 1);
    for (int i0 = first + way; i0 <= last; i0 += STEP * WAYS) {
      f32x4 s[STEP], v[STEP];
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        const int i = min(i0 + k * WAYS, last);
        const float* part = joined_part<D>(p, hkv, i, i == first);
        s[k] = *(const f32x4*)(part + part_sums<32 * GW, D>(x));
        v[k] = *(const f32x4*)(part + part_index<GW, D>(x, 4 * q));
      }
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        if (i0 + k * WAYS > last) break;
        m.add(s[k][0], s[k][1], s[k][2], v[k], s[k][0] != s[k][0]);
      }
    }
  };
  if (mine) {
    const float *of_prefix = row_results<D, kModePrefix>(p, token, head), *of_own = row_results<D, kModeOwn>(p, token, head);
    const f32x4 a = *(const f32x4*)(of_prefix + D), b = *(const f32x4*)(of_own + D);
    // (where a row is in pieces its place for values holds nothing, and is not looked at)
    const f32x4 va = *(const f32x4*)(of_prefix + 4 * q), vb = *(const f32x4*)(of_own + 4 * q);
    no_key = (__float_as_int(b[3]) & 2) != 0;
    take(a, va, std::integral_constant<int, GWP>{});
    take(b, vb, std::integral_constant<int, GWO>{});
  }
  if constexpr (WAYS > 1) {
    values[threadIdx.x] = m.o;
    sums_of[threadIdx.x] = f32x4{m.M, m.l, m.lx, m.nan ? 1.f : 0.f};
    __syncthreads();
    if (way == 0)
      for (int y = 1; y < WAYS; ++y) {
        const f32x4 s = sums_of[y * ROWS * Q + threadIdx.x];
        m.add(s[0], s[1], s[2], values[y * ROWS * Q + threadIdx.x], s[3] != 0.f);
      }
  }
  if (!mine || way > 0) return;
  const float inv = no_key ? 0.f : 1.0f / m.l;
  *(u32x2*)(p.o + token * p.sot + head * p.soh + 4 * q) =
      u32x2{E::pack2(m.o[0] * inv, m.o[1] * inv), E::pack2(m.o[2] * inv, m.o[3] * inv)};
  if (p.lse && q == 0)
    p.lse[(int64_t)head * p.seq.n_tokens + token] = !m.nan && m.M == INFINITY ? m.M : (m.M + log2f(m.lx)) * kLn2;
}

}  // namespace fa2
