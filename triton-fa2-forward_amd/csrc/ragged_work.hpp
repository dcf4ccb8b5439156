// ragged_work.hpp - which rows and keys a workgroup of the ragged attention kernel takes. Sequence lengths
// are known on the device only, so every workgroup works this out from the index vectors: 64 sequences
// at a time, one a lane, their lengths kept in registers for the next piece.
//
// A row tile is BM rows of one KV head's group of query heads of one sequence; every head has the same tiles.
// Two ways to deal them out:
//   * a workgroup per tile (as many workgroups as n_tokens rows in n_seq sequences can have tiles at most).
//     Up to 8 sequences' tiles go by their index in their sequence, highest first: causal tiles of high index see the most
//     keys, so the longest start first. More sequences go one after the other, each from its highest tile down: its tiles
//     share its K and V in an L2, and the search is shorter. Measured on MI355X, by index and by sequence: 4 of up to
//     8192, 16 heads of 64 with the log-sum-exp, 231 and 256 us; 8 of up to 2048, 32 / 8 heads of 128, 116 and 115 to 119;
//     16 of 512 78 and 65; 64 of 128 77 and 46, of 1024 1012 and 689. Windows, whose tiles are nearly even, have the same rule: 4 of up to
//     8192, window 1024, 32 / 8 heads of 128, 513 and 495; 8 of 4096 577 and 557; 8 of 2000, window 128, 16 heads of 64, 44.0 and 42.6; of 8192, 3000
//     and twice 100, window 512, 49.6 and 53.9; 16 of 2048, window 1024, 523 and 494.
//   * `shares` workgroups per head, each an equal share of the head's tiles laid end to end, a tile's length being
//     its keys (an estimate, linear in the tile's index, so that a sequence's sum is a closed form; it only
//     decides where the cuts lie). A share starts and ends inside tiles: a tile cut by a share's end leaves
//     partial results (slot 1 of the share it starts in, slot 0 of the others), which the combine kernel merges. For
//     few or uneven tiles, decoding above all, whatever the lengths are. Where a tile per workgroup would take no
//     longer after all (whole_tiles), that is what the workgroups do.
#pragma once

#include "serve_common.hpp"
#include "serve_launch.hpp"

namespace fa2 {

// The kernel's arguments, read where they lie. The compiler loads an argument once, at the kernel's start, and keeps it;
// there are many here, most of them used before and after the tile loop only, and kept in spilled SGPRs they
// cost the loop vector registers. Behind this point's opaque pointer they are loaded again.
#define FA2_CONSTANT __attribute__((address_space(4)))
using ParamsRef = const FA2_CONSTANT RaggedParams&;
__device__ __forceinline__ ParamsRef params_here() {
  auto p = (const FA2_CONSTANT RaggedParams*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}

// kTileCost of a 32-row tile behind a common prefix, where keys are few and the chain of a tile's loads takes longest; and in e4m3 beside that, as
// the shares are dealt. Measured on MI355X, 32 / 8 heads of 128, costs of 64 / 128 / 256 / 384 / 640: 32 steps of one 16-bit token of their own
// behind 4096 shared 29.5 / 22.2 / 17.7 / 17.7 / 18.1 us, of up to 500 behind 8192 24.2 / 25.7 / 24.5 / 24.6 / 24.8; 16 drafts of one e4m3 token
// of their own behind 64 29.4 / 19.9 / 13.6 / 13.9 / 15.8, of up to 300 behind 32k 51.0 / 54.7 / 53.0 / 50.2 / 49.8. In 16 bits, a whole call with its
// join: 128 steps of up to 300 behind 8192 62 / 55 / 50 / 50 / 53, with heads of 64 54 / 47 / 46 / 42 / 40, of 32 46 / 43 / 39 / 39 / 34, 16 / 16 heads of
// 64 50 / 49 / 46 / 46 / 52; 16 drafts of 5 and up to 300 behind 8192 50 / 48 / 42 / 37 / 33, of 64 39 / 36 / 34 / 30 / 27, of 32 31 / 30 / 27 / 27 / 24.
constexpr int kOwnTileCost = 384, kOwnE4m3Cost = 448;
// The most sequences whose tiles go by their index (above; at most 64, a lane each).
constexpr int kFewSequences = 8;
// Keys of the smallest share: four tiles of 64, or two of 32 for each of four waves. Measured on MI355X, 128 / 256 / 512: steps of
// one sequence of 2000 17.0 / 15.3 / 16.3 us, a chunk of 100 behind 2k 41 / 32 / 32, of 200 behind 4k 43 / 43 / 51.
constexpr int kLeastShare = 256;

// The sequence that this lane holds of a block of 64
struct LaneSequence {
  int first, n_q, n_kv, kv_first;
};

template <bool PAGES>
__device__ __forceinline__ LaneSequence lane_sequence(ParamsRef p, int s) {
  LaneSequence q = {0, 0, 0, 0};
  if (s >= p.seq.n_seq) return q;
  q.first = row_bound(p.seq.cu, s, p.seq.n_tokens);
  q.n_q = max(row_bound(p.seq.cu, s + 1, p.seq.n_tokens) - q.first, 0);
  if constexpr (PAGES) {
    q.n_kv = (int)min((int64_t)max(p.seq.lens[s], 0), (int64_t)p.seq.max_pages << p.seq.page_shift);
  } else {
    q.kv_first = row_bound(p.cu_kv, s, p.kv_tokens);
    q.n_kv = max(row_bound(p.cu_kv, s + 1, p.kv_tokens) - q.kv_first, 0);
  }
  return q;
}

// Sums up to each lane, and the largest and least of a wave, by moves between neighbouring lanes (DPP): a step takes a few cycles
// where one through LDS takes a hundred, and a workgroup's search for its work is a chain of them. Lanes that a move does not reach
// take `old`.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int old, int x) {
  return __builtin_amdgcn_update_dpp(old, x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t moved64(int64_t old, int64_t x) {
  const uint32_t lo = (uint32_t)moved<CTRL, ROWS>((int)(uint32_t)old, (int)(uint32_t)x);
  const uint32_t hi = (uint32_t)moved<CTRL, ROWS>((int)(old >> 32), (int)(x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
// Every lane's value joined by f with those of the lanes before it: 1, 2, 4 and 8 lanes back in its row of 16, then the row's and the
// half wave's before it
template <class F>
__device__ __forceinline__ int64_t wave_fold(int64_t x, bool sums, F&& f) {
  x = f(x, moved64<0x111, 0xf>(sums ? 0 : x, x));
  x = f(x, moved64<0x112, 0xf>(sums ? 0 : x, x));
  x = f(x, moved64<0x114, 0xf>(sums ? 0 : x, x));
  x = f(x, moved64<0x118, 0xf>(sums ? 0 : x, x));
  x = f(x, moved64<0x142, 0xa>(sums ? 0 : x, x));
  return f(x, moved64<0x143, 0xc>(sums ? 0 : x, x));
}
__device__ __forceinline__ int64_t wave_scan(int64_t x, int) {
  return wave_fold(x, true, [](int64_t a, int64_t b) { return a + b; });
}
__device__ __forceinline__ int wave_min(int x) {
  x = min(x, moved<0x111, 0xf>(x, x));
  x = min(x, moved<0x112, 0xf>(x, x));
  x = min(x, moved<0x114, 0xf>(x, x));
  x = min(x, moved<0x118, 0xf>(x, x));
  x = min(x, moved<0x142, 0xa>(x, x));
  x = min(x, moved<0x143, 0xc>(x, x));
  return __builtin_amdgcn_readlane(x, 63);
}

// The leading tokens that all sequences with new tokens have in common, and of whose rows of the table they are read. At
// most p.shared says, whole pages, and none that is a row's own or behind it: every row of the call sees them all.
// Everyone who asks gets the same answer, so that the two passes over the keys agree.
struct Prefix {
  int tokens, row;
};
__device__ __forceinline__ Prefix common_prefix(ParamsRef p, int lane, const LaneSequence& first) {
  int tokens = (int)min((int64_t)max(p.shared[0], 0), (int64_t)p.seq.max_pages << p.seq.page_shift), row = p.seq.n_seq;
  LaneSequence q = first;  // (of the first 64 sequences)
  for (int s = lane;;) {
    if (q.n_q > 0) {
      tokens = min(tokens, max(q.n_kv - q.n_q, 0));
      row = min(row, s);
    }
    s += 64;
    if (s - lane >= p.seq.n_seq) break;
    q = lane_sequence<true>(p, s);
  }
  tokens = wave_min(tokens) & ~((1 << p.seq.page_shift) - 1);
  row = wave_min(row);
  return row == p.seq.n_seq ? Prefix{0, 0} : Prefix{tokens, row};
}

// The block's lane l, wave-uniform
__device__ __forceinline__ LaneSequence sequence_at(const LaneSequence& q, int l) {
  return LaneSequence{__builtin_amdgcn_readlane(q.first, l), __builtin_amdgcn_readlane(q.n_q, l),
                      __builtin_amdgcn_readlane(q.n_kv, l), __builtin_amdgcn_readlane(q.kv_first, l)};
}

template <int BM>
__device__ __forceinline__ int row_tiles(int n_q, int group) {
  return (n_q * group + BM - 1) / BM;
}

// The length of a sequence's tiles on the line that is shared out: tile t's is base + slope t.
struct Lengths {
  int64_t base, slope;
  __device__ int64_t of(int64_t t) const { return base + slope * t; }
  __device__ int64_t before(int64_t t) const { return t * base + slope * (t * (t - 1) / 2); }
};
// ... of a window, at most `cap`, which tiles reach from `full` on.
struct WindowLengths {
  int64_t base, slope, cap, full;
  __device__ int64_t of(int64_t t) const { return min(base + slope * t, cap); }
  __device__ int64_t before(int64_t t) const {
    const int64_t u = min(t, full);
    return u * base + slope * (u * (u - 1) / 2) + (t - u) * cap;
  }
};
template <int BM, int MODE>
__device__ __forceinline__ auto lengths_of(ParamsRef p, int n_q, int n_kv) {
  if constexpr (MODE == kModeWindow) {
    const int64_t slope = BM / p.group, base = (int64_t)max(n_kv - n_q, 0) + slope + kTileCost<BM>;
    const int64_t cap = (int64_t)p.window + p.sinks + slope + kTileCost<BM>;
    const int64_t full = base >= cap ? 0 : slope == 0 ? (int64_t)1 << 31 : (cap - base + slope - 1) / slope;
    return WindowLengths{base, slope, cap, full};
  } else {
    constexpr int64_t kCost = MODE == kModeOwn && BM == 32 ? kOwnTileCost : kTileCost<BM>;
    if (MODE == kModePrefix || !p.causal) return Lengths{(int64_t)n_kv + kCost, 0};
    const int64_t slope = BM / p.group;
    return Lengths{(int64_t)max(n_kv - n_q, 0) + slope + kCost, slope};
  }
}

__device__ __forceinline__ int64_t readlane64(int64_t x, int l) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, l);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)x >> 32), l);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Sequences by their rows of a KV head
enum Rows { kAnyRows, kManyRows, kFewRows };  // more than 32, or at most 32

// A place among the sequences: the block of 64 that starts at s0 is in `lanes`, the sequence is its lane l.
struct Cursor {
  int s0, l, tile;
  LaneSequence lanes;
  // Of a common prefix's passes: the first 64 sequences (loaded once, by every lane for all passes), the rows of all, the prefix, and the
  // shares of this pass among those of the head
  LaneSequence raw;
  int rows_first, rows;
  Prefix prefix;
  int shares, first_share;
  double per_share;
  // Of a window: the sequences that a workgroup takes, and whether it takes one row tile of them
  Rows rows_of;
  bool by_tile;
};
// Sequences whose tiles are dealt out
template <int MODE>
__device__ __forceinline__ int sequences(ParamsRef p) {
  return MODE == kModePrefix ? min(p.seq.n_seq, 1) : p.seq.n_seq;
}
// Lane s of the sequences as the pass takes them: all rows as one sequence's over a prefix; or the keys behind it, kv_first being
// the first one's position
template <bool PAGES, int MODE>
__device__ __forceinline__ LaneSequence lane_sequence(ParamsRef p, int s, const Cursor& c) {
  if constexpr (MODE < kModePrefix) {
    LaneSequence q = lane_sequence<PAGES>(p, s);
    if (MODE == kModeWindow && c.rows_of != kAnyRows && (q.n_q * p.group <= 32) != (c.rows_of == kFewRows)) q.n_q = 0;
    return q;
  }
  if (MODE == kModePrefix) return s == 0 ? LaneSequence{c.rows_first, c.rows, c.prefix.tokens, 0} : LaneSequence{0, 0, 0, 0};
  LaneSequence q = s < 64 ? c.raw : lane_sequence<true>(p, s);
  q.kv_first = c.prefix.tokens;
  q.n_kv = max(q.n_kv - c.prefix.tokens, 0);
  return q;
}
template <int MODE>
__device__ __forceinline__ int shares_of(ParamsRef p, const Cursor& c) {
  return MODE >= kModePrefix ? c.shares : p.shares;
}
template <int MODE>
__device__ __forceinline__ double per_share_of(ParamsRef p, const Cursor& c) {
  return MODE >= kModePrefix ? c.per_share : p.per_share;
}

// The rank-th row tile; false: there are fewer.
template <int BM, bool PAGES, int MODE>
__device__ __forceinline__ bool find_tile(ParamsRef p, int rank, int lane, Cursor* c) {
  c->lanes = lane_sequence<PAGES, MODE>(p, lane, *c);
  if (sequences<MODE>(p) <= kFewSequences) {
    // Tiles of index t and above, over all sequences: A(t) = sum_s max(tiles_s - t, 0). The rank-th tile in the
    // order of falling t has the largest t with A(t) > rank; every lane tries a t of its own.
    const int tiles = row_tiles<BM>(c->lanes.n_q, p.group);
    int hi = 0;
    for (int s = 0; s < sequences<MODE>(p); ++s) hi = max(hi, __builtin_amdgcn_readlane(tiles, s));
    auto above = [&](int t) {
      int a = 0;
      for (int s = 0; s < sequences<MODE>(p); ++s) a += max(__builtin_amdgcn_readlane(tiles, s) - t, 0);
      return a;
    };
    if (above(0) <= rank) return false;
    int lo = 0;
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64;
      const int t = lo + lane * step;
      const uint64_t yes = __builtin_amdgcn_ballot_w64(t < hi && above(t) > rank);
      lo += (__builtin_popcountll(yes) - 1) * step;
      hi = min(lo + step, hi);
    }
    const int nth = rank - __builtin_amdgcn_readfirstlane(above(lo + 1));  // among the sequences with a tile lo
    const uint64_t have = __builtin_amdgcn_ballot_w64(tiles > lo);
    const int before = __builtin_popcountll(have & ((1ull << lane) - 1));
    c->s0 = 0;
    c->l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(((have >> lane) & 1) && before == nth));
    c->tile = lo;
    return true;
  }
  int64_t base = 0;
  for (int s0 = 0; s0 < sequences<MODE>(p); s0 += 64) {
    if (s0) c->lanes = lane_sequence<PAGES, MODE>(p, s0 + lane, *c);
    const int64_t tiles = row_tiles<BM>(c->lanes.n_q, p.group);
    const int64_t upto = base + wave_scan(tiles, lane);
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > rank);
    if (past) {
      c->s0 = s0;
      c->l = __builtin_ctzll(past);
      c->tile = (int)(readlane64(upto, c->l) - 1 - rank);
      return true;
    }
    base = readlane64(upto, 63);
  }
  return false;
}

__device__ __forceinline__ int64_t wave_max(int64_t x) {
  return readlane64(wave_fold(x, false, [](int64_t a, int64_t b) { return max(a, b); }), 63);  // (a scalar: what is chosen by it stays one too)
}

// Whether a tile per workgroup takes no longer than equal shares, as estimated: as many tiles as workgroups at most, whose
// longest costs no more than a share and what sharing costs. With one workgroup a CU, half of those that
// fit, a key takes 5/8 of the time. Measured on MI355X (32 / 8 heads of 128), whole tiles and shares: 4 prompts of 500
// 25 and 41 us; a chunk of 500 behind 500 33 and 40, behind 2k 62 and 53; 4 of 500 behind 4k 146 and 161. Behind a common prefix
// 32-row tiles too, as a cut costs one more of their chains of loads: 32 steps of up to 500 behind 8192 shared 24.6 and 22.9.
template <int BM>
__device__ __forceinline__ bool whole_tiles(int shares, double per_share, int64_t tiles, int64_t total, int64_t longest) {
  if (tiles > shares) return false;
  if (BM == 32) return longest <= (int64_t)((double)total * per_share) + 2 * kOwnTileCost;
  return (2 * tiles <= shares ? 5 * longest / 8 : longest) <= (int64_t)((double)total * per_share) + kShareCost;
}

// Share j: [x, end) of the line, the cursor at the tile that x lies in, `in` from its start; x >= end: nothing.
// With whole_tiles, the j-th tile.
struct Share {
  int64_t x, end, in, size;
};
template <int BM, bool PAGES, int MODE>
__device__ __forceinline__ Share find_share(ParamsRef p, int j, int lane, Cursor* c) {
  auto length = [&]() {
    return lengths_of<BM, MODE>(p, c->lanes.n_q, c->lanes.n_kv).before(row_tiles<BM>(c->lanes.n_q, p.group));
  };
  c->lanes = lane_sequence<PAGES, MODE>(p, lane, *c);
  c->s0 = 0;
  int64_t mine = length();
  int64_t upto = wave_scan(mine, lane);
  int64_t total = readlane64(upto, 63);
  for (int s0 = 64; s0 < sequences<MODE>(p); s0 += 64) {
    c->lanes = lane_sequence<PAGES, MODE>(p, s0 + lane, *c);
    total += readlane64(wave_scan(length(), lane), 63);
  }
  Share w;
  // (the same for every workgroup; how it is rounded does not matter, as long as shares * size reaches the total)
  w.size = max((int64_t)((double)total * per_share_of<MODE>(p, *c)) + 1, (int64_t)kLeastShare);
  w.x = w.size * j;
  w.end = min(w.x + w.size, total);
  w.in = 0;
  if ((BM != 32 || MODE == kModeOwn) && sequences<MODE>(p) <= 64) {
    const auto len = lengths_of<BM, MODE>(p, c->lanes.n_q, c->lanes.n_kv);
    const int64_t tiles = row_tiles<BM>(c->lanes.n_q, p.group), tiles_upto = wave_scan(tiles, lane);
    if (whole_tiles<BM>(shares_of<MODE>(p, *c), per_share_of<MODE>(p, *c), readlane64(tiles_upto, 63), total, wave_max(tiles > 0 ? len.of(tiles - 1) : 0))) {
      const uint64_t past = __builtin_amdgcn_ballot_w64(tiles_upto > j);
      w.end = w.x;
      if (!past) return w;
      c->l = __builtin_ctzll(past);
      c->tile = j - (int)readlane64(tiles_upto - tiles, c->l);
      w.end += readlane64(len.of(c->tile), c->l);
      return w;
    }
  }
  if (w.x >= w.end) return w;
  int64_t base = 0;
  if (sequences<MODE>(p) > 64) c->lanes = lane_sequence<PAGES, MODE>(p, lane, *c);
  while (base + readlane64(upto, 63) <= w.x) {  // (w.x < total: ends within the sequences)
    base += readlane64(upto, 63);
    c->s0 += 64;
    if (c->s0 >= sequences<MODE>(p)) {  // only if the lengths changed since they were summed
      w.end = w.x;
      return w;
    }
    c->lanes = lane_sequence<PAGES, MODE>(p, c->s0 + lane, *c);
    mine = length();
    upto = wave_scan(mine, lane);
  }
  c->l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(base + upto > w.x));
  w.in = w.x - base - readlane64(upto - mine, c->l);
  const LaneSequence q = sequence_at(c->lanes, c->l);
  const auto len = lengths_of<BM, MODE>(p, q.n_q, q.n_kv);
  int lo = 0, hi = row_tiles<BM>(q.n_q, p.group);  // the largest t with before(t) <= in
  while (hi - lo > 1) {
    const int t = (lo + hi) / 2;
    if (len.before(t) <= w.in)
      lo = t;
    else
      hi = t;
  }
  c->tile = lo;
  w.in -= len.before(lo);
  return w;
}

// A cut at x of a tile's length, in its key tiles: the shares on both sides of it compute the same. A cut within the
// tile's first or last key tile is moved to its end, as a piece costs more than a key tile (its prologue,
// epilogue and merge).
__device__ __forceinline__ int cut_at(int64_t x, int64_t length, int key_tiles) {
  const int t = (int)((double)x * key_tiles / (double)length);
  return t <= 1 ? 0 : t >= key_tiles - 1 ? key_tiles : t;
}

// The next tile after the cursor's on the line; false: there is none.
template <int BM, bool PAGES, int MODE>
__device__ __forceinline__ bool next_tile(ParamsRef p, int lane, Cursor* c) {
  const LaneSequence q = sequence_at(c->lanes, c->l);
  if (++c->tile < row_tiles<BM>(q.n_q, p.group)) return true;
  c->tile = 0;
  for (;;) {
    const uint64_t have =
        __builtin_amdgcn_ballot_w64(row_tiles<BM>(c->lanes.n_q, p.group) > 0 && lane > c->l);
    if (have) {
      c->l = __builtin_ctzll(have);
      return true;
    }
    if (c->s0 + 64 >= sequences<MODE>(p)) return false;
    c->s0 += 64;
    c->l = -1;
    c->lanes = lane_sequence<PAGES, MODE>(p, c->s0 + lane, *c);
  }
}

// The (KV head, rank) of a workgroup: a head stays on one XCD where the heads split evenly over them, and on a
// fixed few where the XCDs split evenly over the heads, so that its tiles share K and V in an L2.
__device__ __forceinline__ void head_and_rank(ParamsRef p, int block, int* head, int* rank) {
  const int xcds = 1 << p.xcd_shift;
  const int xcd = block & (xcds - 1), slot = block >> p.xcd_shift;
  if ((p.h_kv & (xcds - 1)) == 0) {
    const int per = p.h_kv >> p.xcd_shift;
    *head = xcd * per + slot % per;
    *rank = slot / per;
  } else {
    *head = block % p.h_kv;
    *rank = block / p.h_kv;
  }
}

// The shares of a head dealt to a common prefix's keys and to those behind it, as their lines' lengths are, whose keys cost
// a 128-row workgroup 3/2 of a 32-row one; true: share `rank` is one of the prefix's. (Every workgroup gets the same.)
template <int BMP, int BMO, bool E4M3>
__device__ __forceinline__ bool deal_shares(ParamsRef p, int rank, int lane, Cursor* c) {
  c->raw = lane_sequence<true>(p, lane);
  c->rows_first = row_bound(p.seq.cu, 0, p.seq.n_tokens);
  c->rows = max(row_bound(p.seq.cu, p.seq.n_seq, p.seq.n_tokens) - c->rows_first, 0);
  c->prefix = common_prefix(p, lane, c->raw);
  // (no keys: only empty results to write. Measured on MI355X, 32 / 8 heads of 128, costs of 16 / 128 / 512: 32 steps of 500 to 1000 keys
  // 30.1 / 30.6 / 30.3 us, 128 of 100 to 200 33.1 / 32.9 / 31.5, 16 drafts of 5 20.7 / 20.4 / 20.4)
  const int64_t cost = c->prefix.tokens == 0 ? 128 : c->prefix.tokens + kTileCost<BMP>;
  double ours = (double)(row_tiles<BMP>(c->rows, p.group) * cost) * (BMP > BMO ? 1.5 : 1.0), own = 0.0;
  for (int s0 = 0; s0 < p.seq.n_seq; s0 += 64) {
    const LaneSequence q = lane_sequence<true, kModeOwn>(p, s0 + lane, *c);
    const int64_t tiles = row_tiles<BMO>(q.n_q, p.group);
    const int64_t line = lengths_of<BMO, kModeOwn>(p, q.n_q, q.n_kv).before(tiles) + (E4M3 ? kOwnE4m3Cost * tiles : 0);
    own += (double)readlane64(wave_scan(line, lane), 63);
  }
  const double share = ours + own > 0.0 ? ours / (ours + own) : 0.5;
  const int prefix = __builtin_amdgcn_readfirstlane(min(max((int)(share * p.shares + 0.5), 1), p.shares - 1));
  const bool is_prefix = rank < prefix;
  c->first_share = is_prefix ? 0 : prefix;
  c->shares = is_prefix ? prefix : p.shares - prefix;
  c->per_share = 1.0 / c->shares;
  return is_prefix;
}

// A share's partial results: slot 1 of the tile that starts in it, slot 0 of the one that it goes on with.
template <int D>
__device__ __forceinline__ float* joined_part(ParamsRef p, int head, int share, int slot) {  // (of a common prefix's passes)
  return p.parts + (((int64_t)head * p.shares + share) * 2 + slot) * (p.part_rows * (D + 4));
}
template <int BM, int D>
__device__ __forceinline__ float* part_of(ParamsRef p, int head, int share, int slot) {
  return p.parts + (((int64_t)head * p.shares + share) * 2 + slot) * (BM * (D + 4));
}

// Where element (row x, dim d) of a partial result lies. 128-row tiles keep the accumulators' layout, four dims a lane
// and 64 lanes side by side, so that a wave's stores and loads are whole KiB; 32-row tiles, merged through LDS
// before, rows of dims. m, l and exact l of every row follow.
template <int GW, int D>
__device__ __forceinline__ int part_index(int x, int d) {
  if constexpr (GW == 1) return x * D + d;
  const int c = x & 31, db = d / 32, h = d / 16 & 1, g = d / 8 & 1, half = d / 4 & 1;
  return (x / 32) * 32 * D + ((2 * db + h) * 2 + half) * 256 + (32 * g + c) * 4 + (d & 3);
}

template <int BM, int D>
__device__ __forceinline__ int part_sums(int x) {
  return BM * D + x * 4;
}

// What the merge of the tile that ends in a share needs: the share it starts in (-1: none ends here, or it lies in
// this share alone), its first row in the sequence and its rows, the sequence's first token, its keys, and the shift of its
// causal mask.
struct alignas(16) Merge {
  int first, row0, rows, token, n_kv, shift;
};
__device__ __forceinline__ Merge* merge_of(ParamsRef p, int head, int share) {
  static_assert(sizeof(Merge) == kMergeBytes);
  return static_cast<Merge*>(p.merges) + (int64_t)head * p.shares + share;
}

}  // namespace fa2
