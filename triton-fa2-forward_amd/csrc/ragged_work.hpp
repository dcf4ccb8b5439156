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
//     16 of 512 78 and 65; 64 of 128 77 and 46, of 1024 1012 and 689.
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

// Keys that a tile costs beside its own: its rows' loads, its merge and stores. Measured on MI355X, in keys of cost
// 64 / 128 / 256 / 384: 4 prompts of 2000 in 128-row tiles (a share of short tiles alone holds many of them)
// 201 / 185 / 164 / 166 us; steps of 64 sequences of 1000 keys in 32-row tiles 46.5 / 47.8 / 48.0 / 49.0.
template <int BM>
constexpr int kTileCost = BM == 32 ? 64 : 256;
// ... and what sharing the tiles out costs a 128-row workgroup: more pieces, the partial results, their merge
constexpr int kShareCost = 640;
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
template <int BM>
__device__ __forceinline__ Lengths lengths_of(ParamsRef p, int n_q, int n_kv) {
  if (!p.causal) return Lengths{(int64_t)n_kv + kTileCost<BM>, 0};
  const int64_t slope = BM / p.group;
  return Lengths{(int64_t)max(n_kv - n_q, 0) + slope + kTileCost<BM>, slope};
}

__device__ __forceinline__ int64_t wave_scan(int64_t x, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int64_t y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  return x;
}
__device__ __forceinline__ int64_t readlane64(int64_t x, int l) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, l);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)x >> 32), l);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// A place among the sequences: the block of 64 that starts at s0 is in `lanes`, the sequence is its lane l.
struct Cursor {
  int s0, l, tile;
  LaneSequence lanes;
};

// The rank-th row tile; false: there are fewer.
template <int BM, bool PAGES>
__device__ __forceinline__ bool find_tile(ParamsRef p, int rank, int lane, Cursor* c) {
  c->lanes = lane_sequence<PAGES>(p, lane);
  if (p.seq.n_seq <= kFewSequences) {
    // Tiles of index t and above, over all sequences: A(t) = sum_s max(tiles_s - t, 0). The rank-th tile in the
    // order of falling t has the largest t with A(t) > rank; every lane tries a t of its own.
    const int tiles = row_tiles<BM>(c->lanes.n_q, p.group);
    int hi = 0;
    for (int s = 0; s < p.seq.n_seq; ++s) hi = max(hi, __builtin_amdgcn_readlane(tiles, s));
    auto above = [&](int t) {
      int a = 0;
      for (int s = 0; s < p.seq.n_seq; ++s) a += max(__builtin_amdgcn_readlane(tiles, s) - t, 0);
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
  for (int s0 = 0; s0 < p.seq.n_seq; s0 += 64) {
    if (s0) c->lanes = lane_sequence<PAGES>(p, s0 + lane);
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
#pragma unroll
  for (int off = 32; off >= 1; off /= 2) x = max(x, (int64_t)__shfl_xor(x, off, 64));
  return readlane64(x, 0);  // (a scalar: what is chosen by it stays one too)
}

// Whether a tile per workgroup takes no longer than equal shares, as estimated: as many tiles as workgroups at most, whose
// longest costs no more than a share and what sharing costs. With one workgroup a CU, half of those that
// fit, a key takes 5/8 of the time. Measured on MI355X (32 / 8 heads of 128), whole tiles and shares: 4 prompts of 500
// 25 and 41 us; a chunk of 500 behind 500 33 and 40, behind 2k 62 and 53; 4 of 500 behind 4k 146 and 161.
__device__ __forceinline__ bool whole_tiles(ParamsRef p, int64_t tiles, int64_t total, int64_t longest) {
  if (tiles > p.shares) return false;
  return (2 * tiles <= p.shares ? 5 * longest / 8 : longest) <= (int64_t)((double)total * p.per_share) + kShareCost;
}

// Share j: [x, end) of the line, the cursor at the tile that x lies in, `in` from its start; x >= end: nothing.
// With whole_tiles, the j-th tile.
struct Share {
  int64_t x, end, in, size;
};
template <int BM, bool PAGES>
__device__ __forceinline__ Share find_share(ParamsRef p, int j, int lane, Cursor* c) {
  auto length = [&]() {
    return lengths_of<BM>(p, c->lanes.n_q, c->lanes.n_kv).before(row_tiles<BM>(c->lanes.n_q, p.group));
  };
  c->lanes = lane_sequence<PAGES>(p, lane);
  c->s0 = 0;
  int64_t mine = length();
  int64_t upto = wave_scan(mine, lane);
  int64_t total = readlane64(upto, 63);
  for (int s0 = 64; s0 < p.seq.n_seq; s0 += 64) {
    c->lanes = lane_sequence<PAGES>(p, s0 + lane);
    total += readlane64(wave_scan(length(), lane), 63);
  }
  Share w;
  // (the same for every workgroup; how it is rounded does not matter, as long as shares * size reaches the total)
  w.size = max((int64_t)((double)total * p.per_share) + 1, (int64_t)kLeastShare);
  w.x = w.size * j;
  w.end = min(w.x + w.size, total);
  w.in = 0;
  if (BM != 32 && p.seq.n_seq <= 64) {
    const Lengths len = lengths_of<BM>(p, c->lanes.n_q, c->lanes.n_kv);
    const int64_t tiles = row_tiles<BM>(c->lanes.n_q, p.group), tiles_upto = wave_scan(tiles, lane);
    if (whole_tiles(p, readlane64(tiles_upto, 63), total, wave_max(tiles > 0 ? len.of(tiles - 1) : 0))) {
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
  if (p.seq.n_seq > 64) c->lanes = lane_sequence<PAGES>(p, lane);
  while (base + readlane64(upto, 63) <= w.x) {  // (w.x < total: ends within the sequences)
    base += readlane64(upto, 63);
    c->s0 += 64;
    if (c->s0 >= p.seq.n_seq) {  // only if the lengths changed since they were summed
      w.end = w.x;
      return w;
    }
    c->lanes = lane_sequence<PAGES>(p, c->s0 + lane);
    mine = length();
    upto = wave_scan(mine, lane);
  }
  c->l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(base + upto > w.x));
  w.in = w.x - base - readlane64(upto - mine, c->l);
  const LaneSequence q = sequence_at(c->lanes, c->l);
  const Lengths len = lengths_of<BM>(p, q.n_q, q.n_kv);
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
template <int BM, bool PAGES>
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
    if (c->s0 + 64 >= p.seq.n_seq) return false;
    c->s0 += 64;
    c->l = -1;
    c->lanes = lane_sequence<PAGES>(p, c->s0 + lane);
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

// A share's partial results: slot 1 of the tile that starts in it, slot 0 of the one that it goes on with.
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
