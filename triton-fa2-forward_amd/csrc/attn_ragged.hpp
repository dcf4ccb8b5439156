// attn_ragged.hpp - attention of packed rows: sequences of different lengths back to back, with K and V
// in packed rows as well (source 0), in pages of 16-bit elements (1) or in pages of e4m3 (2).
//
//   O[r] = sum_n softmax_n(q_r . k_n * sm_scale) v_n over the keys n <= last(r) of the row's sequence,
//   last(r) = n_kv - 1, or with the causal mask n_kv - n_q + (the row's position): the last row sees the
//   last key. A row that sees no key gets O = 0 and a log-sum-exp of -inf.
//
// All query heads of a KV head share a workgroup's rows: row r of a sequence is position r / group, head
// r % group. Lengths are known on the device only, so the grid covers the most row tiles that n_tokens
// rows in n_seq sequences can have, and a workgroup finds its own (sequence, tile) by a scan of cu, 64
// sequences at a time; workgroups past the last tile exit.
//
// The tile arithmetic is attn_fwd_wavesplit.hpp's: 32 rows, S^T = K Q^T and O^T += V^T P^T with
// v_mfma_f32_32x32x16, P in registers, online softmax in base 2 with a lazily moved reference. Here the
// four waves of a workgroup take the key tiles of its 32 rows in turn, each through LDS buffers of its
// own, and merge once in LDS.
#pragma once

#include "attn_fwd_wavesplit.hpp"
#include "serve_common.hpp"
#include "serve_launch.hpp"

namespace fa2 {

// Keys per tile of one wave
constexpr int ragged_block_n(int head_dim) { return head_dim == 128 ? 32 : 64; }

// Sum over the lanes before and at this one
__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  return x;
}

// The rank-th row tile (BM rows of a KV head's group) of the sequences in order, wave-uniform; seq < 0: none
struct RowTile {
  int seq, tile;
};
template <int BM>
__device__ __forceinline__ RowTile find_row_tile(const int32_t* cu, int n_seq, int n_tokens, int group,
                                                 int rank, int lane) {
  int base = 0;
  for (int s0 = 0; s0 < n_seq; s0 += 64) {
    const int s = s0 + lane;
    int tiles = 0;
    if (s < n_seq) {
      const int rows = row_bound(cu, s + 1, n_tokens) - row_bound(cu, s, n_tokens);
      tiles = (max(rows, 0) * group + BM - 1) / BM;
    }
    const int upto = wave_scan(tiles, lane);
    const uint64_t past = __builtin_amdgcn_ballot_w64(base + upto > rank);
    if (past) {
      const int l = __builtin_ctzll(past);
      return RowTile{s0 + l, rank - base - __builtin_amdgcn_readlane(upto - tiles, l)};
    }
    base += __builtin_amdgcn_readlane(upto, 63);
  }
  return RowTile{-1, 0};
}

template <int DT, int D, int SRC>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(2)))
void attn_ragged_kernel(const RaggedParams p) {
  using E = Elem<DT>;
  constexpr bool kE4m3 = SRC == kSourceE4m3;
  constexpr bool kPages = SRC != kSourcePacked;
  constexpr int EB = kE4m3 ? 1 : 2;      // bytes of a cached element
  constexpr int BN = ragged_block_n(D);
  constexpr int KG = 4;                  // key groups: waves
  constexpr int KS = D / 16;             // 16-dim k-steps of S^T = K Q^T
  constexpr int DB = (D + 31) / 32;      // 32-dim row blocks of O^T
  constexpr int NB = BN / 32;            // 32-key row blocks of S^T
  constexpr int NT = BN / 16;            // 16-key k-steps of O^T
  constexpr int CPR = D / 8;             // 16-byte chunks per K / V row in LDS
  constexpr int TCH = BN * CPR;          // chunks per K (or V) tile
  constexpr int NI = TCH / 64 * EB / 2;  // 1 KiB loads per tile
  constexpr int RPI = BN / NI;           // rows of one load (one page: the host's rule on page sizes)
  static_assert(NI >= 1 && BN % NI == 0, "a tile must be whole 1 KiB loads");
  constexpr int QPR = D / 4;             // 16-byte pieces of an fp32 output row

  constexpr int kKvChunks = KG * 2 * TCH;
  constexpr int kMergeChunks = KG * 32 * QPR;
  __shared__ u32x4 lds[kKvChunks > kMergeChunks ? kKvChunks : kMergeChunks];
  __shared__ float sm[KG][32][3];  // m, l, exact l of every wave's rows
  __shared__ int odd[32];          // rows whose sums are not finite

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int c = lane & 31;
  const int g = lane >> 5;

  // ---- which head and row tile: a KV head stays on one XCD where the heads split evenly over them, so
  // that its row tiles share K and V in one L2
  const int xcds = 1 << p.xcd_shift;
  int hkv, rank;
  if ((p.h_kv & (xcds - 1)) == 0) {
    const int per = p.h_kv >> p.xcd_shift, slot = (int)blockIdx.x >> p.xcd_shift;
    hkv = ((int)blockIdx.x & (xcds - 1)) * per + slot % per;
    rank = slot / per;
  } else {
    hkv = (int)blockIdx.x % p.h_kv;
    rank = (int)blockIdx.x / p.h_kv;
  }
  const RowTile rt = find_row_tile<32>(p.seq.cu, p.seq.n_seq, p.seq.n_tokens, p.group, rank, lane);
  if (rt.seq < 0) return;
  const int t_first = row_bound(p.seq.cu, rt.seq, p.seq.n_tokens);
  const int n_q = row_bound(p.seq.cu, rt.seq + 1, p.seq.n_tokens) - t_first;
  int n_kv, kv_first = 0;
  if constexpr (kPages) {
    n_kv = (int)min((int64_t)max(p.seq.lens[rt.seq], 0), (int64_t)p.seq.max_pages << p.seq.page_shift);
  } else {
    kv_first = row_bound(p.cu_kv, rt.seq, p.kv_tokens);
    n_kv = max(row_bound(p.cu_kv, rt.seq + 1, p.kv_tokens) - kv_first, 0);
  }
  const int rows = n_q * p.group;
  const int row0 = rt.tile * 32;  // this workgroup's rows [row0, row_end)
  const int row_end = min(row0 + 32, rows);
  const int shift = n_kv - n_q;   // causal: position i sees keys up to i + shift

  // ---- this lane's row; rows past the last repeat it and are never stored
  const int r = min(row0 + c, rows - 1);
  const int pos = r / p.group;
  u32x4 qreg[KS];
  {
    const int head = hkv * p.group + (r - pos * p.group);
    const uint16_t* qrow = p.q + (int64_t)(t_first + pos) * p.sqt + head * p.sqh + 8 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qreg[ks] = *(const u32x4*)(qrow + 16 * ks);
  }
  // the last key of a position, the end of the keys that some row sees, and of those that every row sees
  auto last_of = [&](int i) { return p.causal ? min(i + shift, n_kv - 1) : n_kv - 1; };
  const int last_key = last_of(pos);
  const int kv_end = max(last_of((row_end - 1) / p.group) + 1, 0);
  const int full_end = max(last_of(row0 / p.group) + 1, 0);

  // ---- this wave's tiles: wave, wave + KG, ...
  const int n_tiles = (kv_end + BN - 1) / BN;
  const int count = (n_tiles - wave + KG - 1) / KG;
  auto key_of = [&](int i) { return (wave + i * KG) * BN; };  // first key of tile i

  // ---- pages of the wave's tiles, a block of 64 table entries in a register: lane x holds the entry of
  // tile x / per_tile, page x % per_tile of the tile. An entry that is no page of the cache reads page 0
  // and makes the rows NaN.
  const int page_shift = p.seq.page_shift;
  const int tile_shift = kPages ? max(0, 31 - __builtin_clz(BN) - page_shift) : 0;  // log2 pages per tile
  int entries = 0, bad = 0;
  auto load_entries = [&](int i0) {
    const int i = i0 + (lane >> tile_shift);
    const int64_t n = (int64_t)(wave + (int64_t)i * KG) * BN + ((int64_t)(lane & ((1 << tile_shift) - 1)) << page_shift);
    int e = 0;
    if (i < count && n < kv_end) e = p.seq.table[rt.seq * p.seq.table_stride + (n >> page_shift)];
    if ((unsigned)e >= (unsigned)p.seq.n_pages) {
      bad = 1;
      e = 0;
    }
    return e;
  };
  // the page of tile i's row x (wave-uniform)
  auto page_of = [&](int i, int x) {
    return __builtin_amdgcn_readlane(entries, ((i << tile_shift) & 63) + (x >> page_shift));
  };

  // ---- K/V rows -> LDS (bf16 / fp16, XOR-swizzled 16-byte chunks as in attn_fwd_kernel.hpp)
  const CacheTensor* const tens[2] = {&p.kc, &p.vc};
  uint32_t off[2][NI];  // this lane's byte offset inside load j
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      if constexpr (kE4m3) {
        off[t][j] = (uint32_t)((lane / (D / 16)) * tens[t]->token + (lane % (D / 16)) * 16);
      } else {
        const int row = lane / CPR, col = lane % CPR, in_tile = j * RPI + row;
        const int key = t == 0 ? k_key<D>(pi_row(in_tile & 31) & 15) : v_key<D>(in_tile & 15);
        off[t][j] = (uint32_t)(row * tens[t]->token + (col ^ key) * 8) * 2u;
      }
    }
  // buffer resource of load j of tile i: the rows of it that lie before kv_end (others read as zeros)
  auto rows_at = [&](int t, int i, int j) {
    const int n0 = i < count ? key_of(i) + j * RPI : kv_end;
    const int valid = min(kv_end - n0, RPI);
    const CacheTensor& x = *tens[t];
    const uint32_t bytes = valid > 0 ? ((uint32_t)(valid - 1) * (uint32_t)x.token + (uint32_t)D) * EB : 0u;
    int64_t at = (int64_t)hkv * x.head;
    if constexpr (kPages)
      at += (int64_t)page_of(i, j * RPI) * x.page + (int64_t)(n0 & ((1 << page_shift) - 1)) * x.token;
    else
      at += (int64_t)(kv_first + n0) * x.token;
    return make_desc(x.data + (valid > 0 ? at * EB : 0), bytes);
  };
  const FA2_LDS char* kbuf = (const FA2_LDS char*)(lds + wave * 2 * TCH);
  const FA2_LDS char* vbuf = kbuf + TCH * 16;
  auto issue = [&](int t, int i) {
    const FA2_LDS char* buf = t == 0 ? kbuf : vbuf;
#pragma unroll
    for (int j = 0; j < NI; ++j) load_lds16(rows_at(t, i, j), off[t][j], lds_addr(buf + j * 1024));
  };
  // e4m3: through registers, converted on the way (16 values of one row a lane)
  struct Raw {
    u32x4 w[NI];
    uint32_t scale[NI];
  };
  auto fetch = [&](int t, int i, Raw& raw) {
    const CacheTensor& x = *tens[t];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int n0 = i < count ? key_of(i) + j * RPI : kv_end;
      const int row = lane / (D / 16);
      const bool ok = n0 + row < kv_end;
      raw.w[j] = u32x4{0u, 0u, 0u, 0u};
      raw.scale[j] = 0u;
      if (ok) {
        const int64_t page = page_of(i, j * RPI);
        const int in_page = (n0 & ((1 << page_shift) - 1)) + row;
        raw.w[j] = *(const u32x4*)(x.data + page * x.page + hkv * x.head + (int64_t)in_page * x.token +
                                   (lane % (D / 16)) * 16);
        raw.scale[j] = x.scale[page * x.scale_page + hkv * x.scale_head + (int64_t)in_page * x.scale_token];
      }
    }
  };
  auto store = [&](int t, const Raw& raw) {
    FA2_LDS char* buf = (FA2_LDS char*)(t == 0 ? kbuf : vbuf);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int row = j * RPI + lane / (D / 16), chunk = lane % (D / 16) * 2;
      const int key = t == 0 ? k_key<D>(pi_row(row & 31) & 15) : v_key<D>(row & 15);
      const float scale = e8m0_to_f32(raw.scale[j]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x2 lo = e4m3_to_16<DT>(raw.w[j][2 * h], scale), hi = e4m3_to_16<DT>(raw.w[j][2 * h + 1], scale);
        *(u32x4 FA2_LDS*)(buf + (row * CPR + ((chunk + h) ^ key)) * 16) = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    }
  };

  // ---- LDS operand reads, as in attn_fwd_kernel.hpp
  const int kk = k_key<D>(c & 15);
  const int vj = (lane & 15) >> 2;
  const int vq = lane & 3;
  const int vsig = ((vq & 1) << 1) | ((vq & 2) >> 1);
  const int vdh = (D == 16) ? 0 : ((lane >> 4) & 1);
  uint32_t koffs[KS], voffs[2][DB];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koffs[ks] = (uint32_t)((pi_row(c) * CPR + ((2 * ks + g) ^ kk)) * 16);
#pragma unroll
  for (int rr = 0; rr < 2; ++rr)
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int row = 8 * g + 4 * rr + vj;
      const int chunk = (4 * db + 2 * vdh + (vsig >> 1)) ^ v_key<D>(row);
      voffs[rr][db] = (uint32_t)(row * (D * 2) + chunk * 16 + (vsig & 1) * 8);
    }
  auto k_operand = [&](int ks, int nb) { return *(const u32x4 FA2_LDS*)(kbuf + koffs[ks] + nb * 32 * CPR * 16); };
  auto v_operand = [&](int t, int db) {
    const u32x2 lo = lds_read_tr(vbuf + voffs[0][db] + t * 16 * D * 2);
    const u32x2 hi = lds_read_tr(vbuf + voffs[1][db] + t * 16 * D * 2);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };

  // ---- the online softmax of one tile, base 2, with a lazily moved reference (attn_fwd_wavesplit.hpp)
  float m_i = -INFINITY, l_i = 0.f, l_exact = 0.f;
  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
  const float qk_scale = p.qk_scale;
  const bool want_exact = p.lse != nullptr;
  auto softmax = [&](f32x16 (&s)[NB], u32x4 (&pb)[NT], int n0) {
    if (n0 + BN > full_end) {
      const int lim = last_key - n0 - 8 * g;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (nb * 32 + 16 * (x / 8) + (x % 8) > lim) s[nb][x] = -INFINITY;
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
    // a row that has seen no key in this wave's tiles yet (reference -inf) gets weights 0, not NaN
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

  const int block = 64 >> tile_shift;  // tiles of one block of entries
  if constexpr (kPages) entries = load_entries(0);
  Raw kraw, vraw;
  if constexpr (kE4m3) {
    fetch(0, 0, kraw);
    fetch(1, 0, vraw);
  } else {
    issue(0, 0);
    issue(1, 0);
    // Q is waited for here: the compiler does not count the asm loads, so its own wait for Q is for
    // everything in flight, and inside the loop it would come every time
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qreg[ks]));
  }
  for (int i = 0; i < count; ++i) {
    if constexpr (kE4m3) store(0, kraw);
    else wait_vm_fence<NI>();  // K_i has landed; V_i may be in flight
    u32x4 kop[KS][NB];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) kop[ks][nb] = k_operand(ks, nb);
    if (kPages && ((i + 1) & (block - 1)) == 0) entries = load_entries(i + 1);
    if constexpr (kE4m3) {
      fetch(0, i + 1, kraw);
    } else {
      wait_lds_fence();  // the operands have left the buffer: refill it
      issue(0, i + 1);
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
    if constexpr (kE4m3) store(1, vraw);
    else wait_vm_fence<NI>();  // V_i has landed; K_{i+1} may be in flight
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] = E::mma(v_operand(t, db), pb[t], acc[db]);
    if constexpr (kE4m3) {
      fetch(1, i + 1, vraw);
    } else {
      wait_lds_fence();
      issue(1, i + 1);
    }
  }

  // ---- merge the waves through LDS: O^T blocks as 16-byte pieces [wave][row][4 dims]
  if (tid < 32) odd[tid] = 0;
  if constexpr (!kE4m3) wait_vm_fence<0>();
  __syncthreads();  // every wave is done with every K/V buffer
  FA2_LDS f32x4* ob = (FA2_LDS f32x4*)lds;
  auto piece = [&](int group, int row, int q) {
    return (group * 32 + row) * QPR + (q ^ (row & (QPR < 8 ? QPR - 1 : 7)));
  };
  if (__builtin_amdgcn_ballot_w64(bad != 0)) m_i = __uint_as_float(0x7fc00000u);
  {
    const float l = pair_sum(l_i);
    const float lx = want_exact ? pair_sum(l_exact) : l;
    // A weight of zero times an infinite or NaN value is NaN: such a value may lie in a key of the tile
    // that the row does not see. Rows whose sums are not finite are computed again below, over the keys
    // that they see alone.
    float test = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int x = 0; x < 16; ++x) test = __builtin_fmaf(acc[db][x], 0.f, test);
    if (row0 + c < row_end) {
      if (test != 0.f) odd[c] = 1;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int q = 8 * db + 4 * (h >> 1) + 2 * g + (h & 1);  // dims 4 q .. 4 q + 3
          if (q < QPR) {
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = acc[db][4 * h + e];
            ob[piece(wave, c, q)] = x;
          }
        }
      if (g == 0) {
        sm[wave][c][0] = m_i;
        sm[wave][c][1] = l;
        sm[wave][c][2] = lx;
      }
    }
  }
  __syncthreads();
  for (int t = tid; t < (row_end - row0) * QPR; t += 256) {
    const int wr = t / QPR, q = t % QPR;
    if (odd[wr]) continue;
    float m = -INFINITY, l = 0.f, lx = 0.f;
    bool nan = false;
#pragma unroll
    for (int x = 0; x < KG; ++x) {
      m = fmaxf(m, sm[x][wr][0]);
      nan |= sm[x][wr][0] != sm[x][wr][0];
    }
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < KG; ++x) {
      const float mw = sm[x][wr][0];
      const float w = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);
      l = __builtin_fmaf(w, sm[x][wr][1], l);
      lx = __builtin_fmaf(w, sm[x][wr][2], lx);
      const f32x4 v = ob[piece(x, wr, q)];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(w, v[e], o[e]);
    }
    if (nan) m = l = lx = __uint_as_float(0x7fc00000u);
    const int opos = (row0 + wr) / p.group;
    const int head = hkv * p.group + (row0 + wr - opos * p.group);
    const float inv_l = last_of(opos) < 0 && !nan ? 0.f : 1.0f / l;  // no key: 0
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv_l;
    uint16_t* orow = p.o + (int64_t)(t_first + opos) * p.sot + head * p.soh + 4 * q;
    *(u32x2*)orow = u32x2{E::pack2(o[0], o[1]), E::pack2(o[2], o[3])};
    if (p.lse && q == 0) p.lse[(int64_t)head * p.seq.n_tokens + t_first + opos] = (m + log2f(lx)) * kLn2;
  }

  // ---- rows with sums that are not finite, a wave per row in turn: 64 keys at a time, one a lane
  for (int wr = wave; wr < row_end - row0; wr += 4) {
    if (!odd[wr]) continue;
    const int opos = (row0 + wr) / p.group;
    const int head = hkv * p.group + (row0 + wr - opos * p.group);
    bool nan = false;
#pragma unroll
    for (int x = 0; x < KG; ++x) nan |= sm[x][wr][0] != sm[x][wr][0];
    const int end = nan ? 0 : last_of(opos) + 1;
    const uint16_t* qrow = p.q + (int64_t)(t_first + opos) * p.sqt + head * p.sqh;
    int page = 0;
    auto row_at = [&](const CacheTensor& x, int n) {
      if constexpr (kPages) {
        page = p.seq.table[rt.seq * p.seq.table_stride + (n >> page_shift)];
        if ((unsigned)page >= (unsigned)p.seq.n_pages) page = 0;
        return x.data + (page * x.page + hkv * x.head + (int64_t)(n & ((1 << page_shift) - 1)) * x.token) * EB;
      } else {
        return x.data + ((int64_t)(kv_first + n) * x.token + hkv * x.head) * EB;
      }
    };
    auto scale_at = [&](const CacheTensor& x, int n) {
      return e8m0_to_f32(x.scale[page * x.scale_page + hkv * x.scale_head +
                                 (int64_t)(n & ((1 << page_shift) - 1)) * x.scale_token]);
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
    float m = -INFINITY, l = 0.f, o[(D + 63) / 64] = {};
    for (int n0 = 0; n0 < end; n0 += 64) {
      const int n = n0 + lane;
      float s = -INFINITY;
      if (n < end) {
        const char* krow = row_at(p.kc, n);
        float scale = 1.f;
        if constexpr (kE4m3) scale = scale_at(p.kc, n);
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
      const float w = n < end ? __builtin_amdgcn_exp2f(s - m_ref) : 0.f;
      m = m_new;
      l = l * alpha + w;
#pragma unroll
      for (int x = 0; x < (D + 63) / 64; ++x) o[x] *= alpha;
      for (int y = 0; y < min(end - n0, 64); ++y) {
        const float wy = __shfl(w, y, 64);
        const char* vrow = row_at(p.vc, n0 + y);
        float scale = 1.f;
        if constexpr (kE4m3) scale = scale_at(p.vc, n0 + y);
#pragma unroll
        for (int x = 0; x < (D + 63) / 64; ++x)
          if (lane + 64 * x < D) o[x] = __builtin_fmaf(wy, value(vrow, scale, lane + 64 * x), o[x]);
      }
    }
#pragma unroll
    for (int o2 = 32; o2 >= 1; o2 /= 2) l += __shfl_xor(l, o2, 64);
    uint16_t* orow = p.o + (int64_t)(t_first + opos) * p.sot + head * p.soh;
#pragma unroll
    for (int x = 0; x < (D + 63) / 64; ++x)
      if (lane + 64 * x < D) orow[lane + 64 * x] = (uint16_t)E::pack2(nan ? l / l : end <= 0 ? 0.f : o[x] / l, 0.f);
    if (p.lse && lane == 0)
      p.lse[(int64_t)head * p.seq.n_tokens + t_first + opos] = no_lse ? l / l : m == INFINITY ? m : (m + log2f(l)) * kLn2;
  }
}

}  // namespace fa2
