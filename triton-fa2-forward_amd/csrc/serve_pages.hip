// serve_pages.hip - the pages of a step, on the GPU from the sequences' lengths: new tokens' pages taken from the free
// ones and entered into the block table, with the step's row starts, lengths, positions and slots; pages given back.
//
// A sequence of l tokens that gets n more needs the entries ceil(l / P) .. ceil((l + n) / P) - 1 of its row of the table. With
// N(s) the needs of the sequences before s and N the sum of all, need i of sequence s takes the free page at
// max(count - N, 0) + N(s) + i of the stack: the N topmost, in order; where fewer are free, the last needs get none (-1).
//
// The arrays are small, and a call is bound by its launches and by chains of loads. So every workgroup sums the lengths for
// itself (the results go to memory of their own, and nothing waits for another workgroup): 256 sequences each,
// and of their tokens and entries a stripe, found by a search over their starts in LDS.
// Measured on MI355X: 256 sequences of one new token 4.2 us, 50 of up to 2048 6.7.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "serve_launch.hpp"

namespace fa2 {

namespace {

// Sums over 64 lanes up to this one
__device__ __forceinline__ int64_t scan64(int64_t x, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int64_t y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  return x;
}

struct Need {
  int64_t held, want, fresh;  // entries that a sequence has and that it will have, its new tokens
};
__device__ __forceinline__ Need need_of(const PagesParams& p, int s) {
  Need n = {0, 0, 0};
  if (s >= p.n_seq) return n;
  const int64_t len = max(p.lens[s], 0), most = p.max_pages, up = (1 << p.page_shift) - 1;
  n.fresh = max(p.fresh[s], 0);
  n.held = min((len + up) >> p.page_shift, most);
  n.want = min((len + n.fresh + up) >> p.page_shift, most);
  return n;
}

// The last of 256 ascending starts that is at most x
__device__ __forceinline__ int last_start(const int64_t* starts, int64_t x) {
  int lo = 0;
#pragma unroll
  for (int step = 128; step >= 1; step /= 2)
    if (starts[lo + step] <= x) lo += step;
  return lo;
}

__global__ __launch_bounds__(256) void pages_extend_kernel(const PagesParams p) {
  __shared__ int64_t starts[257], needs[257];  // the block's sequences' first row and first need
  __shared__ int64_t waves[4][6];
  __shared__ int32_t held_of[256], old_of[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int block = (int)blockIdx.x, stripe = (int)blockIdx.y, stripes = (int)gridDim.y;
  const int s0 = block * 256, s = s0 + tid;
  const int stack = p.count[0];  // (on its way with the lengths)
  // ---- tokens and needs before the block's, of the block, and behind it
  int64_t sums[4] = {0, 0, 0, 0};  // tokens before, needs before, tokens in all, needs in all
  for (int i = tid; i < p.n_seq; i += 256) {
    const Need n = need_of(p, i);
    if (i < s0) {
      sums[0] += n.fresh;
      sums[1] += n.want - n.held;
    }
    sums[2] += n.fresh;
    sums[3] += n.want - n.held;
  }
  const Need mine = need_of(p, s);
  const int64_t upto = scan64(mine.fresh, lane), needs_upto = scan64(mine.want - mine.held, lane);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int off = 32; off >= 1; off /= 2) sums[i] += __shfl_xor(sums[i], off, 64);
  if (lane == 63) {
#pragma unroll
    for (int i = 0; i < 4; ++i) waves[wave][i] = sums[i];
    waves[wave][4] = upto;
    waves[wave][5] = needs_upto;
  }
  __syncthreads();
  int64_t start = 0, need = 0, tokens = 0, total = 0, end = 0, need_end = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    start += waves[w][0];
    need += waves[w][1];
    tokens += waves[w][2];
    total += waves[w][3];
  }
  const int64_t start0 = start, need0 = need;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    end += waves[w][4];
    need_end += waves[w][5];
    if (w < wave) {
      start += waves[w][4];
      need += waves[w][5];
    }
  }
  end += start0;
  need_end += need0;
  start += upto;
  need += needs_upto;
  const int old = s < p.n_seq ? max(p.lens[s], 0) : 0;
  starts[tid + 1] = start;
  needs[tid + 1] = need;
  if (tid == 0) {
    starts[0] = start0;
    needs[0] = need0;
  }
  held_of[tid] = (int)mine.held;
  old_of[tid] = old;
  const int64_t count = min(max(stack, 0), p.n_pages), base = max(count - total, (int64_t)0);
  auto clamp = [](int64_t x) { return (int32_t)min(x, (int64_t)0x7fffffff); };
  if (stripe == 0) {
    if (s < p.n_seq) {
      p.cu_out[s + 1] = clamp(start);
      p.lens_out[s] = clamp(old + mine.fresh);
    }
    if (block == 0 && tid == 0) {
      p.cu_out[0] = 0;
      p.count_out[0] = (int32_t)base;
    }
  }
  __syncthreads();
  auto free_page = [&](int64_t n) { return base + n < count ? p.free_pages[base + n] : -1; };
  // ---- entries of the table
  for (int64_t n = need0 + stripe * 256 + tid; n < need_end; n += (int64_t)stripes * 256) {
    const int q = last_start(needs, n);
    p.table[(s0 + q) * p.table_stride + held_of[q] + (n - needs[q])] = free_page(n);
  }
  // ---- rows, and behind the last sequence's those of none
  const int64_t rows = min(end, (int64_t)p.n_tokens);
  for (int64_t t = start0 + stripe * 256 + tid; t < rows; t += (int64_t)stripes * 256) {
    const int q = last_start(starts, t);
    const int64_t pos = old_of[q] + (t - starts[q]), entry = pos >> p.page_shift;
    int page = -1;
    if (entry < held_of[q])
      page = p.table[(s0 + q) * p.table_stride + entry];
    else if (entry < p.max_pages)
      page = free_page(needs[q] + entry - held_of[q]);
    p.positions[t] = clamp(pos);
    p.slots[t] = (unsigned)page < (unsigned)p.n_pages
                     ? ((int64_t)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1)) : -1;
  }
  if (block == (int)gridDim.x - 1)
    for (int64_t t = tokens + stripe * 256 + tid; t < p.n_tokens; t += (int64_t)stripes * 256) {
      p.positions[t] = -1;
      p.slots[t] = -1;
    }
}

// ---- pages given back: entries first[s] .. last[s] - 1 of every sequence that are pages go on top of the free ones

struct Range {
  int first, last;
};
__device__ __forceinline__ Range range_of(const ReleaseParams& p, int s) {
  return Range{max(p.first[s], 0), min(p.last[s], p.max_pages)};
}

// The range's pages in their order to free_pages[at ..], by a wave; where the next one's go. More than the pool holds are dropped.
__device__ __forceinline__ int64_t push_pages(const ReleaseParams& p, int s, const Range& r, int lane, int64_t at) {
  constexpr int STEP = 4;
  for (int64_t i0 = r.first; i0 < r.last; i0 += 64 * STEP) {
    int page[STEP];
#pragma unroll
    for (int u = 0; u < STEP; ++u)  // (no branch around a load: they are all on their way together)
      page[u] = p.table[s * p.table_stride + min(i0 + 64 * u + lane, (int64_t)r.last - 1)];
#pragma unroll
    for (int u = 0; u < STEP; ++u) {
      const bool is_page = i0 + 64 * u + lane < r.last && (unsigned)page[u] < (unsigned)p.n_pages;
      const uint64_t pages = __builtin_amdgcn_ballot_w64(is_page);
      const int64_t to = at + __builtin_popcountll(pages & ((1ull << lane) - 1));
      if (is_page && to < p.n_pages) p.free_pages[to] = page[u];
      at += __builtin_popcountll(pages);
    }
  }
  return at;
}

// A wave a sequence: how many
__global__ __launch_bounds__(256) void pages_count_kernel(const ReleaseParams p) {
  const int s = (int)(blockIdx.x * 4 + threadIdx.x / 64), lane = threadIdx.x & 63;
  if (s == 0 && lane == 0) p.counts[p.n_seq] = min(max(p.count[0], 0), p.n_pages);
  if (s >= p.n_seq) return;
  const Range r = range_of(p, s);
  int n = 0;
  for (int64_t i = (int64_t)r.first + lane; i < r.last; i += 64)
    n += (unsigned)p.table[s * p.table_stride + i] < (unsigned)p.n_pages;
#pragma unroll
  for (int off = 32; off >= 1; off /= 2) n += __shfl_xor(n, off, 64);
  if (lane == 0) p.counts[s] = n;
}

// ... and where: behind those of the sequences before
__global__ __launch_bounds__(256) void pages_release_kernel(const ReleaseParams p) {
  const int s = (int)(blockIdx.x * 4 + threadIdx.x / 64), lane = threadIdx.x & 63;
  if (s >= p.n_seq) return;
  int64_t at = 0;
  for (int i = lane; i < s; i += 64) at += p.counts[i];
#pragma unroll
  for (int off = 32; off >= 1; off /= 2) at += __shfl_xor(at, off, 64);
  at += p.counts[p.n_seq];
  const Range r = range_of(p, s);
  at = push_pages(p, s, r, lane, at);
  if (s == p.n_seq - 1 && lane == 0) p.count_out[0] = (int32_t)min(at, (int64_t)p.n_pages);
}

// Both in one launch, where few rounds count what lies before the last sequences (one_release): a wave a sequence, 16 a workgroup,
// which counts the pages of all sequences before its own for itself, 16 lanes a sequence and 16 entries a lane at once.
template <int LANES, int STEP>
__device__ __forceinline__ int count_pages(const ReleaseParams& p, int s, const Range& r, int lane) {
  int n = 0;
  for (int64_t i0 = r.first; i0 < r.last; i0 += LANES * STEP) {
    int page[STEP];
#pragma unroll
    for (int u = 0; u < STEP; ++u)
      page[u] = p.table[s * p.table_stride + min(i0 + u * LANES + lane, (int64_t)r.last - 1)];
#pragma unroll
    for (int u = 0; u < STEP; ++u) n += i0 + u * LANES + lane < r.last && (unsigned)page[u] < (unsigned)p.n_pages;
  }
  return n;
}
__global__ __launch_bounds__(1024) void pages_release_once_kernel(const ReleaseParams p) {
  __shared__ int before[16], own[16];  // pages that a wave has counted
  const int lane = threadIdx.x & 63, wave = (int)(threadIdx.x >> 6);
  const int s0 = (int)blockIdx.x * 16, s = s0 + wave;
  const int stack = p.count[0];
  const Range r = s < p.n_seq ? range_of(p, s) : Range{0, 0};
  int n = 0;
  Range next = range_of(p, min((int)(threadIdx.x >> 4), p.n_seq - 1));
  for (int t = (int)(threadIdx.x >> 4); t < s0; t += 64) {
    const Range now = next;
    next = range_of(p, min(t + 64, p.n_seq - 1));
    n += count_pages<16, 16>(p, t, now, lane & 15);
  }
  int mine = count_pages<64, 4>(p, s, r, lane);
#pragma unroll
  for (int off = 32; off >= 1; off /= 2) {
    n += __shfl_xor(n, off, 64);
    mine += __shfl_xor(mine, off, 64);
  }
  if (lane == 0) {
    before[wave] = n;
    own[wave] = mine;
  }
  __syncthreads();
  int64_t at = min(max(stack, 0), p.n_pages);
  for (int w = 0; w < 16; ++w) at += before[w] + (w < wave ? own[w] : 0);
  at = push_pages(p, s, r, lane, at);
  if (s == p.n_seq - 1 && lane == 0) p.count_out[0] = (int32_t)min(at, (int64_t)p.n_pages);
}

// One launch while the last workgroup counts the others' pages in at most 8 rounds of 64 sequences and 256 entries, which all wait for
// their loads. Each workgroup counts for itself, so that the time grows with the square of the sequences; what it saves is a launch,
// about 2.5 us of the host. Measured on MI355X, one launch and two, with a 32nd of the sequences or all of them ended, in a captured
// graph: 16 sequences of up to 4096 pages (no rounds) 12.9 and 18.3, 18.1 and 20.2 us; 128 of 256 (2) 4.3 and 5.0, 5.9 and 5.5; 256 of
// 64 (4) 5.9 and 5.0, 8.4 and 5.6; 256 of 512 (8) 8.6 and 6.3, 13.3 and 6.7 - made call after call with an extension behind it, where
// the host is what counts, 12.8 and 15.4 -; 512 of 512 (16) 14.8 and 7.1, 22 and 7.9; 1024 of 4 (16) 15 and 8.3, 23 and 8.9; 16384 of
// 4 470 and 65, 775 and 67.
constexpr int64_t kOneReleaseRounds = 8;
bool one_release(const ReleaseParams& p) {
  const int64_t before = (p.n_seq - 1) / 16 * 16, entries = std::max(p.max_pages, 1);
  return (before + 63) / 64 * ((entries + 255) / 256) <= kOneReleaseRounds;
}

}  // namespace

int launch_pages_extend(const PagesParams& p, unsigned blocks, unsigned stripes, hipStream_t s) {
  hipLaunchKernelGGL(pages_extend_kernel, dim3(blocks, stripes), dim3(256), 0, s, p);
  return (int)hipGetLastError();
}

int launch_pages_release(const ReleaseParams& p, hipStream_t s) {
  if (one_release(p)) {
    hipLaunchKernelGGL(pages_release_once_kernel, dim3((unsigned)((p.n_seq + 15) / 16)), dim3(1024), 0, s, p);
    return (int)hipGetLastError();
  }
  const unsigned grid = (unsigned)(((int64_t)p.n_seq + 3) / 4);
  hipLaunchKernelGGL(pages_count_kernel, dim3(grid), dim3(256), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(pages_release_kernel, dim3(grid), dim3(256), 0, s, p);
  return (int)hipGetLastError();
}

}  // namespace fa2
