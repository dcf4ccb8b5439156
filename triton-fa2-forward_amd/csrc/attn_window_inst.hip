// attn_window_inst.hip - the instances of the windowed attention kernel for chunks beside single tokens of one (dtype,
// head_dim) pair, compiled once per pair (FA2_DT, FA2_D).
#include "attn_ragged.hpp"

namespace fa2 {

namespace {

template <int SRC>
int launch_form(const RaggedParams& p, unsigned grid, hipStream_t s) {
  if (p.lse)
    hipLaunchKernelGGL((attn_window_mixed_kernel<FA2_DT, FA2_D, SRC, true>), dim3(grid), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((attn_window_mixed_kernel<FA2_DT, FA2_D, SRC, false>), dim3(grid), dim3(256), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    hipLaunchKernelGGL((attn_ragged_combine_kernel<FA2_DT, FA2_D, 4>), dim3((unsigned)(p.h_kv * p.shares) * 4),
                       dim3(combine_threads(FA2_D)), 0, s, p);
    e = hipGetLastError();
  }
  return (int)e;
}

}  // namespace

template <>
int launch_window_mixed<FA2_DT, FA2_D>(const RaggedParams& p, int source, unsigned grid, hipStream_t s) {
  return source == kSourcePages ? launch_form<kSourcePages>(p, grid, s) : launch_form<kSourceE4m3>(p, grid, s);
}

}  // namespace fa2
