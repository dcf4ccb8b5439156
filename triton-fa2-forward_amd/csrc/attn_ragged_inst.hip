// attn_ragged_inst.hip - the ragged attention kernel's instances of one (dtype, head_dim) pair, compiled
// once per pair (FA2_DT, FA2_D).
#include "attn_ragged.hpp"

namespace fa2 {

namespace {

template <int SRC, int GW>
int launch_form(const RaggedParams& p, unsigned grid, hipStream_t s) {
  if (GW > 1 && p.lse)
    hipLaunchKernelGGL((attn_ragged_kernel<FA2_DT, FA2_D, SRC, GW, (GW > 1)>), dim3(grid), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((attn_ragged_kernel<FA2_DT, FA2_D, SRC, GW, false>), dim3(grid), dim3(256), 0, s, p);
  hipError_t e = hipGetLastError();
  if constexpr (SRC != kSourcePacked) {
    if (e == hipSuccess && p.shares > 0) {
      hipLaunchKernelGGL((attn_ragged_combine_kernel<FA2_DT, FA2_D, GW>), dim3(grid * GW), dim3(combine_threads(FA2_D)), 0, s, p);
      e = hipGetLastError();
    }
  }
  return (int)e;
}

}  // namespace

template <>
int launch_ragged<FA2_DT, FA2_D>(const RaggedParams& p, int source, int row_waves, unsigned grid, hipStream_t s) {
  if (row_waves == 1) {
    switch (source) {
      case kSourcePacked: return launch_form<kSourcePacked, 1>(p, grid, s);
      case kSourcePages: return launch_form<kSourcePages, 1>(p, grid, s);
      default: return launch_form<kSourceE4m3, 1>(p, grid, s);
    }
  }
  switch (source) {
    case kSourcePacked: return launch_form<kSourcePacked, 4>(p, grid, s);
    case kSourcePages: return launch_form<kSourcePages, 4>(p, grid, s);
    default: return launch_form<kSourceE4m3, 4>(p, grid, s);
  }
}

}  // namespace fa2
