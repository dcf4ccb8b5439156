// attn_shared_inst.hip - the instances of the attention kernel for batches with a common prefix of one (dtype, head_dim) pair,
// compiled once per pair (FA2_DT, FA2_D).
#include "attn_ragged.hpp"

namespace fa2 {

namespace {

template <int SRC, int GWP, int GWO>
int launch_form(const RaggedParams& p, unsigned grid, hipStream_t s) {
  if (GWP > 1 && p.lse)
    hipLaunchKernelGGL((attn_shared_kernel<FA2_DT, FA2_D, SRC, GWP, GWO, (GWP > 1)>), dim3(grid), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((attn_shared_kernel<FA2_DT, FA2_D, SRC, GWP, GWO, false>), dim3(grid), dim3(256), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    hipLaunchKernelGGL((attn_shared_join_kernel<FA2_DT, FA2_D, GWP, GWO>), dim3((unsigned)shared_join_grid(p)), dim3(1024), 0, s, p);
    e = hipGetLastError();
  }
  return (int)e;
}

template <int SRC>
int launch_source(const RaggedParams& p, int prefix_waves, int own_waves, unsigned grid, hipStream_t s) {
  if (prefix_waves == 1) return launch_form<SRC, 1, 1>(p, grid, s);
  return own_waves == 1 ? launch_form<SRC, 4, 1>(p, grid, s) : launch_form<SRC, 4, 4>(p, grid, s);
}

}  // namespace

template <>
int launch_shared<FA2_DT, FA2_D>(const RaggedParams& p, int source, int prefix_waves, int own_waves, unsigned grid, hipStream_t s) {
  return source == kSourcePages ? launch_source<kSourcePages>(p, prefix_waves, own_waves, grid, s)
                                : launch_source<kSourceE4m3>(p, prefix_waves, own_waves, grid, s);
}

}  // namespace fa2
