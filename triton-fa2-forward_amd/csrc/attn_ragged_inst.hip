// attn_ragged_inst.hip - the ragged attention kernel's instances of one (dtype, head_dim) pair, compiled
// once per pair (FA2_DT, FA2_D).
#include "attn_ragged.hpp"

namespace fa2 {

template <int DT, int D>
int launch_ragged(const RaggedParams& p, int source, unsigned grid, hipStream_t s) {
  switch (source) {
    case kSourcePacked:
      hipLaunchKernelGGL((attn_ragged_kernel<DT, D, kSourcePacked>), dim3(grid), dim3(256), 0, s, p);
      break;
    case kSourcePages:
      hipLaunchKernelGGL((attn_ragged_kernel<DT, D, kSourcePages>), dim3(grid), dim3(256), 0, s, p);
      break;
    default:
      hipLaunchKernelGGL((attn_ragged_kernel<DT, D, kSourceE4m3>), dim3(grid), dim3(256), 0, s, p);
  }
  return (int)hipGetLastError();
}

template int launch_ragged<FA2_DT, FA2_D>(const RaggedParams&, int, unsigned, hipStream_t);

}  // namespace fa2
