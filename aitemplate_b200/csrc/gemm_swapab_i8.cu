// Instantiations of the weight-streaming GEMM for 8-bit integer operands (see gemm_swapab.cuh).
#include "gemm_swapab.cuh"

namespace b200ait {
template <int MX, int R, int H>
void launch_swapab_i8(bool bf16, const CUtensorMap& tw, const CUtensorMap& tx, const GemmParams& p, int num_slabs,
                      int num_groups, cudaStream_t stream) {
  if (bf16)
    launch_swapab<true, MX, R, H, true>(tw, tx, p, num_slabs, num_groups, stream);
  else
    launch_swapab<false, MX, R, H, true>(tw, tx, p, num_slabs, num_groups, stream);
}
#define B200AIT_SWAP(MX, R, H)                                                                                       \
  template void launch_swapab_i8<MX, R, H>(bool, const CUtensorMap&, const CUtensorMap&, const GemmParams&, int, int, \
                                           cudaStream_t);
B200AIT_FOR_EACH_SWAP_KERNEL(B200AIT_SWAP)
#undef B200AIT_SWAP
}  // namespace b200ait
