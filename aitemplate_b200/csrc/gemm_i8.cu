// Instantiations of the tcgen05 GEMM kernel for 8-bit integer operands and fp16 results (see gemm_kernel.cuh).
#include "gemm_i8.cuh"

namespace b200ait {
template <>
void launch_tc_i8<false>(int width, const CUtensorMap& ta, const CUtensorMap& tb, const OutMaps& tout, const CUtensorMap& td0,
                         const GemmParams& p, int grid, cudaStream_t stream) {
  launch_i8<false>(width, ta, tb, tout, td0, p, grid, stream);
}
}  // namespace b200ait
