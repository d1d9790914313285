// Which instantiation of the tcgen05 GEMM kernel takes a launch with 8-bit integer operands: the same choice as for 16-bit operands
// (gemm_bn<BN>.cu, gemm_pair256.cu), without the forms that such a launch never has (row-major B, several destinations, permuted
// batches, alpha, split K).
#pragma once
#include "gemm_kernel.cuh"

namespace b200ait {

template <int BN, bool BF16>
static void launch_i8_width(const CUtensorMap& ta, const CUtensorMap& tb, const OutMaps& tout, const GemmParams& p, int grid,
                            cudaStream_t stream) {
  const bool residual = epi_b1(p.epilogue) != kBinaryNone, one_residual = residual && epi_b2(p.epilogue) == kBinaryNone;
  if ((BN < 128 ? p.vec_ok == 0 : p.tma_store == 0) && gemm_rows_output(p.N, BN, one_residual)) {
    launch_tc<BN, BF16, kRowsEpilogue, false, false, true>(ta, tb, tout, p, grid, stream);
    return;
  }
  // the kernels of one activation are lean on wide tiles: staged store, no residual (a residual comes by TMA on CTA pairs alone)
  if (BN >= 128 && p.tma_store != 0 && !residual) {
    switch (p.epilogue) {
#define B200AIT_CASE(U)                                                                                             \
  case make_epilogue(U, kBinaryNone, kBinaryNone, kUnaryIdentity):                                                  \
    launch_tc<BN, BF16, (BN >= 128 ? make_epilogue(U, kBinaryNone, kBinaryNone, kUnaryIdentity) : -1), false, false, \
              true>(ta, tb, tout, p, grid, stream);                                                                 \
    return;
      B200AIT_CASE(kUnaryIdentity)
      B200AIT_CASE(kUnaryRelu)
      B200AIT_CASE(kUnaryGelu)
      B200AIT_CASE(kUnaryFastGelu)
#undef B200AIT_CASE
    }
  }
  launch_tc<BN, BF16, -1, false, false, true>(ta, tb, tout, p, grid, stream);
}

template <bool BF16>
static void launch_i8(int width, const CUtensorMap& ta, const CUtensorMap& tb, const OutMaps& tout, const CUtensorMap& td0,
                      const GemmParams& p, int grid, cudaStream_t stream) {
  if (width == 64) return launch_i8_width<64, BF16>(ta, tb, tout, p, grid, stream);
  if (width == 128) return launch_i8_width<128, BF16>(ta, tb, tout, p, grid, stream);
  if (width == 256) return launch_i8_width<256, BF16>(ta, tb, tout, p, grid, stream);
  const bool residual = epi_b1(p.epilogue) != kBinaryNone;
  if (p.tma_store == 0 && gemm_rows_output(p.N, 256, residual && epi_b2(p.epilogue) == kBinaryNone)) {
    launch_tc_pair<256, BF16, kRowsEpilogue, false, false, true>(ta, tb, tout, td0, p, grid, stream);
    return;
  }
  if (p.tma_store != 0 && (!residual || p.tma_d0 != 0)) {
    switch (p.epilogue) {
#define B200AIT_CASE(CODE)                                                                    \
  case (CODE):                                                                                \
    launch_tc_pair<256, BF16, (CODE), false, false, true>(ta, tb, tout, td0, p, grid, stream); \
    return;
      B200AIT_FOR_EACH_FAST_EPILOGUE(B200AIT_CASE)
#undef B200AIT_CASE
    }
  }
  launch_tc_pair<256, BF16, -1, false, false, true>(ta, tb, tout, td0, p, grid, stream);
}

}  // namespace b200ait
