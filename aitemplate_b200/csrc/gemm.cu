// gemm_rcr / bmm_rcr family for sm_100a: Y[b] = epilogue(alpha * X[b] . W[b]^T + bias, D0, D1)
// with X [M,K] and W [N,K] both K-contiguous ("RCR": row-major A, column-major B, row-major C).
//
// Replaces the reference's CUTLASS / CuTe-DSL template instantiation for
//   gemm_rcr            python/aitemplate/backend/cuda/gemm_universal/gemm_rcr.py:148-315
//   gemm_rcr_bias*      .../gemm_rcr_bias.py:39-61, common_bias_activation.py, common_bias_broadcast.py:86-128
//   gemm_rcr_bias_permute  .../gemm_rcr_bias_permute.py:55-95, common_permute.py:88-107
//   bmm_rcr             .../bmm_xxx.py:30-155, bmm_common.py:200-434
// by one persistent, warp-specialised kernel:
//   warp 0      TMA producer: cp.async.bulk.tensor loads of 128x64 (A) and BNx64 (B) tiles into a
//               128-byte-swizzled shared-memory ring guarded by full/empty mbarriers
//   warp 1      MMA issuer: tcgen05.mma (M=128, N=BN, K=16) into one of two TMEM
//               accumulators, tcgen05.commit releases smem stages / publishes the accumulator
//   warps 2-9   epilogue: tcgen05.ld of this warp's 32 TMEM lanes, bias / activation / residual in fp32, one
//               rounding, staged TMA or 16-byte global stores (row-major with stride, or permuted)
// The epilogue of tile i overlaps the main loop of tile i+1 (two accumulators).
// Shapes that TMA cannot address (K or a leading stride not a multiple of 8 elements, unaligned
// pointers) run on a plain tiled CUDA-core kernel in this file; there is no host fallback.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <vector>

#include "b200ait.h"
#include "gemm_swapab.cuh"

namespace b200ait {

// ------------------------------------------------------------------------------------------------
// split-K second pass: sums the fp32 partials of every split and applies the fused epilogue.
// One thread per (batch, row, 32-column chunk); a warp reads 4 KB of contiguous partials per split.
template <bool BF16>
__global__ void __launch_bounds__(256) gemm_splitk_reduce_kernel(const GemmParams p) {
  const int chunks = (p.N + 31) / 32;
  const long long total = static_cast<long long>(p.batch) * p.M * chunks;
  const long long idx = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (idx >= total) return;
  const int chunk = static_cast<int>(idx % chunks);
  const long long br = idx / chunks;
  const int row = static_cast<int>(br % p.M), b = static_cast<int>(br / p.M);
  const int col0 = chunk * 32;
  float v[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = 0.f;
  const bool full = p.vec_ok && col0 + 32 <= p.N;
  const long long split_stride = static_cast<long long>(p.batch) * p.M * p.N;
  int s0 = 0;
  if (full) {
    // two splits' 128 bytes per thread are requested before either is added: few threads run here when M is
    // small, so the pass is bound by how many loads each of them keeps in flight
    const float* base = p.partial + (static_cast<long long>(b) * p.M + row) * p.N + col0;
    for (; s0 + 1 < p.splits; s0 += 2) {
      float4 f[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 8; ++q) f[h][q] = __ldcs(reinterpret_cast<const float4*>(base + (s0 + h) * split_stride + q * 4));
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 8; ++q)
          v[q * 4] += f[h][q].x, v[q * 4 + 1] += f[h][q].y, v[q * 4 + 2] += f[h][q].z, v[q * 4 + 3] += f[h][q].w;
    }
  }
  for (int s = s0; s < p.splits; ++s) {
    const float* src = p.partial + ((static_cast<long long>(s) * p.batch + b) * p.M + row) * p.N + col0;
    if (full) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float4 f = *reinterpret_cast<const float4*>(src + q * 4);
        v[q * 4] += f.x, v[q * 4 + 1] += f.y, v[q * 4 + 2] += f.z, v[q * 4 + 3] += f.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col0 + j < p.N) v[j] += src[j];
    }
  }
  epilogue_chunk32<BF16>(p, v, b, row, col0, true);
}

// ------------------------------------------------------------------------------------------------
// CUDA-core kernel for shapes TMA cannot address. 32x32 output tile per block, K staged in smem.
template <bool BF16>
__global__ void __launch_bounds__(256) gemm_simt_kernel(const void* a_, const void* b_, const GemmParams p) {
  using E = Elem16<BF16>;
  using T = typename E::T;
  __shared__ float sa[32][33];
  __shared__ float sb[32][33];
  const int b = blockIdx.z;
  const T* a = static_cast<const T*>(a_) + static_cast<long long>(b) * p.a_bs * p.a_batch_mul;
  const T* w = static_cast<const T*>(b_) + static_cast<long long>(b) * p.b_bs * p.b_batch_mul;
  const long long w_n = p.b_mn ? 1 : p.ldb, w_k = p.b_mn ? p.ldb : 1;  // element strides of B along n and k
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;  // 32 x 8
  const int row0 = blockIdx.y * 32, col0 = blockIdx.x * 32;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < p.K; k0 += 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = ty + i * 8;
      const int k = k0 + tx;
      sa[r][tx] = (row0 + r < p.M && k < p.K) ? E::to_float(a[static_cast<long long>(row0 + r) * p.lda + k]) : 0.f;
      sb[r][tx] = (col0 + r < p.N && k < p.K) ? E::to_float(w[static_cast<long long>(col0 + r) * w_n + k * w_k]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 32; ++kk) {
      const float bv = sb[tx][kk];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(sa[ty + i * 8][kk], bv, acc[i]);
    }
    __syncthreads();
  }
  const int col = col0 + tx;
  if (col >= p.N) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + ty + i * 8;
    if (row < p.M) epilogue_scalar_store<BF16>(p, acc[i], b, row, col);
  }
}

// The same for 8-bit integers whose rows do not start on 16 bytes: 64 elements of K at a time, staged byte by byte as
// words of four, four products per instruction.
template <bool BF16>
__global__ void __launch_bounds__(256) gemm_simt_i8_kernel(const int8_t* a, const int8_t* w, const GemmParams p) {
  constexpr int kWords = 16;
  __shared__ int sa[32][kWords + 1];
  __shared__ int sb[32][kWords + 1];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;  // 32 x 8
  const int row0 = blockIdx.y * 32, col0 = blockIdx.x * 32;
  int acc[4] = {0, 0, 0, 0};
  for (int k0 = 0; k0 < p.K; k0 += 4 * kWords) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = threadIdx.x + 256 * i, r = e >> 6, kk = e & 63, k = k0 + kk;
      reinterpret_cast<int8_t*>(sa[r])[kk] = row0 + r < p.M && k < p.K ? a[static_cast<long long>(row0 + r) * p.lda + k] : int8_t{0};
      reinterpret_cast<int8_t*>(sb[r])[kk] = col0 + r < p.N && k < p.K ? w[static_cast<long long>(col0 + r) * p.ldb + k] : int8_t{0};
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kWords; ++q) {
      const int bv = sb[tx][q];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = __dp4a(sa[ty + i * 8][q], bv, acc[i]);
    }
    __syncthreads();
  }
  const int col = col0 + tx;
  if (col >= p.N) return;
  const float cs = p.col_scale[col];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + ty + i * 8;
    if (row < p.M) epilogue_scalar_store_i8<BF16>(p, scale_column_i8(acc[i], cs), p.row_scale[row], row, col);
  }
}

// ------------------------------------------------------------------------------------------------
// Weight-streaming kernel for M <= 4 (a GEMV per row of X): the run time is the time to read W once, and a
// handful of rows leaves nothing for the tensor core to amortise. One block of 32 warps per SM holds X in
// shared memory and owns a contiguous share of the rows of W; each warp streams one row at a time with
// 16-byte loads that do not allocate in L1 (8 in flight per lane), multiplies on the FMA pipe in fp32 and
// reduces across the lanes. No workspace, no second pass.
constexpr int kRowDotMaxM = 4;
constexpr int kRowDotThreads = 1024;
template <bool BF16, int MR>
__global__ void __launch_bounds__(kRowDotThreads, 1) gemm_rowdot_kernel(const void* a_, const void* b_,
                                                                         const GemmParams p) {
  using T = typename Elem16<BF16>::T;
  extern __shared__ __align__(16) uint8_t rowdot_smem[];
  uint4* xs = reinterpret_cast<uint4*>(rowdot_smem);  // [MR][K / 8]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  const int nvec = p.K >> 3;
  for (int i = threadIdx.x; i < MR * nvec; i += blockDim.x) {
    const int m = i / nvec, v = i - m * nvec;
    xs[i] = (m < p.M) ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a_) + static_cast<long long>(m) * p.lda) + v)
                      : make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  // rows [n_begin, n_end) of W belong to this block
  const int per = (p.N + gridDim.x - 1) / gridDim.x;
  const int n_begin = blockIdx.x * per, n_end = min(p.N, n_begin + per);
  constexpr int kUnroll = 8;
  for (int n = n_begin + warp; n < n_end; n += nwarps) {
    const uint4* w = reinterpret_cast<const uint4*>(static_cast<const T*>(b_) + static_cast<long long>(n) * p.ldb);
    float acc[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[m] = 0.f;
    for (int v0 = lane; v0 < nvec; v0 += 32 * kUnroll) {
      uint4 wq[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        wq[u] = (v0 + 32 * u < nvec) ? __ldcs(w + v0 + 32 * u) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int v = min(v0 + 32 * u, nvec - 1);  // past the end the weights above are zero
        float wf[8];
        unpack8<BF16>(wq[u], wf);
#pragma unroll
        for (int m = 0; m < MR; ++m) {
          float xf[8];
          unpack8<BF16>(xs[m * nvec + v], xf);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[m] = fmaf(xf[j], wf[j], acc[m]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      float t = acc[m];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      if (lane == m && m < p.M) epilogue_scalar_store<BF16>(p, t, 0, m, n);
    }
  }
}

// The same for K < 1024, where a row of W is so short that one row per warp leaves too little in flight and the
// launch's latencies are most of the time: a warp takes up to 8 / KV rows at once (KV 16-byte vectors per lane and row,
// eight loads in flight, four with M = 3 or 4 and K = 256), its first rows are on their way before the block stages X, and all its sums are reduced
// together. M = 1 .. 4 on the tile kernels -> here: K = 1016, N = 512: 8.2 -> 2.8 us, N = 3176: 10.6 -> 3.2 .. 4.0;
// K = 512, N = 3176: 8.2 -> 2.9 .. 4.7; K = 256, N = 100: 7.4 -> 2.6 .. 3.9.
constexpr int kRowDotShortThreads = 512;
template <bool BF16, int MR, int KV>
__global__ void __launch_bounds__(kRowDotShortThreads, 1) gemm_rowdot_short_kernel(const void* a_, const void* b_,
                                                                                   const GemmParams p) {
  using T = typename Elem16<BF16>::T;
  constexpr int kRows = MR == 4 && KV == 1 ? 4 : 8 / KV;  // (32 sums do not fit the registers beside the loads)
  __shared__ uint4 xs[MR * KV * 32];  // [MR][KV * 32], zero past K
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kRowDotShortThreads / 32;
  const int nvec = p.K >> 3;
  // rows [n_begin, n_end) of W belong to this block, row n_begin + i to warp i % kWarps
  const int per = (p.N + gridDim.x - 1) / gridDim.x;
  const int n_begin = blockIdx.x * per, n_end = min(p.N, n_begin + per);
  uint4 wq[kRows][KV];
  auto fetch = [&](int n0) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int n = n0 + r * kWarps;
      const uint4* w = reinterpret_cast<const uint4*>(static_cast<const T*>(b_) + static_cast<long long>(n) * p.ldb);
#pragma unroll
      for (int u = 0; u < KV; ++u)
        wq[r][u] = (n < n_end && lane + 32 * u < nvec) ? __ldcs(w + lane + 32 * u) : make_uint4(0, 0, 0, 0);
    }
  };
  fetch(n_begin + warp);
  for (int i = threadIdx.x; i < MR * KV * 32; i += kRowDotShortThreads) {
    const int m = i / (KV * 32), v = i - m * (KV * 32);
    xs[i] = (m < p.M && v < nvec) ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a_) + static_cast<long long>(m) * p.lda) + v)
                                  : make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  for (int n0 = n_begin + warp; n0 < n_end; n0 += kWarps * kRows) {
    float acc[kRows][MR];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int m = 0; m < MR; ++m) acc[r][m] = 0.f;
#pragma unroll
    for (int u = 0; u < KV; ++u)
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        float xf[8];
        unpack8<BF16>(xs[m * KV * 32 + u * 32 + lane], xf);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          float wf[8];
          unpack8<BF16>(wq[r][u], wf);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[r][m] = fmaf(xf[j], wf[j], acc[r][m]);
        }
      }
    if (n0 + kWarps * kRows < n_end) fetch(n0 + kWarps * kRows);
    // Sums over the lanes, all of them at once: at every step a lane keeps one half of its values and hands over the
    // other (16 shuffles for 16 values instead of 80), and ends with value lane / (32 / kValues).
    constexpr int kValues = kRows * MR;
    float val[kValues];
#pragma unroll
    for (int i = 0; i < kValues; ++i) val[i] = acc[i / MR][i % MR];
#pragma unroll
    for (int o = 16, left = kValues; o > 0; o >>= 1) {
      if (left > 1) {
        left >>= 1;
        const bool upper = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < left; ++i) {
          const float keep = upper ? val[i + left] : val[i], give = upper ? val[i] : val[i + left];
          val[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      } else {
        val[0] += __shfl_xor_sync(0xffffffffu, val[0], o);
      }
    }
    const int i = lane / (32 / kValues), n = n0 + (i / MR) * kWarps;
    if (lane % (32 / kValues) == 0 && n < n_end && i % MR < p.M) epilogue_scalar_store<BF16>(p, val[0], 0, i % MR, n);
  }
}

// ------------------------------------------------------------------------------------------------
// The instantiations the planner chooses from: MX rows of X per group, K split R ways, exchange in H passes.
struct SwapKernel {
  int mx, r, stages;
  void (*launch)(bool bf16, const CUtensorMap& tw, const CUtensorMap& tx, const GemmParams& p, int num_slabs,
                 int num_groups, cudaStream_t stream);
  void (*launch_i8)(bool bf16, const CUtensorMap& tw, const CUtensorMap& tx, const GemmParams& p, int num_slabs,
                    int num_groups, cudaStream_t stream);
  int (*resident)(bool bf16);
};
template <int MX, int R, int H>
static SwapKernel swap_kernel_entry() {
  return SwapKernel{MX, R, SwapCfg<MX, R, H>::kStages,
                    [](bool bf16, const CUtensorMap& tw, const CUtensorMap& tx, const GemmParams& p, int num_slabs,
                       int num_groups, cudaStream_t stream) {
                      if (bf16)
                        launch_swapab<true, MX, R, H>(tw, tx, p, num_slabs, num_groups, stream);
                      else
                        launch_swapab<false, MX, R, H>(tw, tx, p, num_slabs, num_groups, stream);
                    },
                    &launch_swapab_i8<MX, R, H>,
                    [](bool bf16) {
                      return bf16 ? swapab_resident_clusters<true, MX, R, H>() : swapab_resident_clusters<false, MX, R, H>();
                    }};
}
static const std::vector<SwapKernel>& swap_kernels() {
  static const std::vector<SwapKernel> table = {
#define B200AIT_SWAP(MX, R, H) swap_kernel_entry<MX, R, H>(),
      B200AIT_FOR_EACH_SWAP_KERNEL(B200AIT_SWAP)
#undef B200AIT_SWAP
  };
  return table;
}

// Which weight-streaming kernel takes an unbatched problem (nullptr: the tile kernels do).
//
// Up to 63 rows of X: weights of more than 16 MB are bandwidth problems, W is read once at the HBM rate whatever the X tile,
// so one group holds all of X, and K goes two ways, or four / eight ways while the slabs are too few to put most SMs to work
// (from K = 512 on; up to 32 rows from K = 256). Smaller weights are latency problems: a trip to memory takes about 0.7 us, a
// launch about 3 us before the first byte arrives, so the time is the number of ring-fulls a rank streams, plus the exchange
// (each CTA sends (R - 1) / R of its 128 x MX sums through the cluster's shared-memory window, about 40 GB/s per CTA),
// plus a second wave's worth if the units outnumber the resident clusters; up to 64 output tiles of 128 x 128, 48 with an
// added residual, 32 with another epilogue.
//
// From 64 rows on: by the estimates of rules.h, X in groups that are as small as it takes to fill one wave. The tile
// kernels' are the firmer ones where both are close.
static const SwapKernel* plan_swapab(const GemmProblem& g, int tile_width, bool bf16, int from_rows) {
  if (g.n < 128 || g.m < from_rows || g.k < 256) return nullptr;
  const long long slabs = (g.n + 127) / 128, kb_total = (g.k + kBK - 1) / kBK;
  const auto& table = swap_kernels();
  const SwapKernel* best = nullptr;
  double best_us = 0.0;
  if (g.m < 64 && g.n * g.k * 2 > (16ll << 20)) {
    if (g.k < 512 && g.m > 32) return nullptr;
    const int r = (slabs <= sm_count() / 16 && kb_total >= 32) ? 8 : slabs <= sm_count() / 4 ? 4 : 2;
    const int mx = std::max(8 * r, g.m <= 16 ? 16 : g.m <= 32 ? 32 : 64);
    for (const SwapKernel& sk : table)
      if (sk.mx == mx && sk.r == r) return &sk;
    return nullptr;
  }
  if (g.m < 64) {
    if (slabs > (g.swap_epilogue >= 2 ? 32 : g.swap_epilogue == 1 ? 48 : kb_total >= 64 ? 128 : 64)) return nullptr;
    for (const SwapKernel& sk : table) {
      if (kb_total < sk.r) continue;                       // every rank needs a k-block
      const long long units = ((g.m + sk.mx - 1) / sk.mx) * slabs;
      const long long waves = (units + sk.resident(bf16) - 1) / sk.resident(bf16);
      const double kb_rank = static_cast<double>((kb_total + sk.r - 1) / sk.r);
      const double stream = std::max(0.7, kb_rank / sk.stages * 0.7) + kb_rank * 0.06;
      const double tail = 128.0 * sk.mx * 4.0 * (sk.r - 1) / sk.r / 40e3 + 0.005 * sk.mx / sk.r;
      const double us = 3.0 + stream + tail + (waves - 1) * (std::max(stream, tail) + 0.3);
      if (best == nullptr || us < best_us) best = &sk, best_us = us;
    }
    return best;
  }
  for (const SwapKernel& sk : table) {
    if (kb_total < sk.r || !gemm_swap_in_range(g.m, ((g.m + sk.mx - 1) / sk.mx) * slabs, sk.resident(bf16))) continue;
    const double us = gemm_swap_us(g, sk.mx, sk.r, sk.resident(bf16));
    if (best == nullptr || us < best_us) best = &sk, best_us = us;
  }
  return best != nullptr && best_us < 0.97 * gemm_tile_us(g, tile_width, sm_count()) ? best : nullptr;
}

// ------------------------------------------------------------------------------------------------
// host side

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres);
    if (e == cudaSuccess && qres == cudaDriverEntryPointSuccess) fn = reinterpret_cast<EncodeTiledFn>(sym);
  });
  if (!fn) throw Error("cuTensorMapEncodeTiled is not available from the CUDA driver");
  return fn;
}

// 3-D map over a [batch, rows, cols] tensor, cols contiguous; box = [1, box_rows, 128 bytes], 128-byte swizzle
static CUtensorMap make_box_map(const void* base, CUtensorMapDataType type, int elem_bytes, long long cols, long long rows,
                                long long batch, long long row_stride_elems, long long batch_stride_elems, int box_rows) {
  CUtensorMap m;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(batch)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_stride_elems) * elem_bytes,
                           static_cast<cuuint64_t>(batch > 1 ? batch_stride_elems : rows * row_stride_elems) * elem_bytes};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(128 / elem_bytes), static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = get_encode_fn()(&m, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error("cuTensorMapEncodeTiled failed with CUresult " + std::to_string(static_cast<int>(r)));
  return m;
}

CUtensorMap make_tile_map(const void* base, bool bf16, long long cols, long long rows, long long batch,
                          long long row_stride_elems, long long batch_stride_elems, int box_rows) {
  return make_box_map(base, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, cols, rows, batch,
                      row_stride_elems, batch_stride_elems, box_rows);
}

// 5-D map over the GEMM output for the shared-memory-staged store; box = 64 columns x 32 rows,
// 128-byte swizzle. dims / strides are innermost first; strides in elements.
CUtensorMap make_out_map(void* base, bool bf16, const long long (&dims)[5], const long long (&strides)[4]) {
  CUtensorMap m;
  cuuint64_t gd[5], gs[4];
  for (int i = 0; i < 5; ++i) gd[i] = static_cast<cuuint64_t>(dims[i]);
  for (int i = 0; i < 4; ++i) gs[i] = static_cast<cuuint64_t>(strides[i]) * 2;
  cuuint32_t box[5] = {64, 32, 1, 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  CUresult r = get_encode_fn()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, base,
                               gd, gs, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error("cuTensorMapEncodeTiled (output) failed with CUresult " + std::to_string(static_cast<int>(r)));
  return m;
}

struct GemmArgs {
  const void *a, *b, *bias, *d0, *d1;
  void* c;
  long long batch, m, n, k;
  long long lda, ldb, ldc, ldd;
  long long a_bs, b_bs, c_bs, d_bs;
  int epilogue, dtype;
  float alpha;
  int store_mode;
  long long t1, t2, t3;
  int tile_n;  // 0 = choose
  cudaStream_t stream;
  int b_mn = 0;  // B is [K, N] with N contiguous (the reference's "rrr" layouts) instead of [N, K]
  int num_out = 1;                                // destinations: c, then extra_out[0 .. num_out - 2]
  void* extra_out[kMaxOut - 1] = {};              // same shape and strides as c (e.g. peers' copies of the result)
  void* workspace = nullptr;  // fp32 scratch for split-K partial sums (may be null: no split-K)
  long long workspace_bytes = 0;
  int split_k = 0;  // 0 = choose, 1 = off, n = at most n splits
  int* status = nullptr;  // device status word to use instead of the library's allocated one
  int i8_x = 0;  // with i8, where gemm_i8_rowdot says so: `a` holds 16-bit elements of this type, quantised on the way
  int i8 = 0;  // a and b are signed 8-bit integers with a scale per row each (dtype is the result's and the residuals')
  const float *row_scale = nullptr, *col_scale = nullptr;
};

constexpr int kTilePair = kGemmPairWidth;  // tile_n value that asks for 256 x 256 tiles on CTA pairs

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A result of this many bytes is streamed to DRAM while the kernel runs, and its stores set the pace.
constexpr long long kStreamedBytes = 96ll << 20;
// Tile width: 64, 128, 256, or kTilePair.
int choose_tile_n(const GemmProblem& g) {
  // Result streamed to DRAM behind one or two k-blocks per tile (the attention-score shape of bmm_rcr): the run
  // is the drain of the staged stores. A 256-wide tile gives each epilogue warp two 64-column boxes to store
  // through its one staging buffer, the second waiting for the first to drain; 128-wide tiles store one box per
  // tile and overlap the drain with the next tile. Measured, 1024 x [512 x 512 x 64]: 119 us against 133 us;
  // K = 128: 131 against 159 us; from K = 256 on the wider tile wins again (89 against 105 us).
  // Measured later on wider results (us, 128- against 256-wide): K = 64 with N = 1024 .. 4096: 105 against 111 - 126;
  // K = 128 with N = 1024 / 2048: 128 against 118 / 107; K = 40 (rows of 80 bytes, padded to one k-block) with N = 2048 /
  // 4096: 141 against 125 (the wide tile fetches a quarter fewer operand rows, and TMA pays per row). So the narrow
  // tile is taken for one full k-block, and for two only on a narrow result.
  // K = 32 (whole 64-byte rows): 102 us at 1024 x [512 x 512] against 125.
  // Between one and two k-blocks, where the rows are not whole sectors, the estimates are ahead (us, narrow tile, 256-wide, pairs): 695 x
  // [497 x 352 x 104] 101 / 102 / 75, 600 x [400 x 400 x 72] 98 / 83 / 64, 300 x [512 x 512 x 80] 44 / 38 / 41; 512 x [512 x 512 x 96] 66 / 66 / 71.
  if (g.n >= 128 && g.batch * g.m * g.n * 2 > kStreamedBytes &&
      (g.k <= 32 || g.k == kBK || (g.k > kBK && g.k <= 2 * kBK && g.k % 32 == 0 && g.n <= 512)))
    return 128;
  return gemm_best_width(g, sm_count());
}

struct GemmPlan {
  int tile_n;              // choose_tile_n
  const SwapKernel* swap;  // the weight-streaming kernel to take instead, or null
};
// The estimates of one problem take about half a microsecond of host time, which a call of a few microseconds would pay every
// time: each thread keeps the plans of the problem sizes it saw last (by their sizes alone; 64 of them).
static GemmPlan plan_gemm(const GemmProblem& g, bool bf16, bool streams, int from_rows) {
  struct Slot {
    GemmProblem g;
    int sms, flags;
    GemmPlan plan;
  };
  thread_local Slot slots[64] = {};
  const int sms = sm_count(), flags = 1 | (bf16 ? 2 : 0) | (streams ? 4 : 0) | from_rows << 3;
  uint64_t h = static_cast<uint64_t>(g.batch);
  for (const long long v : {g.m, g.n, g.k, g.pitch, static_cast<long long>(g.epilogue * 16 + g.swap_epilogue * 4 + g.generic * 64 + g.pairs * 128 + flags * 256)})
    h = (h ^ static_cast<uint64_t>(v)) * 0x9e3779b97f4a7c15ull;
  Slot& s = slots[h >> 58];
  if (s.flags == flags && s.sms == sms && s.g.batch == g.batch && s.g.m == g.m && s.g.n == g.n && s.g.k == g.k &&
      s.g.epilogue == g.epilogue && s.g.swap_epilogue == g.swap_epilogue && s.g.pitch == g.pitch && s.g.generic == g.generic &&
      s.g.pairs == g.pairs)
    return s.plan;
  GemmPlan plan{choose_tile_n(g), nullptr};
  if (streams) plan.swap = plan_swapab(g, plan.tile_n, bf16, from_rows);
  s = Slot{g, sms, flags, plan};
  return plan;
}

// How many stages of its operand ring a launch uses, where that is fewer than the kernel has. One or two k-blocks per tile: the ring
// runs ahead of the stores by as many tiles, and operands fetched far ahead of use compete with the result
// for DRAM. us with 2 / 3 / 4 / 6 stages of 128-wide tiles, 1024 x [512 x 512 x 64]: 127.5 / 120.6 / 135.8 / 135.7; 768 x [384 x 384
// x 64]: 56 / 53 / 62 / 63; 996 x [258 x 96 x 40]: 22.0 / 22.3 / 22.4 / 24.2; 875 x [392 x 96 x 120]: 40.6 / 35.5 / 35.0 / 39.5;
// 439 x [216 x 72 x 104], row-major B: 13.9 / 14.6 / 15.7 / 16.7; 893 x [69 x 112 x 72]: 10.7 / 10.3 / 10.6 / 11.2. Other widths gain as
// well (621 x [300 x 920 x 80], 256 wide: 104 with three, 111 with all four) or are level, as small results are. Two whole k-blocks
// want all six (512 x [512 x 512 x 128]: 92 / 74.5 / 72 / 70), and so does K = 96, whose rows are whole sectors (512 x [512 x 512 x 96]:
// 73 with three, 66).
int operand_ring_limit(long long k) { return k <= kBK || (k < 2 * kBK && k % 32 != 0) ? 3 : 64; }

// Split-K plan: how many K-splits a problem gets and the fp32 workspace they need.
// Splitting pays when the output tiles cannot fill the SMs but K is deep enough to share out.
struct SplitPlan {
  int tile_n, splits, kb_per_split;
  long long bytes;
};
// `tile_n`: the caller's choice or 0, `planned_tile_n` what is taken for it. `streams`: operands and hints are such that the
// weight-streaming kernels could have taken the problem (gemm_may_split in rules.h).
SplitPlan plan_split_k(const GemmProblem& g, int tile_n, int planned_tile_n, int max_splits, long long workspace_bytes,
                       bool streams) {
  const long long batch = g.batch, m = g.m, n = g.n, k = g.k;
  SplitPlan sp{planned_tile_n, 1, 0, 0};
  const long long num_kb = (k + kBK - 1) / kBK;
  sp.kb_per_split = static_cast<int>(num_kb);
  const long long sms = sm_count();
  if (max_splits == 1 || num_kb < 4 || (max_splits == 0 && streams && !gemm_may_split(m, n, k))) return sp;
  const int width = std::min(sp.tile_n, 256);  // (CTA pairs never split K)
  // One tile row (M <= 128): the run time is the time to stream the weights once. A tcgen05 MMA takes as long
  // as its M x K says, whatever N is, so a CTA consumes weight rows fastest through wide tiles: 128- and
  // 64-wide tiles cap a CTA at half and a quarter of the 256-wide rate, below its share of HBM bandwidth.
  // Take 256-wide tiles and split K to occupy the SMs, unless the fp32 partial sums that costs would add more
  // than ~5 % to the weight traffic (then 128-wide tiles, half the splits).
  if (tile_n == 0 && max_splits == 0 && batch == 1 && m <= kBM && num_kb >= 32) {
    for (int bn : {256, 128}) {
      const long long tiles_n = (n + bn - 1) / bn;
      const long long s = std::min<long long>(std::min<long long>(sms / tiles_n, num_kb / 8), 16);
      if (s < 2 || tiles_n * s * 2 < sms) continue;  // would leave most SMs idle anyway
      if (bn == 256 && s * m * 4 * 20 > k * 2) continue;  // partial sums: s * m * n * 4 bytes against n * k * 2
      if (s * m * n * 4 > workspace_bytes) continue;
      const long long per = (num_kb + s - 1) / s;
      return SplitPlan{bn, static_cast<int>((num_kb + per - 1) / per), static_cast<int>(per),
                       ((num_kb + per - 1) / per) * m * n * 4};
    }
  }
  const long long tiles = ((m + kBM - 1) / kBM) * ((n + width - 1) / width) * batch;
  long long s;
  if (max_splits > 1) {
    s = std::min<long long>(max_splits, num_kb / 2);  // the caller's choice
  } else {
    if (tiles * 2 > sms) return sp;
    // A split adds a second launch and a round trip of fp32 partial sums (4 - 5 us on a small problem): it pays only
    // when it takes that much off the main loop, i.e. from K = 2048 on and with at least 8 k-blocks left per split
    // (384 x 768 x 768: 8.3 us unsplit against 13.9 us in 6 splits; 256 x 768 x 3072: 16.7 us in 4 splits against 18.8).
    if (num_kb < 32) return sp;
    s = std::min<long long>(std::min<long long>(sms / tiles, num_kb / 8), 16);
  }
  while (s > 1 && s * batch * m * n * 4 > workspace_bytes) --s;
  if (s <= 1) return sp;
  sp.tile_n = width;
  const long long per = (num_kb + s - 1) / s;
  sp.splits = static_cast<int>((num_kb + per - 1) / per);  // no empty split
  sp.kb_per_split = static_cast<int>(per);
  sp.bytes = static_cast<long long>(sp.splits) * batch * m * n * 4;
  if (sp.splits <= 1) sp = SplitPlan{width, 1, static_cast<int>(num_kb), 0};
  return sp;
}

// Does this epilogue have instantiations of its own?
static bool has_own_epilogue(int code) {
#define B200AIT_OWN(CODE) \
  if (code == (CODE)) return true;
  B200AIT_FOR_EACH_FAST_EPILOGUE(B200AIT_OWN)
#undef B200AIT_OWN
  return false;
}

// the map of an operand whose rows are g.k elements long
static CUtensorMap operand_map(const GemmArgs& g, const void* base, long long rows, long long batch, long long ld, long long bs,
                               int box_rows) {
  if (g.i8) return make_box_map(base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.k, rows, batch, ld, bs, box_rows);
  return make_tile_map(base, g.dtype == kDTypeBFloat16, g.k, rows, batch, ld, bs, box_rows);
}

void gemm_run(const GemmArgs& g_in) {
  GemmArgs g = g_in;
  long long c_bdiv = 0, c_bs_hi = 0;
  if (g.store_mode == 3) {
    // Permute4DBMM "0213" of the batched GEMMs: [B / d1, d1, M, N] -> [B / d1, M, d1, N], d1 = t1
    // (python/aitemplate/compiler/ops/gemm_universal/bmm_rcr_permute.py, bmm_rrr_permute.py; functor
    // cutlass::layout::Tensor4DPermuteBMM0213 in the reference's CUTLASS fork). Batch b = hi * d1 + lo lands at
    // hi * M * d1 * N + lo * N and rows are d1 * N apart: a plain strided store with a two-level batch stride.
    B200AIT_REQUIRE(g.t1 > 0 && g.batch % g.t1 == 0, "bmm permute: the batch must be a multiple of shape[0]");
    B200AIT_REQUIRE(g.num_out == 1, "bmm permute: one output buffer only");
    c_bdiv = g.t1, c_bs_hi = g.m * g.t1 * g.n;
    g.ldc = g.t1 * g.n, g.c_bs = g.n, g.store_mode = 0;
    if (c_bdiv == 1) c_bdiv = 0, g.c_bs = g.m * g.n;  // d1 = 1: the identity permutation
  }
  B200AIT_REQUIRE(g.dtype == kDTypeHalf || g.dtype == kDTypeBFloat16, "gemm: dtype must be float16 or bfloat16");
  B200AIT_REQUIRE(g.batch >= 0 && g.m >= 0 && g.n >= 0 && g.k >= 0, "gemm: negative dimension");
  if (g.batch == 0 || g.m == 0 || g.n == 0 || g.k == 0) return;  // reference: zero-size problems launch nothing
  B200AIT_REQUIRE(g.a && g.b && g.c, "gemm: null operand pointer with non-zero size");
  B200AIT_REQUIRE(g.m < (1ll << 31) && g.n < (1ll << 31) && g.k < (1ll << 31), "gemm: dimension exceeds int32");
  const int b1 = epi_b1(g.epilogue), b2 = epi_b2(g.epilogue);
  B200AIT_REQUIRE(b1 == kBinaryNone || g.d0, "gemm: epilogue needs d0 but d0 is null");
  B200AIT_REQUIRE(b2 == kBinaryNone || g.d1, "gemm: epilogue needs d1 but d1 is null");
  const bool bf16 = g.dtype == kDTypeBFloat16;

  GemmParams p{};
  p.M = static_cast<int>(g.m), p.N = static_cast<int>(g.n), p.K = static_cast<int>(g.k);
  p.batch = static_cast<int>(g.batch);
  p.a_batch_mul = (g.batch > 1 && g.a_bs == 0) ? 0 : 1;
  p.b_batch_mul = (g.batch > 1 && g.b_bs == 0) ? 0 : 1;
  p.b_mn = g.b_mn;
  p.bias = g.bias, p.d0 = g.d0, p.d1 = g.d1, p.out = g.c;
  p.lda = g.lda, p.ldb = g.ldb, p.a_bs = g.a_bs, p.b_bs = g.b_bs;
  p.ldc = g.ldc, p.ldd = g.ldd, p.c_bs = g.c_bs, p.d_bs = g.d_bs;
  p.alpha = g.alpha, p.epilogue = g.epilogue;
  p.row_scale = g.row_scale, p.col_scale = g.col_scale;
  p.store_mode = 0;
  p.t1 = 1, p.t3 = 1, p.d = 1;
  p.c_bdiv = static_cast<int>(c_bdiv), p.c_bs_hi = c_bs_hi;
  bool vec = (g.n % 8 == 0) && aligned16(g.c) && (g.c_bs % 8 == 0);
  if (g.bias) vec = vec && aligned16(g.bias);
  B200AIT_REQUIRE(g.num_out >= 1 && g.num_out <= kMaxOut, "gemm: between 1 and 8 output buffers");
  B200AIT_REQUIRE(g.num_out == 1 || !g.b_mn, "gemm: several output buffers are not built for row-major B");
  for (int i = 1; i < g.num_out; ++i) {
    B200AIT_REQUIRE(g.extra_out[i - 1] != nullptr, "gemm: null extra output buffer");
    vec = vec && aligned16(g.extra_out[i - 1]);
  }
  if (b1 != kBinaryNone) vec = vec && aligned16(g.d0) && (g.ldd % 8 == 0) && (g.d_bs % 8 == 0);
  if (b2 != kBinaryNone) vec = vec && aligned16(g.d1) && (g.ldd % 8 == 0) && (g.d_bs % 8 == 0);
  if (g.store_mode == 0) {
    vec = vec && (g.ldc % 8 == 0);
  } else if (g.store_mode == 1) {
    // Permute5D "20314": [M/t1, t1, t2, t3, d] -> [t2, M/t1, t3, t1, d], d = N/(t2*t3)
    // (python/aitemplate/compiler/ops/gemm_universal/gemm_rcr_bias_permute.py:59-69)
    B200AIT_REQUIRE(g.t1 > 0 && g.t2 > 0 && g.t3 > 0, "gemm permute: shape entries must be positive");
    B200AIT_REQUIRE(g.m % g.t1 == 0 && g.n % (g.t2 * g.t3) == 0, "gemm permute: M %% t1 or N %% (t2*t3) != 0");
    B200AIT_REQUIRE(g.batch == 1, "gemm permute 20314 is not batched");
    const long long d = g.n / (g.t2 * g.t3);
    p.store_mode = 1;
    p.t1 = static_cast<int>(g.t1), p.t3 = static_cast<int>(g.t3), p.d = static_cast<int>(d);
    p.rs_hi = g.t3 * g.t1 * d, p.rs_lo = d;
    p.cs2 = (g.m / g.t1) * g.t3 * g.t1 * d, p.cs3 = g.t1 * d;
    vec = vec && (d % 8 == 0);
  } else if (g.store_mode == 2) {
    // Permute4D "0213": [M/t1, t1, t2, d] -> [M/t1, t2, t1, d], d = N/t2
    // (python/aitemplate/compiler/ops/gemm_universal/gemm_rcr_permute.py, bmm_rcr_permute.py layout "0213")
    B200AIT_REQUIRE(g.t1 > 0 && g.t2 > 0, "gemm permute: shape entries must be positive");
    B200AIT_REQUIRE(g.m % g.t1 == 0 && g.n % g.t2 == 0, "gemm permute: M %% t1 or N %% t2 != 0");
    const long long d = g.n / g.t2;
    p.store_mode = 1;
    p.t1 = static_cast<int>(g.t1), p.t3 = static_cast<int>(g.t2), p.d = static_cast<int>(d);
    p.rs_hi = g.t2 * g.t1 * d, p.rs_lo = d;
    p.cs2 = 0, p.cs3 = g.t1 * d;
    vec = vec && (d % 8 == 0);
  } else {
    throw Error("gemm: unknown store mode");
  }
  p.vec_ok = vec ? 1 : 0;
  p.status = g.status ? g.status : device_status_word();
  p.splits = 1;
  const long long k_block = g.i8 ? kBKOf<true> : kBK;
  p.kb_per_split = static_cast<int>((g.k + k_block - 1) / k_block);
  p.partial = nullptr;

  // (8-bit operands of any K: boxes end in zeros past it, and the copy needs no more than the pitch and the address)
  const bool tma_w_i8 = g.ldb % 16 == 0 && aligned16(g.b);
  const bool tma_ok = g.i8 ? g.lda % 16 == 0 && aligned16(g.a) && tma_w_i8
                           : (g.k % 8 == 0) && (g.lda % 8 == 0) && (g.ldb % 8 == 0) && aligned16(g.a) && aligned16(g.b) &&
                                 (g.a_bs % 8 == 0) && (g.b_bs % 8 == 0) && g.batch < 65536 * 32;
  B200AIT_REQUIRE(tma_ok || g.num_out == 1, "gemm: several output buffers need TMA-addressable operands");
  if (g.i8 && tma_w_i8 && g.tile_n == 0 && gemm_i8_rowdot(g.m, g.n, g.k, g.i8_x != 0)) {
    run_rowdot_i8(g.a, g.i8_x, g.b, p, bf16, g.stream);
    return;
  }
  // M <= 4, deep K, the caller left tile width and split-K to the library: stream W once on the CUDA cores
  const long long rowdot_smem = (g.m <= 1 ? 1 : g.m <= 2 ? 2 : 4) * g.k * 2;
  if (tma_ok && !g.i8 && g.batch == 1 && !g.b_mn && g.num_out == 1 && g.tile_n == 0 && g.split_k == 0 &&
      gemm_rowdot_long(g.m, g.n, g.k)) {
    const unsigned grid = static_cast<unsigned>(std::min<long long>(sm_count(), (g.n + 3) / 4));
    const int smem = static_cast<int>(rowdot_smem);
#define B200AIT_ROWDOT(BF, MR)                                                                                 \
  do {                                                                                                         \
    static std::atomic<uint64_t> configured{0};                                                                \
    opt_in_smem_once(configured, reinterpret_cast<const void*>(&gemm_rowdot_kernel<BF, MR>), 160 * 1024);      \
    ::b200ait::count_launch(), gemm_rowdot_kernel<BF, MR><<<grid, kRowDotThreads, smem, g.stream>>>(g.a, g.b, p);                         \
  } while (0)
    if (bf16) {
      if (g.m <= 1) B200AIT_ROWDOT(true, 1); else if (g.m <= 2) B200AIT_ROWDOT(true, 2); else B200AIT_ROWDOT(true, 4);
    } else {
      if (g.m <= 1) B200AIT_ROWDOT(false, 1); else if (g.m <= 2) B200AIT_ROWDOT(false, 2); else B200AIT_ROWDOT(false, 4);
    }
#undef B200AIT_ROWDOT
    B200AIT_CUDA_CHECK(cudaGetLastError());
    return;
  }
  // the same for shorter rows, where they are not too many (rules.h); below K = 256 the tile kernels are level or ahead (K =
  // 128, N = 8192: 4.8 against 3.1 .. 6.0 us)
  if (tma_ok && !g.i8 && g.batch == 1 && g.m <= kRowDotMaxM && !g.b_mn && g.num_out == 1 && g.tile_n == 0 && g.split_k == 0 &&
      gemm_rowdot_short(g.m, g.n, g.k, p.vec_ok != 0, bf16)) {
    const unsigned grid = static_cast<unsigned>(std::min<long long>(sm_count(), (g.n + 3) / 4));
#define B200AIT_ROWDOT(MR, KV)                                                                                    \
  do {                                                                                                            \
    ::b200ait::count_launch();                                                                                    \
    if (bf16)                                                                                                     \
      gemm_rowdot_short_kernel<true, MR, KV><<<grid, kRowDotShortThreads, 0, g.stream>>>(g.a, g.b, p);            \
    else                                                                                                          \
      gemm_rowdot_short_kernel<false, MR, KV><<<grid, kRowDotShortThreads, 0, g.stream>>>(g.a, g.b, p);           \
  } while (0)
#define B200AIT_ROWDOT_K(MR)                       \
  do {                                             \
    if (g.k <= 256) B200AIT_ROWDOT(MR, 1);         \
    else if (g.k <= 512) B200AIT_ROWDOT(MR, 2);    \
    else B200AIT_ROWDOT(MR, 4);                    \
  } while (0)
    if (g.m <= 1) B200AIT_ROWDOT_K(1); else if (g.m <= 2) B200AIT_ROWDOT_K(2); else B200AIT_ROWDOT_K(4);
#undef B200AIT_ROWDOT_K
#undef B200AIT_ROWDOT
    B200AIT_CUDA_CHECK(cudaGetLastError());
    return;
  }
  // few rows of X, or few output tiles: the weight-streaming kernel where its planner takes the problem
  const bool streams = tma_ok && g.batch == 1 && !g.b_mn && g.num_out == 1 && g.tile_n == 0 && g.split_k == 0;
  // (row-major B: its boxes are not rows of K, and the figures of rules.h do not hold)
  // (8-bit operands count as 16-bit ones of half the length: the estimates are about boxes of 128 bytes and their MMAs. Over 50 problems of 6 .. 8192
  // rows, 64 .. 8192 columns and depths the kernel so chosen takes 2.0 % longer on average than the best of it and the four widths, 22 % at
  // worst: 120 x 7296 x 768 5.8 us, with 128-wide tiles 4.8. Where N is no multiple of 8 the estimates are those of the 16-bit loop, which
  // takes longer than the 8-bit one; the 16 such problems among them are 2.6 % behind on average, 15 % at worst, 46 x 2043 x 128 6.0 us, 64-wide 5.2)
  const long long lda = g.i8 ? g.lda / 2 : g.lda, ldb = g.i8 ? g.ldb / 2 : g.ldb, k16 = g.i8 ? (g.k + 1) / 2 : g.k;
  const long long pitch = g.b_mn ? kBK : gemm_copy_row_us(lda) > gemm_copy_row_us(ldb) ? lda : ldb;
  GemmProblem problem{g.batch, g.m, g.n, k16, 0, 0, pitch, g.b_mn || g.num_out > 1};
  // CTA pairs do not write permuted batches, and with an epilogue read from the parameters (two residuals, an activation without an
  // instantiation of its own) they need K to hide it behind: 829 x 6824 x 216 + add + add 23.6 us, 128-wide tiles 17.9, 1234 x 4768 x 72
  // mul_tanh 19.7 and 15.0. Over 260 problems with such epilogues, from K = 512 on none is slower than by the rule of whole waves before.
  const bool own_epilogue = has_own_epilogue(p.epilogue) && (b1 != kBinaryNone || p.alpha == 1.f);
  problem.pairs = p.c_bdiv == 0 && (g.batch > 1 || own_epilogue || k16 >= 512);
  GemmPlan planned{g.tile_n, nullptr};
  {
    const int code = p.epilogue;
    // what the weight-streaming kernel's short store loop does without an activation pre-pass: bias [+ relu]
    // [+ one added residual [+ relu]] into a row-major output
    const bool added = epi_b1(code) == kBinaryAdd;
    const bool plain = (epi_b1(code) == kBinaryNone || added) && epi_b2(code) == kBinaryNone &&
                       (epi_u2(code) == kUnaryIdentity || (added && epi_u2(code) == kUnaryRelu)) &&
                       (epi_u1(code) == kUnaryIdentity || epi_u1(code) == kUnaryRelu) && p.store_mode == 0;
    problem.swap_epilogue = !plain ? 2 : added ? 1 : 0;
    problem.epilogue = b1 != kBinaryNone ? 1 : epi_u1(code) != kUnaryIdentity && epi_u1(code) != kUnaryRelu ? 2 : 0;
    if (g.tile_n == 0) planned = plan_gemm(problem, bf16, streams, g.i8 ? 1 : 5);
    if (const SwapKernel* sk = planned.swap) {
      const int num_groups = static_cast<int>((g.m + sk->mx - 1) / sk->mx);
      const int num_slabs = static_cast<int>((g.n + 127) / 128);
      CUtensorMap tw = operand_map(g, g.b, g.n, 1, g.ldb, 0, 128);
      CUtensorMap tx = operand_map(g, g.a, g.m, 1, g.lda, 0, sk->mx);
      (g.i8 ? sk->launch_i8 : sk->launch)(bf16, tw, tx, p, num_slabs, num_groups, g.stream);
      return;
    }
  }
  if (!tma_ok) {
    dim3 grid(static_cast<unsigned>((g.n + 31) / 32), static_cast<unsigned>((g.m + 31) / 32),
              static_cast<unsigned>(g.batch));
    B200AIT_REQUIRE(grid.y < 65536 && grid.z < 65536, "gemm: unaligned problem too large for the CUDA-core kernel");
    count_launch();
    if (g.i8 && bf16)
      gemm_simt_i8_kernel<true><<<grid, 256, 0, g.stream>>>(static_cast<const int8_t*>(g.a), static_cast<const int8_t*>(g.b), p);
    else if (g.i8)
      gemm_simt_i8_kernel<false><<<grid, 256, 0, g.stream>>>(static_cast<const int8_t*>(g.a), static_cast<const int8_t*>(g.b), p);
    else if (bf16)
      gemm_simt_kernel<true><<<grid, 256, 0, g.stream>>>(g.a, g.b, p);
    else
      gemm_simt_kernel<false><<<grid, 256, 0, g.stream>>>(g.a, g.b, p);
    B200AIT_CUDA_CHECK(cudaGetLastError());
    return;
  }

  B200AIT_REQUIRE(g.tile_n == 0 || g.tile_n == 64 || g.tile_n == 128 || g.tile_n == 256 || g.tile_n == kTilePair,
                  "gemm: tile_n must be 64, 128, 256 or 512 (256 x 256 tiles on CTA pairs)");
  const bool ws_ok = g.workspace != nullptr && aligned16(g.workspace);
  const bool force_pair = g.tile_n == kTilePair;
  SplitPlan sp = force_pair || g.i8 ? SplitPlan{g.tile_n ? g.tile_n : planned.tile_n, 1, p.kb_per_split, 0}
                            : plan_split_k(problem, g.tile_n, planned.tile_n, g.num_out > 1 ? 1 : g.split_k, ws_ok ? g.workspace_bytes : 0,
                                           streams);
  if (g.num_out > 1 && sp.tile_n == 64 && g.tile_n == 0) sp.tile_n = 128;  // several destinations need the staged store
  const int bn = std::min(sp.tile_n, 256);
  // CTA pairs (256 x 256 tiles, cta_group::2): a third less operand traffic per flop into each SM, and a residual comes by
  // TMA into the staging boxes where the single-CTA kernels load it per thread.
  B200AIT_REQUIRE(!(force_pair && p.c_bdiv != 0), "bmm permute: the CTA-pair tiles do not take the permuted store");
  const bool pair = sp.tile_n == kTilePair;
  p.splits = sp.splits;
  p.kb_per_split = sp.kb_per_split;
  p.partial = static_cast<float*>(g.workspace);
  const long long a_batch = p.a_batch_mul ? g.batch : 1, b_batch = p.b_batch_mul ? g.batch : 1;
  CUtensorMap ta = operand_map(g, g.a, g.m, a_batch, g.lda, g.a_bs, kBM);
  CUtensorMap tb = g.b_mn ? make_tile_map(g.b, bf16, g.n, g.k, b_batch, g.ldb, g.b_bs, kBK)  // 64 x 64 boxes
                          : operand_map(g, g.b, g.n, b_batch, g.ldb, g.b_bs, pair ? bn / 2 : bn);
  // Staged TMA store: row-major output with 16-byte aligned rows, or a permuted output whose 64-column
  // groups and 32-row groups each stay inside one contiguous run of the destination.
  OutMaps tout;
  for (int i = 0; i < kMaxOut; ++i) tout.m[i] = ta;  // placeholders: only the first num_out are ever read
  p.tma_store = 0;
  p.num_out = g.num_out;
  if (bn >= 128 && p.splits == 1 && p.vec_ok) {
    for (int i = 0; i < g.num_out; ++i) {
      void* dst = i == 0 ? g.c : g.extra_out[i - 1];
      if (p.store_mode == 0) {
        const long long bs = g.batch > 1 ? g.c_bs : g.m * g.ldc;
        if (p.c_bdiv != 0) {  // batch coordinate split into (lo, hi)
          const long long dims[5] = {g.n, g.m, p.c_bdiv, g.batch / p.c_bdiv, 1};
          const long long strides[4] = {g.ldc, g.c_bs, p.c_bs_hi, p.c_bs_hi};
          tout.m[i] = make_out_map(dst, bf16, dims, strides);
        } else {
          const long long dims[5] = {g.n, g.m, g.batch, 1, 1};
          const long long strides[4] = {g.ldc, bs, bs, bs};
          tout.m[i] = make_out_map(dst, bf16, dims, strides);
        }
        p.tma_store = 1;
      } else if (p.d % 64 == 0 && p.t1 % 32 == 0 && g.batch == 1) {
        // destination [c2][row / t1][c3][row % t1][d]: dims innermost first (d, t1, t3, M / t1, c2 extent)
        const long long c2_extent = g.n / (static_cast<long long>(p.d) * p.t3);
        const long long dims[5] = {p.d, p.t1, p.t3, g.m / p.t1, c2_extent};
        const long long strides[4] = {p.rs_lo, p.cs3, p.rs_hi, p.cs2 > 0 ? p.cs2 : p.rs_hi * (g.m / p.t1)};
        tout.m[i] = make_out_map(dst, bf16, dims, strides);
        p.tma_store = 1;
      }
    }
  }
  B200AIT_REQUIRE(g.num_out == 1 || p.tma_store,
                  "gemm: several output buffers need the staged TMA store (tile_n >= 128, no split-K, N and the "
                  "output strides multiples of 8, 16-byte aligned pointers)");
  p.tiles_m = pair ? (p.M + 2 * kBM - 1) / (2 * kBM) : (p.M + kBM - 1) / kBM;
  p.tiles_n = (p.N + bn - 1) / bn;
  p.num_tiles = p.tiles_m * p.tiles_n * p.batch;
  p.num_units = p.num_tiles * p.splits;
  const FastDiv by_batch(p.tiles_m * p.tiles_n), by_group(kGroupM * p.tiles_n), by_rest(std::max(1, p.tiles_m % kGroupM));
  p.batch_mul = by_batch.mul, p.batch_shr = by_batch.shr, p.group_mul = by_group.mul, p.group_shr = by_group.shr;
  p.rest_mul = by_rest.mul, p.rest_shr = by_rest.shr;
  p.ring_limit = operand_ring_limit(k16);
  const int grid = pair ? 2 * std::min(p.num_units, sm_count() / 2) : std::min(p.num_units, sm_count());
  CUtensorMap td0 = ta;
  p.tma_d0 = 0;
  if (pair && p.tma_store && b1 != kBinaryNone && b2 == kBinaryNone) {
    // residual boxes of 32 rows x 64 columns, fetched by the epilogue warps into their staging buffers
    td0 = make_tile_map(g.d0, bf16, g.n, g.m, g.batch, g.ldd, g.d_bs, 32);
    p.tma_d0 = 1;
  }
  if (g.i8 && bf16)
    launch_tc_i8<true>(sp.tile_n, ta, tb, tout, td0, p, grid, g.stream);
  else if (g.i8)
    launch_tc_i8<false>(sp.tile_n, ta, tb, tout, td0, p, grid, g.stream);
  else if (pair)
    launch_tc_pair256(bf16, ta, tb, tout, td0, p, grid, g.stream);
  else if (bn == 256)
    launch_tc_width<256>(bf16, ta, tb, tout, p, grid, g.stream);
  else if (bn == 128)
    launch_tc_width<128>(bf16, ta, tb, tout, p, grid, g.stream);
  else
    launch_tc_width<64>(bf16, ta, tb, tout, p, grid, g.stream);
  if (p.splits > 1) {
    const long long total = static_cast<long long>(p.batch) * p.M * ((p.N + 31) / 32);
    const unsigned blocks = static_cast<unsigned>((total + 255) / 256);
    if (bf16)
      ::b200ait::count_launch(), gemm_splitk_reduce_kernel<true><<<blocks, 256, 0, g.stream>>>(p);
    else
      ::b200ait::count_launch(), gemm_splitk_reduce_kernel<false><<<blocks, 256, 0, g.stream>>>(p);
    B200AIT_CUDA_CHECK(cudaGetLastError());
  }
}

}  // namespace b200ait

using namespace b200ait;

// Generic entry point: every gemm_rcr* / bmm_rcr* op of the path maps onto it.
// `workspace` (may be null) is fp32 scratch for split-K partial sums; split_k: 0 = library chooses,
// 1 = never split, n > 1 = at most n splits. Without a workspace the GEMM never splits.
B200AIT_EXPORT int b200ait_gemm_rcr(const void* a, const void* b, const void* bias, const void* d0, const void* d1,
                                    void* c, int64_t batch, int64_t m, int64_t n, int64_t k, int64_t lda, int64_t ldb,
                                    int64_t ldc, int64_t ldd, int64_t a_batch_stride, int64_t b_batch_stride,
                                    int64_t c_batch_stride, int64_t d_batch_stride, int epilogue, int dtype,
                                    float alpha, int store_mode, int64_t t1, int64_t t2, int64_t t3, int tile_n,
                                    void* workspace, int64_t workspace_bytes, int split_k, cudaStream_t stream) {
  return guarded("b200ait_gemm_rcr", [&] {
    GemmArgs g{a,   b,   bias,           d0,             d1,             c,
               batch, m,   n,              k,              lda,            ldb,
               ldc, ldd, a_batch_stride, b_batch_stride, c_batch_stride, d_batch_stride,
               epilogue, dtype, alpha, store_mode, t1, t2, t3, tile_n, stream};
    g.workspace = workspace;
    g.workspace_bytes = workspace_bytes;
    g.split_k = split_k;
    gemm_run(g);
  });
}

static void check_i8(const GemmArgs& g, const float* b_scale) {
  B200AIT_REQUIRE(g.dtype == kDTypeHalf || g.dtype == kDTypeBFloat16, "gemm: dtype must be float16 or bfloat16");
  B200AIT_REQUIRE(g.m >= 0 && g.n >= 0 && g.k >= 0, "gemm: negative dimension");
  // (the kernels count past the last row and column, up to two 256-row tiles or a step of eight columns for 16 warps and as much ahead)
  constexpr long long kMost = (1ll << 31) - 1024;
  B200AIT_REQUIRE(g.m <= kMost && g.n <= kMost, "gemm: dimension exceeds int32");
  // sums of K products of at most 2^14 each stay below 2^31
  B200AIT_REQUIRE(g.k < (1 << 17), "gemm: 8-bit operands take up to 131071 columns");
  if (g.m == 0 || g.n == 0) return;
  B200AIT_REQUIRE(g.k != 0, "gemm: 8-bit operands have no columns");
  B200AIT_REQUIRE(g.a && g.b && g.c, "gemm: null operand pointer with non-zero size");
  B200AIT_REQUIRE(b_scale != nullptr, "gemm: 8-bit operands need the scales of their rows");
  const bool residual = epi_b1(g.epilogue) != kBinaryNone || epi_b2(g.epilogue) != kBinaryNone;
  B200AIT_REQUIRE(g.lda >= g.k && g.ldb >= g.k && g.ldc >= g.n && (!residual || g.ldd >= g.n), "gemm: a row pitch is shorter than the row");
  auto at = [](const void* ptr, unsigned bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; };
  B200AIT_REQUIRE(at(g.bias, 2) && at(g.d0, 2) && at(g.d1, 2) && at(g.c, 2) && at(b_scale, 4), "gemm: a pointer is not aligned to its type");
}

// gemm_rcr of signed 8-bit integers: c = epilogue(sum_k a[m, k] b[n, k] * a_scale[m] * b_scale[n] + bias, d0, d1).
B200AIT_EXPORT int b200ait_gemm_rcr_i8(const void* a, const float* a_scale, const void* b, const float* b_scale,
                                       const void* bias, const void* d0, const void* d1, void* c, int64_t m, int64_t n,
                                       int64_t k, int64_t lda, int64_t ldb, int64_t ldc, int64_t ldd, int epilogue, int dtype,
                                       int tile_n, cudaStream_t stream) {
  return guarded("b200ait_gemm_rcr_i8", [&] {
    GemmArgs g{a, b, bias, d0, d1, c, 1, m, n, k, lda, ldb, ldc, ldd, 0, 0, 0, 0, epilogue, dtype, 1.f, 0, 1, 1, 1, tile_n, stream};
    check_i8(g, b_scale);
    B200AIT_REQUIRE(m == 0 || n == 0 || a_scale, "gemm: 8-bit operands need the scales of their rows");
    B200AIT_REQUIRE((reinterpret_cast<uintptr_t>(a_scale) & 3u) == 0, "gemm: a pointer is not aligned to its type");
    g.i8 = 1, g.row_scale = a_scale, g.col_scale = b_scale;
    gemm_run(g);
  });
}

// The same with its left operand in 16 bits, quantised on the way (quantize.cu): by the product's own kernel for a few rows, else
// into `scratch`.
static int64_t i8_pitch(int64_t k) { return (k + 15) / 16 * 16; }
static int64_t x16_scratch_bytes(int64_t m, int64_t n, int64_t k, int64_t ldb, const void* b, int tile_n) {
  if (m <= 0 || n <= 0 || k <= 0 || (tile_n == 0 && ldb % 16 == 0 && aligned16(b) && gemm_i8_rowdot(m, n, k, true))) return 0;
  return m * i8_pitch(k) + m * 4;
}
B200AIT_EXPORT int b200ait_gemm_rcr_i8_x16_scratch_bytes(const void* b, int64_t m, int64_t n, int64_t k, int64_t ldb, int tile_n,
                                                         int64_t* bytes_out) {
  return guarded("b200ait_gemm_rcr_i8_x16_scratch_bytes", [&] {
    B200AIT_REQUIRE(bytes_out, "bytes_out is null");
    *bytes_out = x16_scratch_bytes(m, n, k, ldb, b, tile_n);
  });
}
B200AIT_EXPORT int b200ait_gemm_rcr_i8_x16(const void* x, int x_dtype, const void* b, const float* b_scale, const void* bias,
                                           const void* d0, const void* d1, void* c, int64_t m, int64_t n, int64_t k, int64_t ldx,
                                           int64_t ldb, int64_t ldc, int64_t ldd, int epilogue, int dtype, int tile_n, void* scratch,
                                           int64_t scratch_bytes, cudaStream_t stream) {
  return guarded("b200ait_gemm_rcr_i8_x16", [&] {
    B200AIT_REQUIRE(x_dtype == kDTypeHalf || x_dtype == kDTypeBFloat16, "gemm: x must be float16 or bfloat16");
    GemmArgs g{x, b, bias, d0, d1, c, 1, m, n, k, ldx, ldb, ldc, ldd, 0, 0, 0, 0, epilogue, dtype, 1.f, 0, 1, 1, 1, tile_n, stream};
    check_i8(g, b_scale);
    if (m == 0 || n == 0) return;
    B200AIT_REQUIRE((reinterpret_cast<uintptr_t>(x) & 1u) == 0, "gemm: a pointer is not aligned to its type");
    g.i8 = 1, g.col_scale = b_scale;
    const int64_t needed = x16_scratch_bytes(m, n, k, ldb, b, tile_n);
    if (needed == 0) {
      g.i8_x = x_dtype;
    } else {
      const int64_t pitch = i8_pitch(k);
      B200AIT_REQUIRE(scratch && aligned16(scratch) && scratch_bytes >= needed, "gemm: the scratch for quantised rows is missing or too small");
      float* scale = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + m * pitch);
      if (b200ait_quantize_rows(scratch, scale, x, m, k, ldx, pitch, 0, 0, x_dtype, stream) != 0) throw Error(last_error());
      g.a = scratch, g.lda = pitch, g.row_scale = scale;
    }
    gemm_run(g);
  });
}

// b200ait_gemm_rcr with B stored [batch, k, n] (n contiguous, row stride ldb): the reference's gemm_rrr / bmm_rrr
// layouts (python/aitemplate/compiler/ops/gemm_universal/gemm_rrr.py, bmm_xxx.py "rrr"). Same kernel, the B tile
// reaches the tensor core as an MN-major operand.
B200AIT_EXPORT int b200ait_gemm_rrr(const void* a, const void* b, const void* bias, const void* d0, const void* d1,
                                    void* c, int64_t batch, int64_t m, int64_t n, int64_t k, int64_t lda, int64_t ldb,
                                    int64_t ldc, int64_t ldd, int64_t a_batch_stride, int64_t b_batch_stride,
                                    int64_t c_batch_stride, int64_t d_batch_stride, int epilogue, int dtype,
                                    float alpha, int tile_n, void* workspace, int64_t workspace_bytes, int split_k,
                                    cudaStream_t stream) {
  return guarded("b200ait_gemm_rrr", [&] {
    GemmArgs g{a,   b,   bias,           d0,             d1,             c,
               batch, m,   n,              k,              lda,            ldb,
               ldc, ldd, a_batch_stride, b_batch_stride, c_batch_stride, d_batch_stride,
               epilogue, dtype, alpha, 0, 1, 1, 1, tile_n, stream};
    g.b_mn = 1;
    g.workspace = workspace;
    g.workspace_bytes = workspace_bytes;
    g.split_k = split_k;
    gemm_run(g);
  });
}

// bmm_rcr_permute / bmm_rrr_permute (python/aitemplate/compiler/ops/gemm_universal/bmm_rcr_permute.py:28-116,
// bmm_rrr_permute.py; generated signature python/aitemplate/backend/cuda/gemm_universal/bmm_common.py:56-81 with the
// Permute4DBMM_0213 epilogue of bmm_permute_common.py): c[b] = alpha * a[b] @ op(b[b]) for a [batch, m, k] and
// b [batch, n, k] (b_row_major = 0) or [batch, k, n] (b_row_major = 1), stored as
// [batch / d1, d1, m, n].permute(0, 2, 1, 3), i.e. c has the shape [batch / d1, m, d1, n]. A batch stride of 0
// broadcasts that operand.
B200AIT_EXPORT int b200ait_bmm_permute0213(const void* a, const void* b, void* c, int64_t batch, int64_t m, int64_t n,
                                           int64_t k, int64_t a_batch_stride, int64_t b_batch_stride, int64_t d1,
                                           int b_row_major, int dtype, float alpha, int tile_n, cudaStream_t stream) {
  return guarded("b200ait_bmm_permute0213", [&] {
    B200AIT_REQUIRE(d1 > 0, "bmm permute: shape[0] must be positive");
    GemmArgs g{a, b, nullptr, nullptr, nullptr, c, batch, m, n, k, k, b_row_major ? n : k, n, n,
               a_batch_stride, b_batch_stride, m * n, m * n, 0, dtype, alpha, 3, d1, 1, 1, tile_n, stream};
    g.b_mn = b_row_major ? 1 : 0;
    g.split_k = 1;
    gemm_run(g);
  });
}

// The same GEMM with its result written to num_out buffers of identical shape and strides (1 <= num_out <= 8)
// by the epilogue's TMA stores: outs[0] is usually this GPU's buffer and the others are peer-mapped pointers
// to other GPUs' buffers, so that a rank that computes one column block of Y = X W^T places it in every
// rank's full Y while the next tile is being computed (no separate gather pass). Never splits K; needs the
// staged store (N and ldc multiples of 8, 16-byte aligned pointers).
B200AIT_EXPORT int b200ait_gemm_rcr_multi_out(const void* a, const void* b, const void* bias, const void* d0,
                                              void* const* outs, int num_out, int64_t m, int64_t n, int64_t k,
                                              int64_t lda, int64_t ldb, int64_t ldc, int64_t ldd, int epilogue,
                                              int dtype, float alpha, int tile_n, cudaStream_t stream) {
  return guarded("b200ait_gemm_rcr_multi_out", [&] {
    B200AIT_REQUIRE(outs != nullptr && num_out >= 1 && num_out <= kMaxOut, "outs: 1 to 8 output pointers");
    GemmArgs g{a, b, bias, d0, nullptr, outs[0], 1, m, n, k, lda, ldb, ldc, ldd, 0, 0, 0, 0,
               epilogue, dtype, alpha, 0, 1, 1, 1, tile_n, stream};
    g.num_out = num_out;
    for (int i = 1; i < num_out; ++i) g.extra_out[i - 1] = outs[i];
    g.split_k = 1;
    gemm_run(g);
  });
}

// The most split-K workspace that b200ait_gemm_rcr or b200ait_gemm_rrr would use for a problem of these sizes if given enough.
B200AIT_EXPORT int b200ait_gemm_rcr_workspace_bytes(int64_t batch, int64_t m, int64_t n, int64_t k, int tile_n,
                                                    int split_k, int64_t* bytes_out) {
  return guarded("b200ait_gemm_rcr_workspace_bytes", [&] {
    B200AIT_REQUIRE(bytes_out, "bytes_out is null");
    *bytes_out = 0;
    if (batch <= 0 || m <= 0 || n <= 0 || k <= 0) return;
    if (tile_n == kTilePair) return;
    const GemmProblem g{batch, m, n, k, 0, 0, k, false};
    *bytes_out = plan_split_k(g, tile_n, tile_n ? tile_n : choose_tile_n(g), split_k, 1ll << 62, false).bytes;
  });
}

// The same for one unbatched launch of b200ait_gemm_rcr: 0 for the kernels that take none.
B200AIT_EXPORT int b200ait_gemm_rcr_scratch_bytes(int64_t m, int64_t n, int64_t k, int tile_n, int split_k, int64_t* bytes_out) {
  return guarded("b200ait_gemm_rcr_scratch_bytes", [&] {
    B200AIT_REQUIRE(bytes_out, "bytes_out is null");
    *bytes_out = 0;
    if (m <= 0 || n <= 0 || k <= 0 || k % 8 != 0 || tile_n == kTilePair || split_k == 1) return;
    if (tile_n == 0 && split_k == 0 && !gemm_may_split(m, n, k)) return;
    const GemmProblem g{1, m, n, k, 0, 0, k, false};
    *bytes_out = plan_split_k(g, tile_n, tile_n ? tile_n : choose_tile_n(g), split_k, 1ll << 62, false).bytes;
  });
}

// Entry points with the argument order of the reference's generated per-op functions
// (python/aitemplate/backend/cuda/gemm_universal/common_bias.py:77-97: a, b, bias, c, workspace, split_k,
//  pointers to the dims of a [M,K], b [N,K] and c [M,N], stream). *c_dim0/*c_dim1 are written.
static int gemm_rcr_bias_named(const char* name, int epilogue, void* a, void* b, void* bias, void* d0, void* d1,
                               void* c, int64_t* a_dim0, int64_t* a_dim1, int64_t* b_dim0, int64_t* b_dim1,
                               int64_t* c_dim0, int64_t* c_dim1, bool need_bias, cudaStream_t stream) {
  return guarded(name, [&] {
    B200AIT_REQUIRE(a_dim0 && a_dim1 && b_dim0 && b_dim1, "null dimension pointer");
    const int64_t m = *a_dim0, k = *a_dim1, n = *b_dim0;
    B200AIT_REQUIRE(*b_dim1 == k, "a and b disagree on K");
    if (c_dim0) *c_dim0 = m;
    if (c_dim1) *c_dim1 = n;
    if (m != 0 && n != 0 && k != 0) B200AIT_REQUIRE(!need_bias || bias, "bias_ptr is null!");
    GemmArgs g{a, b, bias, d0, d1, c, 1, m, n, k, k, k, n, n, 0, 0, 0, 0, epilogue, kDTypeHalf, 1.f, 0, 1, 1, 1, 0,
               stream};
    gemm_run(g);
  });
}

#define B200AIT_DEFINE_GEMM_BIAS(NAME, U1)                                                                         \
  B200AIT_EXPORT int b200ait_##NAME(void* a, void* b, void* bias, void* c, uint8_t* workspace, int split_k,        \
                                    int64_t* a_dim0, int64_t* a_dim1, int64_t* b_dim0, int64_t* b_dim1,            \
                                    int64_t* c_dim0, int64_t* c_dim1, cudaStream_t stream) {                       \
    (void)workspace;                                                                                               \
    (void)split_k;                                                                                                 \
    return gemm_rcr_bias_named("b200ait_" #NAME, make_epilogue(U1, kBinaryNone, kBinaryNone, kUnaryIdentity), a, b, \
                               bias, nullptr, nullptr, c, a_dim0, a_dim1, b_dim0, b_dim1, c_dim0, c_dim1, true,    \
                               stream);                                                                            \
  }
B200AIT_DEFINE_GEMM_BIAS(gemm_rcr_bias, kUnaryIdentity)
B200AIT_DEFINE_GEMM_BIAS(gemm_rcr_bias_relu, kUnaryRelu)
B200AIT_DEFINE_GEMM_BIAS(gemm_rcr_bias_gelu, kUnaryGelu)
B200AIT_DEFINE_GEMM_BIAS(gemm_rcr_bias_fast_gelu, kUnaryFastGelu)
B200AIT_DEFINE_GEMM_BIAS(gemm_rcr_bias_sigmoid, kUnarySigmoid)
B200AIT_DEFINE_GEMM_BIAS(gemm_rcr_bias_tanh, kUnaryTanh)
B200AIT_DEFINE_GEMM_BIAS(gemm_rcr_bias_swish, kUnarySwish)
B200AIT_DEFINE_GEMM_BIAS(gemm_rcr_bias_hardswish, kUnaryHardswish)
#undef B200AIT_DEFINE_GEMM_BIAS

// python/aitemplate/backend/cuda/gemm_universal/gemm_rcr.py (common.py:172-198): no bias operand
B200AIT_EXPORT int b200ait_gemm_rcr_plain(void* a, void* b, void* c, uint8_t* workspace, int split_k, int64_t* a_dim0,
                                          int64_t* a_dim1, int64_t* b_dim0, int64_t* b_dim1, int64_t* c_dim0,
                                          int64_t* c_dim1, cudaStream_t stream) {
  (void)workspace;
  (void)split_k;
  return gemm_rcr_bias_named("b200ait_gemm_rcr_plain", 0, a, b, nullptr, nullptr, nullptr, c, a_dim0, a_dim1, b_dim0,
                             b_dim1, c_dim0, c_dim1, false, stream);
}

// python/aitemplate/backend/cuda/gemm_universal/common_bias_broadcast.py:276-305: d0 (and d1) precede c
#define B200AIT_DEFINE_GEMM_BIAS_D0(NAME, U1, B1, U2)                                                                \
  B200AIT_EXPORT int b200ait_##NAME(void* a, void* b, void* bias, void* d0, void* c, uint8_t* workspace,             \
                                    int split_k, int64_t* a_dim0, int64_t* a_dim1, int64_t* b_dim0, int64_t* b_dim1, \
                                    int64_t* c_dim0, int64_t* c_dim1, cudaStream_t stream) {                         \
    (void)workspace;                                                                                                 \
    (void)split_k;                                                                                                   \
    return gemm_rcr_bias_named("b200ait_" #NAME, make_epilogue(U1, B1, kBinaryNone, U2), a, b, bias, d0, nullptr, c, \
                               a_dim0, a_dim1, b_dim0, b_dim1, c_dim0, c_dim1, true, stream);                        \
  }
#define B200AIT_DEFINE_GEMM_BIAS_D0_D1(NAME, U1, B1, B2, U2)                                                         \
  B200AIT_EXPORT int b200ait_##NAME(void* a, void* b, void* bias, void* d0, void* d1, void* c, uint8_t* workspace,   \
                                    int split_k, int64_t* a_dim0, int64_t* a_dim1, int64_t* b_dim0, int64_t* b_dim1, \
                                    int64_t* c_dim0, int64_t* c_dim1, cudaStream_t stream) {                         \
    (void)workspace;                                                                                                 \
    (void)split_k;                                                                                                   \
    return gemm_rcr_bias_named("b200ait_" #NAME, make_epilogue(U1, B1, B2, U2), a, b, bias, d0, d1, c, a_dim0,       \
                               a_dim1, b_dim0, b_dim1, c_dim0, c_dim1, true, stream);                                \
  }
B200AIT_DEFINE_GEMM_BIAS_D0(gemm_rcr_bias_add, kUnaryIdentity, kBinaryAdd, kUnaryIdentity)
B200AIT_DEFINE_GEMM_BIAS_D0(gemm_rcr_bias_add_relu, kUnaryIdentity, kBinaryAdd, kUnaryRelu)
B200AIT_DEFINE_GEMM_BIAS_D0(gemm_rcr_bias_mul, kUnaryIdentity, kBinaryMul, kUnaryIdentity)
B200AIT_DEFINE_GEMM_BIAS_D0(gemm_rcr_bias_mul_tanh, kUnaryIdentity, kBinaryMul, kUnaryTanh)
B200AIT_DEFINE_GEMM_BIAS_D0(gemm_rcr_bias_sigmoid_mul, kUnarySigmoid, kBinaryMul, kUnaryIdentity)
B200AIT_DEFINE_GEMM_BIAS_D0(gemm_rcr_bias_sigmoid_mul_tanh, kUnarySigmoid, kBinaryMul, kUnaryTanh)
B200AIT_DEFINE_GEMM_BIAS_D0_D1(gemm_rcr_bias_add_add, kUnaryIdentity, kBinaryAdd, kBinaryAdd, kUnaryIdentity)
B200AIT_DEFINE_GEMM_BIAS_D0_D1(gemm_rcr_bias_add_add_relu, kUnaryIdentity, kBinaryAdd, kBinaryAdd, kUnaryRelu)
B200AIT_DEFINE_GEMM_BIAS_D0_D1(gemm_rcr_bias_mul_add, kUnaryIdentity, kBinaryMul, kBinaryAdd, kUnaryIdentity)
#undef B200AIT_DEFINE_GEMM_BIAS_D0
#undef B200AIT_DEFINE_GEMM_BIAS_D0_D1

// python/aitemplate/backend/cuda/gemm_universal/gemm_rcr_bias_permute.py:55-95 (layout "20314", shape (t1,t2,t3))
B200AIT_EXPORT int b200ait_gemm_rcr_bias_permute(void* a, void* b, void* bias, void* c, uint8_t* workspace,
                                                 int split_k, int64_t* a_dim0, int64_t* a_dim1, int64_t* b_dim0,
                                                 int64_t* b_dim1, int64_t* c_dim0, int64_t* c_dim1, int64_t t1,
                                                 int64_t t2, int64_t t3, cudaStream_t stream) {
  (void)workspace;
  (void)split_k;
  return guarded("b200ait_gemm_rcr_bias_permute", [&] {
    B200AIT_REQUIRE(a_dim0 && a_dim1 && b_dim0 && b_dim1, "null dimension pointer");
    const int64_t m = *a_dim0, k = *a_dim1, n = *b_dim0;
    B200AIT_REQUIRE(*b_dim1 == k, "a and b disagree on K");
    if (c_dim0) *c_dim0 = m;
    if (c_dim1) *c_dim1 = n;
    if (m != 0 && n != 0 && k != 0) B200AIT_REQUIRE(bias, "bias_ptr is null!");
    GemmArgs g{a, b, bias, nullptr, nullptr, c, 1, m, n, k, k, k, n, n, 0, 0, 0, 0, 0, kDTypeHalf, 1.f, 1, t1, t2, t3,
               0, stream};
    gemm_run(g);
  });
}

// python/aitemplate/backend/cuda/gemm_universal/bmm_common.py:56-81: a [B,M,K], b [B,N,K], c [B,M,N]
B200AIT_EXPORT int b200ait_bmm_rcr(void* a, void* b, void* c, uint8_t* workspace, int64_t* a_dim0, int64_t* a_dim1,
                                   int64_t* a_dim2, int64_t* b_dim0, int64_t* b_dim1, int64_t* b_dim2,
                                   int64_t* c_dim0, int64_t* c_dim1, int64_t* c_dim2, cudaStream_t stream) {
  (void)workspace;
  return guarded("b200ait_bmm_rcr", [&] {
    B200AIT_REQUIRE(a_dim0 && a_dim1 && a_dim2 && b_dim0 && b_dim1 && b_dim2, "null dimension pointer");
    const int64_t ba = *a_dim0, m = *a_dim1, k = *a_dim2, bb = *b_dim0, n = *b_dim1;
    B200AIT_REQUIRE(*b_dim2 == k, "a and b disagree on K");
    B200AIT_REQUIRE(ba == bb || ba == 1 || bb == 1, "batch sizes are not broadcastable");
    const int64_t batch = ba > bb ? ba : bb;
    if (c_dim0) *c_dim0 = batch;
    if (c_dim1) *c_dim1 = m;
    if (c_dim2) *c_dim2 = n;
    GemmArgs g{a, b, nullptr, nullptr, nullptr, c, batch, m, n, k, k, k, n, n,
               (ba == 1 && batch > 1) ? 0 : m * k, (bb == 1 && batch > 1) ? 0 : n * k, m * n, m * n,
               0, kDTypeHalf, 1.f, 0, 1, 1, 1, 0, stream};
    gemm_run(g);
  });
}


// ------------------------------------------------------------------------------------------------
// Split-K GEMM for callers that must not allocate device memory.
//
// Some hosts of this library run where cudaMalloc is off limits: inside a serving process whose
// memory pool was sized and handed out at start-up, under a framework allocator that owns the whole
// device, or on a path that has to stay free of driver allocation calls because those serialise
// with other work. b200ait_gemm_rcr needs two pieces of device memory beyond its operands: the
// fp32 scratch for split-K partial sums (the caller's `workspace`) and the status word the kernels
// report into (allocated by the library on first use). This entry point needs neither from the
// caller and allocates neither: both live in the file-scope array below, which is part of the
// library image, so every GPU that loads the library holds these 16 MiB + 256 bytes until the
// process exits.
namespace b200ait {
constexpr long long kStaticScratchHeader = 256;               // status word, padded to the alignment
constexpr long long kStaticScratchBytes = 16ll << 20;         // split-K partial sums: at most 16 MiB
static __device__ __align__(256) unsigned char g_static_scratch[kStaticScratchHeader + kStaticScratchBytes];

// In host code `g_static_scratch` is only a handle for the runtime, not an address a kernel can
// use; the device address comes from cudaGetSymbolAddress, asked once per device with that device
// current.
static unsigned char* static_scratch_device_ptr() {
  constexpr int kMaxDev = 64;
  static std::mutex mu;
  static unsigned char* ptrs[kMaxDev] = {};
  int dev = 0;
  B200AIT_CUDA_CHECK(cudaGetDevice(&dev));
  B200AIT_REQUIRE(dev >= 0 && dev < kMaxDev, "device ordinal out of range");
  std::lock_guard<std::mutex> lock(mu);
  if (!ptrs[dev]) {
    void* p = nullptr;
    B200AIT_CUDA_CHECK(cudaGetSymbolAddress(&p, g_static_scratch));
    B200AIT_REQUIRE(p != nullptr, "cudaGetSymbolAddress returned a null address for the static scratch");
    ptrs[dev] = static_cast<unsigned char*>(p);
  }
  return ptrs[dev];
}
}  // namespace b200ait

// Same computation and arguments as b200ait_gemm_rcr, minus the workspace: split-K partial sums go
// to the library's static scratch. Calls no cudaMalloc / cudaFree and no allocating library routine.
//   * Limit: the partial sums of two splits must fit, 2 * batch * m * n * 4 bytes <= 16 MiB;
//     larger problems are rejected with an error (use b200ait_gemm_rcr with your own workspace).
//     Within the limit the library may use fewer splits than b200ait_gemm_rcr would.
//   * The first call on each device looks up the scratch address (cudaGetSymbolAddress) and sets
//     kernel attributes; make that first call outside any stream capture.
//   * Every call on a device shares the one scratch area and it keeps whatever the last call left
//     there. Each call rewrites all partial sums it later reads and clears the status word first,
//     but two calls that overlap on the GPU (different streams) race on it: keep calls to this entry
//     point stream-ordered per device.
//   * status_out (device pointer, may be null) receives the kernel status word after the GEMM
//     (0 = clean), stream-ordered; read it after synchronising the stream.
B200AIT_EXPORT int b200ait_gemm_rcr_static_scratch(const void* a, const void* b, const void* bias, const void* d0,
                                                   const void* d1, void* c, int64_t batch, int64_t m, int64_t n,
                                                   int64_t k, int64_t lda, int64_t ldb, int64_t ldc, int64_t ldd,
                                                   int64_t a_batch_stride, int64_t b_batch_stride,
                                                   int64_t c_batch_stride, int64_t d_batch_stride, int epilogue,
                                                   int dtype, float alpha, int store_mode, int64_t t1, int64_t t2,
                                                   int64_t t3, int tile_n, int split_k, int* status_out,
                                                   cudaStream_t stream) {
  return guarded("b200ait_gemm_rcr_static_scratch", [&] {
    B200AIT_REQUIRE(batch >= 0 && m >= 0 && n >= 0 && k >= 0, "gemm: negative dimension");
    // limit check without forming the product first: 2 * batch * m * n * 4 can leave int64 for absurd
    // dimensions and would then slip under the limit
    const long long cap_elems = kStaticScratchBytes / 8;  // fp32 partial sums of two splits
    bool fits = true;
    long long elems = 1;
    for (long long d : {(long long)batch, (long long)m, (long long)n}) {
      if (d == 0) { elems = 0; break; }
      if (elems > cap_elems / d) { fits = false; break; }
      elems *= d;
    }
    if (!fits || elems > cap_elems) {
      const std::string need = fits ? std::to_string(elems * 8) : std::string("more than 2^40");
      throw Error("problem too large for the static scratch: two splits of " + std::to_string(batch) + " x " +
                  std::to_string(m) + " x " + std::to_string(n) + " fp32 partial sums need " + need +
                  " bytes, the limit is " + std::to_string(kStaticScratchBytes) +
                  "; call b200ait_gemm_rcr with a caller-provided workspace instead");
    }
    unsigned char* scratch = static_scratch_device_ptr();
    int* status = reinterpret_cast<int*>(scratch);
    B200AIT_CUDA_CHECK(cudaMemsetAsync(status, 0, sizeof(int), stream));  // must start at zero
    GemmArgs g{a,   b,   bias,           d0,             d1,             c,
               batch, m,   n,              k,              lda,            ldb,
               ldc, ldd, a_batch_stride, b_batch_stride, c_batch_stride, d_batch_stride,
               epilogue, dtype, alpha, store_mode, t1, t2, t3, tile_n, stream};
    g.workspace = scratch + kStaticScratchHeader;
    g.workspace_bytes = kStaticScratchBytes;
    g.split_k = split_k;
    g.status = status;
    gemm_run(g);
    if (status_out)
      B200AIT_CUDA_CHECK(cudaMemcpyAsync(status_out, status, sizeof(int), cudaMemcpyDeviceToDevice, stream));
  });
}

