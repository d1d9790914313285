// gemm_rcr_i8 for one or two rows of X in 8 bits, one to four in 16: the run time is the time to read W once, and there is nothing for the tensor core to
// amortise. One block per SM holds X in shared memory and owns a contiguous share of the rows of W; a warp streams R rows at a time,
// KV 16-byte vectors of each per lane, eight vectors in flight while the eight before them are multiplied (four products per
// instruction, exact 32-bit sums), adds up across the lanes and runs the fused epilogue. X may come in 16 bits: then every
// block quantises it for itself (rowteam.cuh; a few KB out of L2) while its first rows of W are on their way, which saves the
// launch of quantize_rows and a trip through memory.
//
// Bound: HBM, N K bytes. The floor of 4096 x 4096 is 2.6 us at the measured copy rate, of 8192 x 8192 10.2; a launch alone takes about 2. One row in
// a graph with other weights at every call takes 5.6 and 12.7 us, with W in L2 3.7 and 7.5.
#include "gemm_kernel.cuh"
#include "rowteam.cuh"

namespace b200ait {

constexpr int kRowDotI8Threads = 512;
constexpr int kRowDotI8Smem = 160 * 1024;  // for the rows of X (gemm_i8_rowdot)

// X to shared memory, `pad` bytes a row, zeros past K
template <int MR>
__device__ __forceinline__ void stage_rows_i8(const GemmParams& p, const int8_t* x, int8_t* xs, int pad) {
  const bool vectors = p.lda % 16 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
#pragma unroll 1
  for (int m = 0; m < MR; ++m) {
    const int8_t* row = x + m * p.lda;
    const int whole = m < p.M && vectors ? p.K & ~15 : 0;
    for (int k = static_cast<int>(threadIdx.x) * 16; k < whole; k += kRowDotI8Threads * 16)
      *reinterpret_cast<uint4*>(xs + m * pad + k) = *reinterpret_cast<const uint4*>(row + k);
    for (int k = whole + static_cast<int>(threadIdx.x); k < pad; k += kRowDotI8Threads)
      xs[m * pad + k] = m < p.M && k < p.K ? row[k] : int8_t{0};
  }
}
// ... quantised from 16 bits, with its scales
template <int MR, bool X_BF16>
__device__ __forceinline__ void quantize_rows_i8(const GemmParams& p, const uint16_t* x, int8_t* xs, float* scales, uint32_t* most, int pad) {
  using E = Elem16<X_BF16>;
  const bool vectors = p.K % 8 == 0 && p.lda % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
  const int step = vectors ? 8 : 1;
  auto load = [&](const uint16_t* at, float (&v)[8]) {
    if (vectors) {
      unpack8<X_BF16>(*reinterpret_cast<const uint4*>(at), v);
    } else {
      v[0] = E::to_float(*reinterpret_cast<const typename E::T*>(at));
#pragma unroll
      for (int j = 1; j < 8; ++j) v[j] = 0.f;
    }
  };
#pragma unroll 1
  for (int m = 0; m < MR; ++m) {
    uint32_t mine = 0;
    if (m < p.M) {
      for (int k = static_cast<int>(threadIdx.x) * step; k < p.K; k += kRowDotI8Threads * step) {
        float v[8];
        load(x + m * p.lda + k, v);
        take_magnitudes<8>(mine, v);
      }
    }
    mine = __reduce_max_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == 0) most[m * (kRowDotI8Threads / 32) + (threadIdx.x >> 5)] = mine;
  }
  __syncthreads();
#pragma unroll 1
  for (int m = 0; m < MR; ++m) {
    const int lane = threadIdx.x & 31;
    const RowScale s = row_scale_of(__reduce_max_sync(0xffffffffu, lane < kRowDotI8Threads / 32 ? most[m * (kRowDotI8Threads / 32) + lane] : 0u));
    if (threadIdx.x == 0) scales[m] = s.scale;
    const int end = m < p.M ? p.K : 0;
    for (int k = static_cast<int>(threadIdx.x) * step; k < end; k += kRowDotI8Threads * step) {
      float v[8];
      load(x + m * p.lda + k, v);
      if (vectors)
        *reinterpret_cast<uint2*>(xs + m * pad + k) = quantize_unit(s, v);
      else
        xs[m * pad + k] = quantize_value(s, v[0]);
    }
    for (int k = end + static_cast<int>(threadIdx.x); k < pad; k += kRowDotI8Threads) xs[m * pad + k] = 0;
  }
}

// X_TYPE: 0 signed 8-bit integers, 1 fp16, 2 bf16
template <bool BF16, int MR, int KV, int X_TYPE>
__global__ void __launch_bounds__(kRowDotI8Threads, 1) gemm_rowdot_i8_kernel(const void* x, const int8_t* w, const GemmParams p) {
  constexpr int R = 8 / KV, kWarps = kRowDotI8Threads / 32, kValues = R * MR;
  extern __shared__ __align__(16) int8_t xs[];  // [MR][pad]
  __shared__ float scales[MR];
  __shared__ uint32_t most[X_TYPE == 0 ? 1 : MR * kWarps];
  grid_release();
  grid_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nvec = p.K >> 4, pad = (p.K + 15) & ~15, turns = (nvec + 32 * KV - 1) / (32 * KV) > 0 ? (nvec + 32 * KV - 1) / (32 * KV) : 1;
  // rows [n_begin, n_end) of W belong to this block, row n_begin + i to warp i % kWarps
  const int per = (p.N + gridDim.x - 1) / gridDim.x;
  const int n_begin = blockIdx.x * per, n_end = min(p.N, n_begin + per);
  // one step: KV vectors of R rows from row n0 on, the t-th of `turns` shares of K
  auto fetch = [&](int n0, int t, uint4 (&wq)[R][KV]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int n = n0 + r * kWarps;
      const uint4* row = reinterpret_cast<const uint4*>(w + static_cast<long long>(n) * p.ldb) + t * 32 * KV + lane;
#pragma unroll
      for (int u = 0; u < KV; ++u)
        wq[r][u] = n < n_end && t * 32 * KV + u * 32 + lane < nvec ? ld_stream(row + u * 32) : make_uint4(0, 0, 0, 0);
    }
  };
  uint4 wa[R][KV], wb[R][KV];
  int n0 = n_begin + warp, t = 0;
  fetch(n0, t, wa);
  if constexpr (X_TYPE == 0)
    stage_rows_i8<MR>(p, static_cast<const int8_t*>(x), xs, pad);
  else
    quantize_rows_i8<MR, X_TYPE == 2>(p, static_cast<const uint16_t*>(x), xs, scales, most, pad);
  __syncthreads();
  int acc[R][MR];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[r][m] = 0;
  auto step = [&](uint4 (&cur)[R][KV], uint4 (&next)[R][KV]) {
    const int at_n = n0, at_t = t;
    if (++t == turns) t = 0, n0 += kWarps * R;
    if (n0 < n_end) fetch(n0, t, next);
#pragma unroll
    for (int u = 0; u < KV; ++u) {
      const int v = min(at_t * 32 * KV + u * 32 + lane, (pad >> 4) - 1);  // past the end the vectors of W are zeros
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const int4 xv = *reinterpret_cast<const int4*>(xs + m * pad + v * 16);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint4& q = cur[r][u];
          acc[r][m] = __dp4a(static_cast<int>(q.x), xv.x, acc[r][m]);
          acc[r][m] = __dp4a(static_cast<int>(q.y), xv.y, acc[r][m]);
          acc[r][m] = __dp4a(static_cast<int>(q.z), xv.z, acc[r][m]);
          acc[r][m] = __dp4a(static_cast<int>(q.w), xv.w, acc[r][m]);
        }
      }
    }
    if (at_t != turns - 1) return;
    if (p.K & 15) {  // the last elements, a lane each
      const int k = (p.K & ~15) + lane;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int n = at_n + r * kWarps;
        const int wv = k < p.K && n < n_end ? w[static_cast<long long>(n) * p.ldb + k] : 0;
#pragma unroll
        for (int m = 0; m < MR; ++m) acc[r][m] += wv * xs[m * pad + min(k, pad - 1)];
      }
    }
    // Sums over the lanes, all at once: at every step a lane keeps one half of its values and hands over the other, and ends
    // with value lane / (32 / kValues).
    int val[kValues];
#pragma unroll
    for (int i = 0; i < kValues; ++i) val[i] = acc[i / MR][i % MR], acc[i / MR][i % MR] = 0;
#pragma unroll
    for (int o = 16, left = kValues; o > 0; o >>= 1) {
      if (left > 1) {
        left >>= 1;
        const bool upper = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < left; ++i) {
          const int keep = upper ? val[i + left] : val[i], give = upper ? val[i] : val[i + left];
          val[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      } else {
        val[0] += __shfl_xor_sync(0xffffffffu, val[0], o);
      }
    }
    const int i = lane / (32 / kValues), n = at_n + (i / MR) * kWarps, m = i % MR;
    if (lane % (32 / kValues) == 0 && n < n_end && m < p.M)
      epilogue_scalar_store_i8<BF16>(p, scale_column_i8(val[0], p.col_scale[n]), X_TYPE == 0 ? p.row_scale[m] : scales[m], m, n);
  };
  while (n0 < n_end) {
    step(wa, wb);
    if (n0 < n_end) step(wb, wa);
  }
}

template <bool BF16, int MR, int KV, int X_TYPE>
static void launch_rowdot_i8(const void* x, const int8_t* w, const GemmParams& p, cudaStream_t stream) {
  auto* kernel = &gemm_rowdot_i8_kernel<BF16, MR, KV, X_TYPE>;
  static std::atomic<uint64_t> configured{0};
  opt_in_smem_once(configured, reinterpret_cast<const void*>(kernel), kRowDotI8Smem);
  const int grid = std::min(sm_count(), (p.N + 3) / 4), smem = MR * ((p.K + 15) & ~15);
  // Early whatever the size: a block per SM at most, which walks one share of W. One after the other in a graph, one and two rows by 32
  // matrices of 128 x 320 .. 14336 x 4096 out of L2 and from HBM, 0.25 .. 0.6 us less each (1024 x 1024 2.07 us, 2.52 late; from HBM 2.37, 2.85; 8192 x
  // 8192 from HBM 12.7, 13.1), but for one row by 8192 x 8192 out of L2, which is level.
  launch_early(kernel, dim3(static_cast<unsigned>(grid)), kRowDotI8Threads, static_cast<size_t>(smem), stream, true, 1, x, w, p);
}

// x_type: 0 for 8-bit rows with p.row_scale, else the DType of 16-bit ones
void run_rowdot_i8(const void* x, int x_type, const void* w, const GemmParams& p, bool bf16, cudaStream_t stream) {
  const int8_t* w8 = static_cast<const int8_t*>(w);
  const int type = x_type == 0 ? 0 : x_type == kDTypeBFloat16 ? 2 : 1;
  const int mr = p.M <= 1 ? 1 : p.M <= 2 ? 2 : 4, kv = p.K <= 512 ? 1 : p.K <= 1024 ? 2 : p.K <= 2048 ? 4 : 8;
  switch (((bf16 ? 1 : 0) * 3 + type) * 100 + mr * 10 + kv) {
#define B200AIT_ONE(BF, MR, KV, TYPE) \
  case ((BF) * 3 + (TYPE)) * 100 + (MR) * 10 + (KV): return launch_rowdot_i8<(BF) != 0, MR, KV, TYPE>(x, w8, p, stream);
#define B200AIT_KVS(BF, MR, TYPE) B200AIT_ONE(BF, MR, 1, TYPE) B200AIT_ONE(BF, MR, 2, TYPE) B200AIT_ONE(BF, MR, 4, TYPE) B200AIT_ONE(BF, MR, 8, TYPE)
#define B200AIT_ROWS(BF, TYPE) B200AIT_KVS(BF, 1, TYPE) B200AIT_KVS(BF, 2, TYPE)
    B200AIT_ROWS(0, 0) B200AIT_ROWS(0, 1) B200AIT_ROWS(0, 2) B200AIT_ROWS(1, 0) B200AIT_ROWS(1, 1) B200AIT_ROWS(1, 2)
    B200AIT_KVS(0, 4, 1) B200AIT_KVS(0, 4, 2) B200AIT_KVS(1, 4, 1) B200AIT_KVS(1, 4, 2)  // (8-bit rows: rules.h sends no more than two)
#undef B200AIT_ROWS
#undef B200AIT_KVS
#undef B200AIT_ONE
  }
  throw Error("no kernel for as many rows of 8-bit integers");
}

}  // namespace b200ait
