// quantize_rows: rows of 16-bit activations to signed 8-bit integers with a scale per row, the left operand of
// b200ait_gemm_rcr_i8. With v = act(x), or act(x[:, :n]) * x[:, n:] for the two halves of a gated feed-forward's first product,
//   scale = max |v| / 127,   q = round(127 v / max |v|)   (ties to even; rowteam.cuh)
// The reference has no 8-bit activations; the activations are those of its GEMM epilogues (epilogue.cuh).
//
// Bound: HBM, 2 n bytes read (4 n gated) and n written per row. The row stays in registers between the search for its largest value
// and the rounding, so it crosses HBM once.
#include "rowteam.cuh"

namespace b200ait {

struct QuantizeParams {
  const void* x;
  int8_t* q;
  float* scale;
  long long rows, x_pitch, q_pitch;
  int n, activation;
};

template <int VEC, int CNT, int MOST, bool GATED, bool BF16>
__global__ void __launch_bounds__(kTeamBlock<MOST>) quantize_rows_kernel(const QuantizeParams p) {
  grid_release();
  grid_wait();
  constexpr bool BLOCK = MOST > 32;
  using T = typename Elem16<BF16>::T;
  using Raw = RawUnit<VEC>;
  __shared__ uint32_t words[1][32];
  const RowTeam<BLOCK> team{words, BLOCK ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x & 31),
                            BLOCK ? static_cast<int>(blockDim.x) : 32};
  const long long row = BLOCK ? static_cast<long long>(blockIdx.x)
                              : static_cast<long long>(blockIdx.x) * kTeamWarpsPerBlock + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int units = p.n / VEC;
  const T* x = static_cast<const T*>(p.x) + row * p.x_pitch;
  typename Raw::Type raw[CNT], up[GATED ? CNT : 1];
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    const int u = team.tid + i * team.threads;
    raw[i] = u < units ? ld_stream(reinterpret_cast<const typename Raw::Type*>(x) + u) : Raw::zero();
    if (GATED) up[i] = u < units ? ld_stream(reinterpret_cast<const typename Raw::Type*>(x + p.n) + u) : Raw::zero();
  }
  float v[CNT * VEC];
#pragma unroll
  for (int i = 0; i < CNT; ++i) unpack_unit<VEC, BF16>(raw[i], &v[i * VEC]);
  if (p.activation != kUnaryIdentity) apply_unary_vec(p.activation, v);
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    if (GATED) {
      float f[VEC];
      unpack_unit<VEC, BF16>(up[i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i * VEC + j] *= f[j];
    }
    if (team.tid + i * team.threads < units) {  // (an activation of the zeros past the end need not be 0)
#pragma unroll
      for (int j = 0; j < VEC; ++j) most = max(most, magnitude_bits(v[i * VEC + j]));
    }
  }
  const RowScale s = row_scale_of(team.most(most, 0));
  if (team.tid == 0) p.scale[row] = s.scale;
  int8_t* q = p.q + row * p.q_pitch;
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    const int u = team.tid + i * team.threads;
    if (u < units) store_quantized<VEC>(q, u, s, &v[i * VEC]);
  }
}

// Rows longer than the registers of a block hold (32768 elements): a block walks its row twice, the second time out of L2.
template <bool BF16>
__global__ void __launch_bounds__(kTeamMaxThreads) quantize_long_rows_kernel(const QuantizeParams p, const bool gated) {
  using E = Elem16<BF16>;
  using T = typename E::T;
  __shared__ uint32_t words[1][32];
  const RowTeam<true> team{words, static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x)};
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_pitch;
  auto value = [&](int i) {
    const float v = apply_unary(p.activation, E::to_float(x[i]));
    return gated ? v * E::to_float(x[p.n + i]) : v;
  };
  uint32_t most = 0;
  for (int i = team.tid; i < p.n; i += team.threads) most = max(most, magnitude_bits(value(i)));
  const RowScale s = row_scale_of(team.most(most, 0));
  if (team.tid == 0) p.scale[row] = s.scale;
  int8_t* q = p.q + row * p.q_pitch;
  for (int i = team.tid; i < p.n; i += team.threads) {
    const float v = value(i);
    store_quantized<1>(q, i, s, &v);
  }
}

template <int VEC, int CNT, int MOST, bool GATED, bool BF16>
static void launch_quantize(const QuantizeParams& p, int threads, cudaStream_t stream) {
  constexpr bool BLOCK = MOST > 32;
  const long long blocks = BLOCK ? p.rows : (p.rows + kTeamWarpsPerBlock - 1) / kTeamWarpsPerBlock;
  const int block = BLOCK ? threads : 32 * kTeamWarpsPerBlock;
  const bool early = blocks_start_early(blocks, block, sm_count(), 2048) || !in_capture(stream);
  launch_early(&quantize_rows_kernel<VEC, CNT, MOST, GATED, BF16>, dim3(static_cast<unsigned>(blocks)), block, 0, stream, early, 1, p);
}

template <bool GATED, bool BF16>
static void quantize_dispatch(const QuantizeParams& p, bool vector_ok, cudaStream_t stream) {
  const TeamShape t = team_shape(p.rows, p.n, vector_ok, sm_count());
  if (t.cnt == 0) {
    count_launch();
    quantize_long_rows_kernel<BF16><<<static_cast<unsigned>(p.rows), t.threads, 0, stream>>>(p, GATED);
    B200AIT_CUDA_CHECK(cudaGetLastError());
    return;
  }
  for_team_shape(t, [&](auto vec, auto cnt, auto most) {
    launch_quantize<decltype(vec)::value, decltype(cnt)::value, decltype(most)::value, GATED, BF16>(p, t.threads, stream);
  });
}

}  // namespace b200ait

using namespace b200ait;

B200AIT_EXPORT int b200ait_quantize_rows(void* q, float* scale, const void* x, int64_t rows, int64_t n, int64_t x_pitch,
                                         int64_t q_pitch, int activation, int gated, int dtype, cudaStream_t stream) {
  return guarded("b200ait_quantize_rows", [&] {
    B200AIT_REQUIRE(dtype == kDTypeHalf || dtype == kDTypeBFloat16, "quantize_rows: dtype must be float16 or bfloat16");
    B200AIT_REQUIRE(rows >= 0 && n >= 0, "quantize_rows: negative dimension");
    B200AIT_REQUIRE(activation >= kUnaryIdentity && activation <= kUnaryHardswish, "quantize_rows: unknown activation");
    if (rows == 0 || n == 0) return;
    B200AIT_REQUIRE(q && scale && x, "quantize_rows: null pointer with non-zero size");
    B200AIT_REQUIRE(rows < (1ll << 31) && n < (1ll << 30), "quantize_rows: dimension exceeds int32");
    B200AIT_REQUIRE(x_pitch >= (gated ? 2 * n : n) && q_pitch >= n, "quantize_rows: a row pitch is shorter than the row");
    auto aligned = [](const void* ptr, unsigned to) { return (reinterpret_cast<uintptr_t>(ptr) & (to - 1)) == 0; };
    const bool vector_ok = n % 8 == 0 && x_pitch % 8 == 0 && q_pitch % 8 == 0 && aligned(x, 16) && aligned(q, 8);
    const QuantizeParams p{x, static_cast<int8_t*>(q), scale, rows, x_pitch, q_pitch, static_cast<int>(n), activation};
    const bool bf16 = dtype == kDTypeBFloat16;
    if (gated && bf16)
      quantize_dispatch<true, true>(p, vector_ok, stream);
    else if (gated)
      quantize_dispatch<true, false>(p, vector_ok, stream);
    else if (bf16)
      quantize_dispatch<false, true>(p, vector_ok, stream);
    else
      quantize_dispatch<false, false>(p, vector_ok, stream);
  });
}
