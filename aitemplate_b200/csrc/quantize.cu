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
  InnerRows inside;
  int n, activation;
};

template <int CNT, int THREADS, bool ALIGNED, bool GATED, bool BF16>
__global__ void __launch_bounds__(kTeamBlock<THREADS>) quantize_rows_kernel(const QuantizeParams p) {
  grid_release();
  grid_wait();
  using Team = RowTeam<CNT, THREADS, ALIGNED>;
  __shared__ uint32_t words[1][32];
  __shared__ uint2 staged[kTeamBlock<THREADS> / THREADS][Team::kStagedBytes / 8];
  const long long row = Team::row();
  if (row >= p.rows) return;
  const uint16_t* x = static_cast<const uint16_t*>(p.x) + row * p.x_pitch;
  const uint16_t* lo = static_cast<const uint16_t*>(p.x);
  const uint16_t* hi = lo + (p.rows - 1) * p.x_pitch + (GATED ? 2 * p.n : p.n);
  const bool inner = row >= p.inside.begin && row < p.inside.end;
  const Team team(words, p.n, x);
  uint4 raw[CNT], up[GATED ? CNT : 1];
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    raw[i] = team.load(x, inner, lo, hi, i);
    if (GATED) up[i] = team.template load_off<true>(x + p.n, i);
  }
  float v[CNT * 8];
#pragma unroll
  for (int i = 0; i < CNT; ++i) unpack8<BF16>(raw[i], &v[i * 8]);
  if (p.activation != kUnaryIdentity) apply_unary_vec_of<true>(p.activation, v);
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    if (GATED) {
      float f[8];
      unpack8<BF16>(up[i], f);
      by_pairs<8>(&v[i * 8], [&](uint64_t a, int j) { return mul2(a, pack2(f[j], f[j + 1])); });
    }
    team.clear_rest(&v[i * 8], i);
    take_magnitudes<8>(most, &v[i * 8]);
  }
  const RowScale s = row_scale_of(team.most(most, 0));
  if (team.tid == 0) p.scale[row] = s.scale;
  uint2 b[CNT];
#pragma unroll
  for (int i = 0; i < CNT; ++i) b[i] = quantize_unit(s, &v[i * 8]);
  team.store_bytes(p.q + row * p.q_pitch, b, staged[threadIdx.x / THREADS]);
}

// Rows longer than the registers of a block hold (32768 elements), or results at an odd place: a block walks its row twice, the
// second time out of L2. Bound by its loads of single elements: 1000 x 40000 takes 116 us, gated 2 x 40000 (swish) 109, where HBM would take 18 and
// 31; 1000 x 32768, which fits, 25 and 39.
template <bool BF16>
__global__ void __launch_bounds__(kTeamMaxThreads) quantize_long_rows_kernel(const QuantizeParams p, const bool gated) {
  using E = Elem16<BF16>;
  using T = typename E::T;
  __shared__ uint32_t words[1][32];
  const RowTeam<1, kTeamMaxThreads, true> team(words, p.n, nullptr);
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_pitch;
  auto value = [&](int i) {
    const float v = apply_unary_of<true>(p.activation, E::to_float(x[i]));
    return gated ? mul_exact(v, E::to_float(x[p.n + i])) : v;  // (as the pairs of the other kernel: small products are not flushed)
  };
  uint32_t most = 0;
  for (int i = team.tid; i < p.n; i += kTeamMaxThreads) {
    const float v = value(i);
    take_magnitudes<1>(most, &v);
  }
  const RowScale s = row_scale_of(team.most(most, 0));
  if (team.tid == 0) p.scale[row] = s.scale;
  int8_t* q = p.q + row * p.q_pitch;
  for (int i = team.tid; i < p.n; i += kTeamMaxThreads) q[i] = quantize_value(s, value(i));
}

template <int CNT, int THREADS, bool ALIGNED, bool GATED, bool BF16>
static void launch_quantize(const QuantizeParams& p, cudaStream_t stream) {
  constexpr int kBlock = kTeamBlock<THREADS>;
  const long long blocks = THREADS > 32 ? p.rows : (p.rows + kTeamWarpsPerBlock - 1) / kTeamWarpsPerBlock;
  const auto kernel = &quantize_rows_kernel<CNT, THREADS, ALIGNED, GATED, BF16>;
  static std::atomic<uint64_t> done{0};
  prefer_l1_once(done, reinterpret_cast<const void*>(kernel), kBlock);
  const bool early = blocks_start_early(blocks, kBlock, sm_count(), 2048) || !in_capture(stream);
  launch_early(kernel, dim3(static_cast<unsigned>(blocks)), kBlock, 0, stream, early, 1, p);
}

template <bool GATED, bool BF16>
static void quantize_dispatch(const QuantizeParams& p, bool lie_well, bool aligned, cudaStream_t stream) {
  // us with one / four units a thread: 333 x 2 x 768 1.9 / 2.3, x 2048 2.6 / 3.1, x 4096 3.8 / 4.0; 600 x 4096 4.9 / 5.4; 1000 x 4096 6.7 / 6.8,
  // x 1280 3.8 / 3.8; 2000 x 4096 11.4 / 10.2, x 1280 6.0 / 5.3
  const TeamShape t = team_shape(p.rows, p.n, aligned, 4ll * sm_count(), 1);
  if (t.cnt == 0 || !lie_well) {
    count_launch();
    quantize_long_rows_kernel<BF16><<<static_cast<unsigned>(p.rows), kTeamMaxThreads, 0, stream>>>(p, GATED);
    B200AIT_CUDA_CHECK(cudaGetLastError());
    return;
  }
  for_team_shape<1>(t, [&](auto cnt, auto threads, auto whole) {
    launch_quantize<decltype(cnt)::value, decltype(threads)::value, decltype(whole)::value, GATED, BF16>(p, stream);
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
    if (rows == 0) return;
    B200AIT_REQUIRE(n != 0, "quantize_rows: the rows have no columns");  // (and so no largest value to scale by)
    B200AIT_REQUIRE(q && scale && x, "quantize_rows: null pointer with non-zero size");
    B200AIT_REQUIRE(rows < (1ll << 31) && n < (1ll << 30), "quantize_rows: dimension exceeds int32");
    B200AIT_REQUIRE(x_pitch >= (gated ? 2 * n : n) && q_pitch >= n, "quantize_rows: a row pitch is shorter than the row");
    B200AIT_REQUIRE(multiple_of(x, 2) && multiple_of(scale, 4), "quantize_rows: a pointer is not aligned to its type");
    const bool lie_well = multiple_of(q, 8) && q_pitch % 8 == 0;
    const bool aligned = n % 8 == 0 && x_pitch % 8 == 0 && multiple_of(x, 16);
    const QuantizeParams p{x, static_cast<int8_t*>(q), scale, rows, x_pitch, q_pitch, inner_rows(rows, x_pitch),
                           static_cast<int>(n), activation};
    const bool bf16 = dtype == kDTypeBFloat16;
    if (gated && bf16)
      quantize_dispatch<true, true>(p, lie_well, aligned, stream);
    else if (gated)
      quantize_dispatch<true, false>(p, lie_well, aligned, stream);
    else if (bf16)
      quantize_dispatch<false, true>(p, lie_well, aligned, stream);
    else
      quantize_dispatch<false, false>(p, lie_well, aligned, stream);
  });
}
