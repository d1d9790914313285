// residual_norm: what stands between two blocks of a transformer, in one pass over the rows:
//   p   = post_norm(x) * post_gamma + post_beta        (or x: no norm after the block)
//   sum = residual_scale * residual + gate * p         (the residual stream; stored rounded to 16 bits where it is asked for)
//   y   = norm(sum) * gamma + beta                     (of the unrounded sum)
// norm: layer, (v - mean) / sqrt(var + eps), or rms, v / sqrt(mean(v^2) + eps). gate, gamma and beta are one vector or one per equal part
// of the rows (a gate per sample). y in 16 bits, or in 8 with a scale per row (rowteam.cuh), the left operand of b200ait_gemm_rcr_i8.
// Next of kin in the reference: layernorm (python/aitemplate/backend/cuda/layernorm_sigmoid_mul/layernorm_sigmoid_mul.py:72-83)
// behind an element-wise add; here the row is read once and the statistics are taken from registers, in fp32, the variance
// about the mean.
//
// Bound: HBM, up to 8 n bytes per row (x, residual, sum, y; 7 n with y in 8 bits).
#include "rowteam.cuh"

namespace b200ait {

enum RowNorm : int { kNormNone = 0, kNormLayer = 1, kNormRms = 2 };

// Which of the vectors that rows share goes with a row: row / (rows that share one), by multiply-high with constants of the host (a
// 64-bit division takes as long as four values: 8192 x 1280 with three of them 17.9 us, 15.6 so, both with the results of the run
// before overwritten in L2).
struct RowParts {
  int rows = 1;
  unsigned mul = 0, shr = 0;
  __device__ __forceinline__ int of(long long row) const { return fast_div(static_cast<int>(row), rows, mul, shr); }
};

struct ResidualNormParams {
  const void *x, *residual, *gate, *post_gamma, *post_beta, *gamma, *beta;
  void *sum, *y;
  float* scale;  // of y in 8 bits
  long long rows, y_pitch;
  InnerRows inside;  // of x and residual
  RowParts whole, gate_part, gamma_part, beta_part;  // whole: one vector for all rows
  int n, post, norm;
  float residual_scale, eps;
};

// Turns the row in `v` into its norm, without gamma and beta. `slot` and slot + 1 are the reductions' words. What is not the row's
// is 0 before and after.
template <int CNT, int THREADS, bool ALIGNED>
__device__ __forceinline__ void normalize_row(const RowTeam<CNT, THREADS, ALIGNED>& team, float (&v)[CNT * 8], int kind, float inv_n,
                                              float eps, int slot) {
  float lo, hi;
  if (kind == kNormLayer) {
    uint64_t s = pack2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < CNT * 8; j += 2) s = add2(s, pack2(v[j], v[j + 1]));
    unpack2(s, lo, hi);
    const float less = -team.sum(lo + hi, slot) * inv_n;
    by_pairs<CNT * 8>(v, [&](uint64_t x, int) { return add2(x, pack2(less, less)); });
#pragma unroll
    for (int i = 0; i < CNT; ++i) team.clear_rest(&v[i * 8], i);
  }
  uint64_t q = pack2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < CNT * 8; j += 2) {
    const uint64_t x = pack2(v[j], v[j + 1]);
    q = fma2(x, x, q);
  }
  unpack2(q, lo, hi);
  const float rstd = rsqrtf(fmaf(team.sum(lo + hi, slot + 1), inv_n, eps));
  by_pairs<CNT * 8>(v, [&](uint64_t x, int) { return mul2(x, pack2(rstd, rstd)); });
}

// Registers for 1024 threads an SM (64) where a block has half as many, so that two of them take turns between memory and barriers
// (4000 x 16384 to 8 bits 101 -> 76 us), and for skewed rows (8192 x 5001 111 -> 102); else for 768 (8192 x 8192 with both norms 86 us, 88
// with 64 registers). Five and six units a thread take the registers of 512 threads (8192 x 1280 with both norms 20.0, 21.0 with those of 640).
template <int CNT, int THREADS, bool ALIGNED>
constexpr int kNormBlocksPerSm = (CNT > 4 ? 512 : THREADS >= 512 || !ALIGNED ? 1024 : 768) / kTeamBlock<THREADS>;
// Vectors that rows share are loaded ahead of the statistics that come before their use where that fits these registers, which is where rows
// are few: in a graph 250 x 4096 to 8 bits with both norms and a gate 4.3 -> 4.0 us, 290 x 2048 3.6 -> 3.1, 100 x 1024 2.9 -> 2.6. With four units a
// thread it would take those of 640 threads (8192 x 4096 to 8 bits 45 -> 58), with five it gains nothing (8192 x 1280 20.0, 21.4), nor where a
// warp has a row, without barriers to wait at (24576 x 768 25.2, 26.2).
template <int CNT, int THREADS, bool ALIGNED>
constexpr bool kNormLoadsAhead = ALIGNED && THREADS > 32 && THREADS <= 256 && CNT <= 2;

template <int CNT, int THREADS, bool ALIGNED, bool QUANTIZE, bool BF16>
__global__ void __launch_bounds__(kTeamBlock<THREADS>, (kNormBlocksPerSm<CNT, THREADS, ALIGNED>)) residual_norm_kernel(const ResidualNormParams p) {
  grid_release();
  grid_wait();
  using Team = RowTeam<CNT, THREADS, ALIGNED>;
  __shared__ uint32_t words[5][32];
  __shared__ uint2 staged[kTeamBlock<THREADS> / THREADS][QUANTIZE ? Team::kStagedBytes / 8 : 1];
  const long long row = Team::row();
  if (row >= p.rows) return;
  const long long at = row * p.n, all = p.rows * p.n;
  const Team team(words, p.n, static_cast<const uint16_t*>(p.x) + at);
  const float inv_n = 1.f / static_cast<float>(p.n);
  const bool inner = row >= p.inside.begin && row < p.inside.end;
  uint4 xr[CNT], rr[CNT];
  auto fetch = [&](const void* tensor, uint4 (&raw)[CNT]) {
    const uint16_t* t = static_cast<const uint16_t*>(tensor);
#pragma unroll
    for (int i = 0; i < CNT; ++i) raw[i] = team.load(t + at, inner, t, t + all, i);
  };
  fetch(p.x, xr);
  if (p.residual != nullptr) fetch(p.residual, rr);
  float v[CNT * 8];
  auto clear_rest = [&] {
#pragma unroll
    for (int i = 0; i < CNT; ++i) team.clear_rest(&v[i * 8], i);
  };
#pragma unroll
  for (int i = 0; i < CNT; ++i) unpack8<BF16>(xr[i], &v[i * 8]);
  // A vector of those that rows share, and every pair of values with the same two of it. Where registers allow, it is on its way while the
  // statistics ahead of its use are taken.
  constexpr bool kAhead = kNormLoadsAhead<CNT, THREADS, ALIGNED>;
  uint4 ahead[2][kAhead ? CNT : 1];
  auto vector_of = [&](const void* vectors, const RowParts& part) {
    return static_cast<const uint16_t*>(vectors) + static_cast<long long>(part.of(row)) * p.n;
  };
  auto load_ahead = [&](const void* vectors, const RowParts& part, int slot) {
    if constexpr (kAhead) {
      if (vectors != nullptr) {
        const uint16_t* vector = vector_of(vectors, part);
#pragma unroll
        for (int i = 0; i < CNT; ++i) ahead[slot][i] = team.template load_off<false>(vector, i);
      }
    }
  };
  auto with = [&](const void* vectors, const RowParts& part, int slot, auto&& f) {
    const uint16_t* vector = kAhead && slot >= 0 ? nullptr : vector_of(vectors, part);
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      float a[8];
      unpack8<BF16>(kAhead && slot >= 0 ? ahead[slot < 0 ? 0 : slot][kAhead ? i : 0] : team.template load_off<false>(vector, i), a);
      by_pairs<8>(&v[i * 8], [&](uint64_t x, int j) { return f(x, pack2(a[j], a[j + 1])); });
    }
  };
  auto times = [](uint64_t x, uint64_t a) { return mul2(x, a); };
  auto plus = [](uint64_t x, uint64_t a) { return add2(x, a); };
  load_ahead(p.gate, p.gate_part, 1);
  if (p.post != kNormNone) {
    load_ahead(p.post_gamma, p.whole, 0);
    clear_rest();
    normalize_row(team, v, p.post, inv_n, p.eps, 0);
    if (p.post_gamma) with(p.post_gamma, p.whole, 0, times);
    if (p.post_beta) with(p.post_beta, p.whole, -1, plus);
  }
  if (p.gate) with(p.gate, p.gate_part, 1, times);
  if (p.residual != nullptr) {
    const uint64_t scale = pack2(p.residual_scale, p.residual_scale);
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      float r[8];
      unpack8<BF16>(rr[i], r);
      by_pairs<8>(&v[i * 8], [&](uint64_t a, int j) { return fma2(pack2(r[j], r[j + 1]), scale, a); });
    }
  }
  load_ahead(p.gamma, p.gamma_part, 0);
  load_ahead(p.beta, p.beta_part, 1);
  if (p.sum != nullptr) {
#pragma unroll
    for (int i = 0; i < CNT; ++i) team.template store<BF16>(static_cast<uint16_t*>(p.sum) + at, i, &v[i * 8]);
  }
  clear_rest();
  normalize_row(team, v, p.norm, inv_n, p.eps, 2);
  if (p.gamma) with(p.gamma, p.gamma_part, 0, times);
  if (p.beta) with(p.beta, p.beta_part, 1, plus);
  if constexpr (QUANTIZE) {
    clear_rest();
    uint32_t most = 0;
    take_magnitudes<CNT * 8>(most, v);
    const RowScale s = row_scale_of(team.most(most, 4));
    if (team.tid == 0) p.scale[row] = s.scale;
    uint2 b[CNT];
#pragma unroll
    for (int i = 0; i < CNT; ++i) b[i] = quantize_unit(s, &v[i * 8]);
    team.store_bytes(static_cast<int8_t*>(p.y) + row * p.y_pitch, b, staged[threadIdx.x / THREADS]);
  } else {
#pragma unroll
    for (int i = 0; i < CNT; ++i) team.template store<BF16>(static_cast<uint16_t*>(p.y) + at, i, &v[i * 8]);
  }
}

// Rows longer than the registers of a block hold, or operands that do not lie alike: a block walks its row once for each statistic and once to write,
// after the first time out of L2, and works the sum out anew each time. Bound by its loads of single elements: 1000 x 40000 with a residual takes 204 us
// (rms), 239 to 8 bits, 350 with both norms and a gate, where HBM would take 49, 43 and 49; 1000 x 32768, which fits, 47.
template <bool QUANTIZE, bool BF16>
__global__ void __launch_bounds__(kTeamMaxThreads) residual_norm_long_rows_kernel(const ResidualNormParams p) {
  using E = Elem16<BF16>;
  using T = typename E::T;
  __shared__ uint32_t words[5][32];
  const RowTeam<1, kTeamMaxThreads, true> team(words, p.n, nullptr);
  const long long row = blockIdx.x;
  const float inv_n = 1.f / static_cast<float>(p.n);
  auto at = [&](const void* base, long long r, int i) { return E::to_float(static_cast<const T*>(base)[r * p.n + i]); };
  auto statistics = [&](int kind, auto&& value, int slot, float& mean, float& rstd) {
    mean = 0.f;
    if (kind == kNormLayer) {
      float s = 0.f;
      for (int i = team.tid; i < p.n; i += kTeamMaxThreads) s += value(i);
      mean = team.sum(s, slot) * inv_n;
    }
    float q = 0.f;
    for (int i = team.tid; i < p.n; i += kTeamMaxThreads) {
      const float d = value(i) - mean;
      q = fmaf(d, d, q);
    }
    rstd = rsqrtf(fmaf(team.sum(q, slot + 1), inv_n, p.eps));
  };
  float post_mean = 0.f, post_rstd = 1.f, mean, rstd;
  if (p.post != kNormNone) statistics(p.post, [&](int i) { return at(p.x, row, i); }, 0, post_mean, post_rstd);
  auto total = [&](int i) {
    float v = at(p.x, row, i);
    if (p.post != kNormNone) {
      v = (v - post_mean) * post_rstd;
      if (p.post_gamma) v *= at(p.post_gamma, 0, i);
      if (p.post_beta) v += at(p.post_beta, 0, i);
    }
    if (p.gate) v *= at(p.gate, p.gate_part.of(row), i);
    return p.residual ? fmaf(p.residual_scale, at(p.residual, row, i), v) : v;
  };
  statistics(p.norm, total, 2, mean, rstd);
  auto result = [&](int i, float v) {
    v = (v - mean) * rstd;
    if (p.gamma) v *= at(p.gamma, p.gamma_part.of(row), i);
    if (p.beta) v += at(p.beta, p.beta_part.of(row), i);
    return v;
  };
  RowScale s;
  if constexpr (QUANTIZE) {
    uint32_t most = 0;
    for (int i = team.tid; i < p.n; i += kTeamMaxThreads) {
      const float y = result(i, total(i));
      take_magnitudes<1>(most, &y);
    }
    s = row_scale_of(team.most(most, 4));
    if (team.tid == 0) p.scale[row] = s.scale;
  }
  for (int i = team.tid; i < p.n; i += kTeamMaxThreads) {
    const float v = total(i), y = result(i, v);
    if (p.sum) static_cast<T*>(p.sum)[row * p.n + i] = E::from_float(v);
    if constexpr (QUANTIZE) {
      (static_cast<int8_t*>(p.y) + row * p.y_pitch)[i] = quantize_value(s, y);
    } else {
      static_cast<T*>(p.y)[row * p.n + i] = E::from_float(y);
    }
  }
}

template <int CNT, int THREADS, bool ALIGNED, bool QUANTIZE, bool BF16>
static void launch_residual_norm(const ResidualNormParams& p, cudaStream_t stream) {
  constexpr int kBlock = kTeamBlock<THREADS>;
  const long long blocks = THREADS > 32 ? p.rows : (p.rows + kTeamWarpsPerBlock - 1) / kTeamWarpsPerBlock;
  const auto kernel = &residual_norm_kernel<CNT, THREADS, ALIGNED, QUANTIZE, BF16>;
  static std::atomic<uint64_t> done{0};
  prefer_l1_once(done, reinterpret_cast<const void*>(kernel), kBlock);
  const bool early = blocks_start_early(blocks, kBlock, sm_count(), 2048) || !in_capture(stream);
  launch_early(kernel, dim3(static_cast<unsigned>(blocks)), kBlock, 0, stream, early, 1, p);
}

template <bool QUANTIZE, bool BF16>
static void residual_norm_dispatch(const ResidualNormParams& p, bool lie_well, bool aligned, cudaStream_t stream) {
  // us with one / two / four units a thread, to 8 bits: 100 x 1024 2.3 / 2.1 / 2.5, x 4096 2.6 / 2.4 / 2.4, x 8192 3.9 / 3.4 / 3.3; with both norms
  // 100 x 2048 3.3 / 3.1 / 3.5, 333 x 4096 5.3 / 4.9 / 5.2, 600 x 4096 8.4 / 7.1 / 6.1, 2000 x 1280 10.0 / 7.6 / 7.0
  const TeamShape t = team_shape(p.rows, p.n, aligned, 2ll * sm_count(), 2);
  if (t.cnt == 0 || !lie_well) {
    count_launch();
    residual_norm_long_rows_kernel<QUANTIZE, BF16><<<static_cast<unsigned>(p.rows), kTeamMaxThreads, 0, stream>>>(p);
    B200AIT_CUDA_CHECK(cudaGetLastError());
    return;
  }
  for_team_shape<2>(t, [&](auto cnt, auto threads, auto whole) {
    launch_residual_norm<decltype(cnt)::value, decltype(threads)::value, decltype(whole)::value, QUANTIZE, BF16>(p, stream);
  });
}

}  // namespace b200ait

using namespace b200ait;

B200AIT_EXPORT int b200ait_residual_norm(void* sum, void* y, float* y_scale, const void* x, const void* residual,
                                         const void* gate, const void* post_gamma, const void* post_beta, const void* gamma,
                                         const void* beta, int64_t rows, int64_t n, int64_t gates, int64_t gammas, int64_t betas,
                                         int64_t y_pitch, int post_norm, int norm, float residual_scale, float eps, int dtype,
                                         cudaStream_t stream) {
  return guarded("b200ait_residual_norm", [&] {
    B200AIT_REQUIRE(dtype == kDTypeHalf || dtype == kDTypeBFloat16, "residual_norm: dtype must be float16 or bfloat16");
    B200AIT_REQUIRE(rows >= 0 && n >= 0, "residual_norm: negative dimension");
    B200AIT_REQUIRE(norm == kNormLayer || norm == kNormRms, "residual_norm: the norm is layer (1) or rms (2)");
    B200AIT_REQUIRE(post_norm >= kNormNone && post_norm <= kNormRms, "residual_norm: the norm after the block is none (0), layer (1) or rms (2)");
    B200AIT_REQUIRE(post_norm != kNormNone || (!post_gamma && !post_beta), "residual_norm: post_gamma and post_beta need a norm after the block");
    if (rows == 0) return;
    B200AIT_REQUIRE(n != 0 || !y_scale, "residual_norm: the rows have no columns");  // (and so no largest value to scale by)
    if (n == 0) return;
    B200AIT_REQUIRE(x && y, "residual_norm: null pointer with non-zero size");
    B200AIT_REQUIRE(rows < (1ll << 31) && n < (1ll << 30), "residual_norm: dimension exceeds int32");
    const bool quantize = y_scale != nullptr;
    B200AIT_REQUIRE(!quantize || y_pitch >= n, "residual_norm: a row pitch is shorter than the row");
    ResidualNormParams p{x, residual, gate, post_gamma, post_beta, gamma, beta, sum, y, y_scale, rows, y_pitch, inner_rows(rows, n),
                         {}, {}, {}, {},
                         static_cast<int>(n), post_norm, norm, residual_scale, eps};
    p.whole.rows = static_cast<int>(rows);
    p.whole.mul = FastDiv(p.whole.rows).mul, p.whole.shr = FastDiv(p.whole.rows).shr;
    auto part = [&](const void* ptr, int64_t count, const char* what, RowParts& parts) {
      if (!ptr) return;
      B200AIT_REQUIRE(count > 0 && rows % count == 0, std::string("residual_norm: the rows do not fall into equal parts, one for each ") + what);
      const FastDiv by(static_cast<int>(rows / count));
      parts.rows = static_cast<int>(rows / count), parts.mul = by.mul, parts.shr = by.shr;
    };
    part(gate, gates, "gate", p.gate_part);
    part(gamma, gammas, "gamma", p.gamma_part);
    part(beta, betas, "beta", p.beta_part);
    for (const void* ptr : {x, residual, gate, post_gamma, post_beta, gamma, beta, static_cast<const void*>(sum)})
      B200AIT_REQUIRE(multiple_of(ptr, 2), "residual_norm: a pointer is not aligned to its type");
    B200AIT_REQUIRE(multiple_of(y, quantize ? 1 : 2) && multiple_of(y_scale, 4), "residual_norm: a pointer is not aligned to its type");
    const bool lie_well = quantize ? lie_alike({x, residual, sum}) && multiple_of(y, 8) && y_pitch % 8 == 0 : lie_alike({x, residual, sum, y});
    bool aligned = n % 8 == 0 && multiple_of(x, 16);
    for (const void* vector : {gate, post_gamma, post_beta, gamma, beta}) aligned = aligned && multiple_of(vector, 16);
    const bool bf16 = dtype == kDTypeBFloat16;
    if (quantize && bf16)
      residual_norm_dispatch<true, true>(p, lie_well, aligned, stream);
    else if (quantize)
      residual_norm_dispatch<true, false>(p, lie_well, aligned, stream);
    else if (bf16)
      residual_norm_dispatch<false, true>(p, lie_well, aligned, stream);
    else
      residual_norm_dispatch<false, false>(p, lie_well, aligned, stream);
  });
}
