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

struct ResidualNormParams {
  const void *x, *residual, *gate, *post_gamma, *post_beta, *gamma, *beta;
  void *sum, *y;
  float* scale;  // of y in 8 bits
  long long rows, y_pitch;
  long long gate_part, gamma_part, beta_part;  // rows that share a vector
  int n, post, norm;
  float residual_scale, eps;
};

// normalises the row in `v`: layer or rms, without gamma and beta. `slot` and slot + 1 are the reductions' words.
template <int VEC, int CNT, bool BLOCK>
__device__ __forceinline__ void normalize_row(const RowTeam<BLOCK>& team, float (&v)[CNT * VEC], int kind, int units, float inv_n,
                                              float eps, int slot) {
  float mean = 0.f;
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < CNT * VEC; ++i) s += v[i];  // (past the end of the row are zeros)
    mean = team.sum(s, slot) * inv_n;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    if (team.tid + i * team.threads < units) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = v[i * VEC + j] - mean;
        q = fmaf(d, d, q);
      }
    }
  }
  const float rstd = rsqrtf(fmaf(team.sum(q, slot + 1), inv_n, eps));
#pragma unroll
  for (int i = 0; i < CNT * VEC; ++i) v[i] = (v[i] - mean) * rstd;
}

template <int VEC, int CNT, int MOST, bool QUANTIZE, bool BF16>
__global__ void __launch_bounds__(kTeamBlock<MOST>)
    residual_norm_kernel(const ResidualNormParams p) {
  grid_release();
  grid_wait();
  constexpr bool BLOCK = MOST > 32;
  using T = typename Elem16<BF16>::T;
  using Raw = RawUnit<VEC>;
  using Unit = typename Raw::Type;
  __shared__ uint32_t words[5][32];
  const RowTeam<BLOCK> team{words, BLOCK ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x & 31),
                            BLOCK ? static_cast<int>(blockDim.x) : 32};
  const long long row = BLOCK ? static_cast<long long>(blockIdx.x)
                              : static_cast<long long>(blockIdx.x) * kTeamWarpsPerBlock + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int units = p.n / VEC;
  const float inv_n = 1.f / static_cast<float>(p.n);
  auto unit_at = [&](int i) { return team.tid + i * team.threads; };
  auto row_of = [&](const void* base, long long r) { return reinterpret_cast<const Unit*>(static_cast<const T*>(base) + r * p.n); };
  Unit xr[CNT], rr[CNT];
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    const int u = unit_at(i);
    xr[i] = u < units ? ld_stream(row_of(p.x, row) + u) : Raw::zero();
    rr[i] = p.residual != nullptr && u < units ? ld_stream(row_of(p.residual, row) + u) : Raw::zero();
  }
  float v[CNT * VEC];
#pragma unroll
  for (int i = 0; i < CNT; ++i) unpack_unit<VEC, BF16>(xr[i], &v[i * VEC]);
  // v *= a or v += a, for a vector that rows share
  auto times = [&](const void* base, long long r) {
    const Unit* a = row_of(base, r);
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      float f[VEC];
      unpack_unit<VEC, BF16>(unit_at(i) < units ? a[unit_at(i)] : Raw::zero(), f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i * VEC + j] *= f[j];
    }
  };
  auto plus = [&](const void* base, long long r) {
    const Unit* a = row_of(base, r);
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      float f[VEC];
      unpack_unit<VEC, BF16>(unit_at(i) < units ? a[unit_at(i)] : Raw::zero(), f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i * VEC + j] += f[j];
    }
  };
  if (p.post != kNormNone) {
    normalize_row<VEC, CNT, BLOCK>(team, v, p.post, units, inv_n, p.eps, 0);
    if (p.post_gamma) times(p.post_gamma, 0);
    if (p.post_beta) plus(p.post_beta, 0);
  }
  if (p.gate) times(p.gate, row / p.gate_part);
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    float f[VEC];
    unpack_unit<VEC, BF16>(rr[i], f);
    const bool inside = unit_at(i) < units;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i * VEC + j] = inside ? fmaf(p.residual_scale, f[j], v[i * VEC + j]) : 0.f;
    if (p.sum != nullptr && inside)
      store_unit<VEC, BF16>(static_cast<T*>(p.sum) + row * p.n, unit_at(i), &v[i * VEC]);
  }
  normalize_row<VEC, CNT, BLOCK>(team, v, p.norm, units, inv_n, p.eps, 2);
  if (p.gamma) times(p.gamma, row / p.gamma_part);
  if (p.beta) plus(p.beta, row / p.beta_part);
  if constexpr (QUANTIZE) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      if (unit_at(i) < units) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) most = max(most, magnitude_bits(v[i * VEC + j]));
      }
    }
    const RowScale s = row_scale_of(team.most(most, 4));
    if (team.tid == 0) p.scale[row] = s.scale;
    int8_t* q = static_cast<int8_t*>(p.y) + row * p.y_pitch;
#pragma unroll
    for (int i = 0; i < CNT; ++i)
      if (unit_at(i) < units) store_quantized<VEC>(q, unit_at(i), s, &v[i * VEC]);
  } else {
#pragma unroll
    for (int i = 0; i < CNT; ++i)
      if (unit_at(i) < units) store_unit<VEC, BF16>(static_cast<T*>(p.y) + row * p.n, unit_at(i), &v[i * VEC]);
  }
}

// Rows longer than the registers of a block hold: a block walks its row once for each statistic and once to write, after the first
// time out of L2, and works the sum out anew each time.
template <bool QUANTIZE, bool BF16>
__global__ void __launch_bounds__(kTeamMaxThreads) residual_norm_long_rows_kernel(const ResidualNormParams p) {
  using E = Elem16<BF16>;
  using T = typename E::T;
  __shared__ uint32_t words[5][32];
  const RowTeam<true> team{words, static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x)};
  const long long row = blockIdx.x;
  const float inv_n = 1.f / static_cast<float>(p.n);
  auto at = [&](const void* base, long long r, int i) { return E::to_float(static_cast<const T*>(base)[r * p.n + i]); };
  auto statistics = [&](int kind, auto&& value, int slot, float& mean, float& rstd) {
    mean = 0.f;
    if (kind == kNormLayer) {
      float s = 0.f;
      for (int i = team.tid; i < p.n; i += team.threads) s += value(i);
      mean = team.sum(s, slot) * inv_n;
    }
    float q = 0.f;
    for (int i = team.tid; i < p.n; i += team.threads) {
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
    if (p.gate) v *= at(p.gate, row / p.gate_part, i);
    return p.residual ? fmaf(p.residual_scale, at(p.residual, row, i), v) : v;
  };
  statistics(p.norm, total, 2, mean, rstd);
  auto result = [&](int i, float v) {
    v = (v - mean) * rstd;
    if (p.gamma) v *= at(p.gamma, row / p.gamma_part, i);
    if (p.beta) v += at(p.beta, row / p.beta_part, i);
    return v;
  };
  RowScale s;
  if constexpr (QUANTIZE) {
    uint32_t most = 0;
    for (int i = team.tid; i < p.n; i += team.threads) most = max(most, magnitude_bits(result(i, total(i))));
    s = row_scale_of(team.most(most, 4));
    if (team.tid == 0) p.scale[row] = s.scale;
  }
  for (int i = team.tid; i < p.n; i += team.threads) {
    const float v = total(i), y = result(i, v);
    if (p.sum) static_cast<T*>(p.sum)[row * p.n + i] = E::from_float(v);
    if constexpr (QUANTIZE) {
      store_quantized<1>(static_cast<int8_t*>(p.y) + row * p.y_pitch, i, s, &y);
    } else {
      static_cast<T*>(p.y)[row * p.n + i] = E::from_float(y);
    }
  }
}

template <int VEC, int CNT, int MOST, bool QUANTIZE, bool BF16>
static void launch_residual_norm(const ResidualNormParams& p, int threads, cudaStream_t stream) {
  constexpr bool BLOCK = MOST > 32;
  const long long blocks = BLOCK ? p.rows : (p.rows + kTeamWarpsPerBlock - 1) / kTeamWarpsPerBlock;
  const int block = BLOCK ? threads : 32 * kTeamWarpsPerBlock;
  const bool early = blocks_start_early(blocks, block, sm_count(), 2048) || !in_capture(stream);
  launch_early(&residual_norm_kernel<VEC, CNT, MOST, QUANTIZE, BF16>, dim3(static_cast<unsigned>(blocks)), block, 0, stream, early, 1,
               p);
}

template <bool QUANTIZE, bool BF16>
static void residual_norm_dispatch(const ResidualNormParams& p, bool vector_ok, cudaStream_t stream) {
  const TeamShape t = team_shape(p.rows, p.n, vector_ok, sm_count());
  if (t.cnt == 0) {
    count_launch();
    residual_norm_long_rows_kernel<QUANTIZE, BF16><<<static_cast<unsigned>(p.rows), t.threads, 0, stream>>>(p);
    B200AIT_CUDA_CHECK(cudaGetLastError());
    return;
  }
  for_team_shape(t, [&](auto vec, auto cnt, auto most) {
    launch_residual_norm<decltype(vec)::value, decltype(cnt)::value, decltype(most)::value, QUANTIZE, BF16>(p, t.threads, stream);
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
    if (rows == 0 || n == 0) return;
    B200AIT_REQUIRE(x && y, "residual_norm: null pointer with non-zero size");
    B200AIT_REQUIRE(rows < (1ll << 31) && n < (1ll << 30), "residual_norm: dimension exceeds int32");
    const bool quantize = y_scale != nullptr;
    B200AIT_REQUIRE(!quantize || y_pitch >= n, "residual_norm: a row pitch is shorter than the row");
    ResidualNormParams p{x, residual, gate, post_gamma, post_beta, gamma, beta, sum, y, y_scale, rows, y_pitch, rows, rows, rows,
                         static_cast<int>(n), post_norm, norm, residual_scale, eps};
    auto part = [&](const void* ptr, int64_t count, const char* what, long long& rows_of_part) {
      if (!ptr) return;
      B200AIT_REQUIRE(count > 0 && rows % count == 0, std::string("residual_norm: the rows do not fall into equal parts, one for each ") + what);
      rows_of_part = rows / count;
    };
    part(gate, gates, "gate", p.gate_part);
    part(gamma, gammas, "gamma", p.gamma_part);
    part(beta, betas, "beta", p.beta_part);
    bool vector_ok = n % 8 == 0;
    for (const void* ptr : {x, residual, gate, post_gamma, post_beta, gamma, beta, static_cast<const void*>(sum)})
      vector_ok = vector_ok && (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0;
    vector_ok = vector_ok && (quantize ? (reinterpret_cast<uintptr_t>(y) & 7u) == 0 && y_pitch % 8 == 0
                                       : (reinterpret_cast<uintptr_t>(y) & 15u) == 0);
    const bool bf16 = dtype == kDTypeBFloat16;
    if (quantize && bf16)
      residual_norm_dispatch<true, true>(p, vector_ok, stream);
    else if (quantize)
      residual_norm_dispatch<true, false>(p, vector_ok, stream);
    else if (bf16)
      residual_norm_dispatch<false, true>(p, vector_ok, stream);
    else
      residual_norm_dispatch<false, false>(p, vector_ok, stream);
  });
}
