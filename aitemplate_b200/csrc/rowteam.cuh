// What the kernels share that hold a row in registers from its one read to its one write: a warp or a block ("team") per row, CNT
// units of VEC elements a thread, unit i of thread t at t + i * team. Reductions over the row, and the step from fp32 values to
// signed 8-bit ones with a scale per row.
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "epilogue.cuh"
#include "ptx.cuh"
#include "rules.h"

namespace b200ait {

constexpr int kTeamMaxThreads = 1024;
constexpr int kTeamWarpsPerBlock = 8;  // rows of a block where a warp takes a row

// threads of a block whose teams have up to MOST
template <int MOST>
constexpr int kTeamBlock = MOST == 32 ? 32 * kTeamWarpsPerBlock : MOST;

// A reduction needs one barrier: each has words of its own (`slot`), so no thread can overwrite what another still reads.
template <bool BLOCK>
struct RowTeam {
  uint32_t (*words)[32];  // [slots][warps], shared
  int tid, threads;

  __device__ __forceinline__ float sum(float v, int slot) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (BLOCK) {
      const int lane = tid & 31;
      if (lane == 0) words[slot][tid >> 5] = __float_as_uint(v);
      __syncthreads();
      v = lane < (threads >> 5) ? __uint_as_float(words[slot][lane]) : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
  }
  // the largest of unsigned words
  __device__ __forceinline__ uint32_t most(uint32_t v, int slot) const {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (BLOCK) {
      const int lane = tid & 31;
      if (lane == 0) words[slot][tid >> 5] = v;
      __syncthreads();
      v = __reduce_max_sync(0xffffffffu, lane < (threads >> 5) ? words[slot][lane] : 0u);
    }
    return v;
  }
};

// VEC elements as they lie in memory
template <int VEC>
struct RawUnit;
template <>
struct RawUnit<8> {
  using Type = uint4;
  static __device__ __forceinline__ uint4 zero() { return make_uint4(0, 0, 0, 0); }
};
template <>
struct RawUnit<1> {
  using Type = uint16_t;
  static __device__ __forceinline__ uint16_t zero() { return 0; }
};
template <int VEC, bool BF16>
__device__ __forceinline__ void unpack_unit(const typename RawUnit<VEC>::Type& raw, float* f) {
  if constexpr (VEC == 8) {
    unpack8<BF16>(raw, f);
  } else {
    f[0] = Elem16<BF16>::to_float(*reinterpret_cast<const typename Elem16<BF16>::T*>(&raw));
  }
}
template <int VEC, bool BF16>
__device__ __forceinline__ void store_unit(void* base, long long unit, const float* f) {
  if constexpr (VEC == 8) {
    static_cast<uint4*>(base)[unit] = pack8<BF16>(f);
  } else {
    static_cast<typename Elem16<BF16>::T*>(base)[unit] = Elem16<BF16>::from_float(f[0]);
  }
}

// ------------------------------------------------------------------------------------------------ 8-bit values
// q = round(127 v / amax), ties to even, with amax the largest |v| of the row; scale = amax / 127.
//
// The quotient is formed so that for 16-bit v its rounding is that of the exact quotient: r0 = v * (127 / amax) is a step or so of
// fp32 off; its remainder 127 v - r0 * amax is exact in one FMA (127 v has at most 18 bits), and r0 + remainder / amax is then the
// nearest fp32 to the quotient. 127 v / amax is a tie only where it is one exactly, and away from ties it keeps more than 2^-20 of its
// own size from them (both mantissas have at most 11 bits), sixteen steps of fp32. Adding 1.5 * 2^23 rounds to a whole number, ties to
// even, and leaves it in the low bits. Five packed instructions for two values; a division would take eight for each.
//
// The largest |v| is found among the bit patterns without their sign, as integers: it has no trouble with values under 2^-126,
// which the compiler's arithmetic here takes for zero, and infinities and NaN come out on top.
struct RowScale {
  float scale;                // what one step of q is worth
  float prescale, amax, inv, back;  // amax after prescaling, 127 / amax, 1 / amax
  bool flat;                  // all q are 0: a row of zeros (scale 0), or one with an infinity or NaN in it (scale NaN)
};
__device__ __forceinline__ float mul_exact(float a, float b) {  // without flushing small values to zero
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ RowScale row_scale_of(uint32_t amax_bits) {
  RowScale s;
  const float amax = __uint_as_float(amax_bits);
  asm("div.rn.f32 %0, %1, %2;" : "=f"(s.scale) : "f"(amax), "f"(127.f));
  const bool finite = amax_bits < 0x7f800000u;
  if (!finite) s.scale = __uint_as_float(0x7fffffffu);
  s.flat = amax_bits == 0u || !finite;
  // 127 v must not overflow, and 1 / amax neither
  s.prescale = amax > 0x1p100f ? 0x1p-64f : amax < 0x1p-60f ? 0x1p64f : 1.f;
  s.amax = mul_exact(amax, s.prescale);
  s.inv = __fdiv_rn(127.f, s.amax);
  s.back = __fdiv_rn(1.f, s.amax);
  return s;
}
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// N values (N even) -> N bytes in N / 4 words (one value: N = 1)
template <int N>
__device__ __forceinline__ void quantize_values(const RowScale& s, const float* v, uint32_t* words) {
  static_assert(N == 1 || N % 4 == 0, "whole words");
  uint32_t b[N == 1 ? 2 : N];
  const uint64_t inv = pack2(s.inv, s.inv), back = pack2(s.back, s.back), less = pack2(-s.amax, -s.amax);
  const uint64_t steps = pack2(127.f, 127.f), whole = pack2(12582912.f, 12582912.f);
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    float v0 = v[j], v1 = N == 1 ? 0.f : v[j + 1];
    if (s.prescale != 1.f) v0 = mul_exact(v0, s.prescale), v1 = mul_exact(v1, s.prescale);
    const uint64_t x = pack2(v0, v1);
    const uint64_t r0 = mul2(x, inv), r = fma2(fma2(r0, less, mul2(x, steps)), back, r0);
    float m0, m1;
    unpack2(add2(r, whole), m0, m1);
    b[j] = __float_as_uint(m0), b[j + 1] = __float_as_uint(m1);
  }
  if constexpr (N == 1) {
    words[0] = s.flat ? 0u : b[0] & 0xffu;
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const uint32_t lo = __byte_perm(b[j], b[j + 1], 0x0040), hi = __byte_perm(b[j + 2], b[j + 3], 0x0040);
      words[j / 4] = s.flat ? 0u : __byte_perm(lo, hi, 0x5410);
    }
  }
}
template <int VEC>
__device__ __forceinline__ void store_quantized(int8_t* row, long long unit, const RowScale& s, const float* v) {
  uint32_t w[VEC == 8 ? 2 : 1];
  quantize_values<VEC>(s, v, w);
  if constexpr (VEC == 8) {
    reinterpret_cast<uint2*>(row)[unit] = make_uint2(w[0], w[1]);
  } else {
    row[unit] = static_cast<int8_t>(w[0]);
  }
}

// ------------------------------------------------------------------------------------------------ host
// How a row of n elements is laid over threads: `cnt` units of `vec` elements each (0: the row is too long and is walked), by a warp
// (most = 32) or by a block of `threads` whose kernel is built for up to `most`.
struct TeamShape {
  int vec, cnt, threads, most;
};
inline TeamShape team_shape(long long rows, long long n, bool vector_ok, int sms) {
  auto shape = [](int vec, long long units, long long per) {
    const int t = static_cast<int>(std::max<long long>(32, ((units + per - 1) / per + 31) / 32 * 32));
    const int cnt = static_cast<int>(std::max<long long>(1, (units + t - 1) / t));
    return TeamShape{vec, cnt, t, t == 32 && vec == 8 ? 32 : t <= 256 ? 256 : t <= 512 ? 512 : 1024};
  };
  if (!vector_ok) {
    if (n > 32ll * kTeamMaxThreads) return TeamShape{1, 0, kTeamMaxThreads, kTeamMaxThreads};
    TeamShape t = shape(1, n, n <= 8ll * kTeamMaxThreads ? 8 : 32);
    t.cnt = n <= 8ll * kTeamMaxThreads ? 8 : 32, t.most = kTeamMaxThreads;
    return t;
  }
  const long long units = n / 8;
  if (units > 4ll * kTeamMaxThreads) return TeamShape{8, 0, kTeamMaxThreads, kTeamMaxThreads};
  // A few rows are a matter of latency: a unit a thread. Many are one of bytes in flight: up to four.
  return shape(8, units, rows <= 2ll * sms && units <= kTeamMaxThreads ? 1 : 4);
}

// Calls `launch` with (VEC, CNT, MOST) as compile-time numbers. Of block-wide shapes with 16-byte units only these come about: one unit
// a thread, or four, and three where a block has 64 or 96 threads.
template <int N>
using TeamInt = std::integral_constant<int, N>;
template <class F>
inline void for_team_shape(const TeamShape& t, F&& launch) {
  switch (t.vec * 100000 + t.most * 10 + (t.vec == 8 ? t.cnt : t.cnt == 32 ? 1 : 0)) {
#define B200AIT_TEAM(VEC, CNT, MOST) \
  case (VEC) * 100000 + (MOST) * 10 + ((VEC) == 8 ? (CNT) : (CNT) == 32 ? 1 : 0): return launch(TeamInt<VEC>{}, TeamInt<CNT>{}, TeamInt<MOST>{});
    B200AIT_TEAM(8, 1, 32) B200AIT_TEAM(8, 2, 32) B200AIT_TEAM(8, 3, 32) B200AIT_TEAM(8, 4, 32)
    B200AIT_TEAM(8, 1, 256) B200AIT_TEAM(8, 3, 256) B200AIT_TEAM(8, 4, 256)
    B200AIT_TEAM(8, 1, 512) B200AIT_TEAM(8, 4, 512) B200AIT_TEAM(8, 1, 1024) B200AIT_TEAM(8, 4, 1024)
    B200AIT_TEAM(1, 8, 1024) B200AIT_TEAM(1, 32, 1024)
#undef B200AIT_TEAM
  }
  throw Error("no kernel for rows of this length");
}

}  // namespace b200ait
