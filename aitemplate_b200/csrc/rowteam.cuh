// What the kernels share that hold a row in registers from its one read to its one write: a team of THREADS threads (a warp, or
// a whole block) per row, CNT units of 8 elements a thread, unit i of thread t at t + i * THREADS. Reductions over the row, and the
// step from fp32 values to signed 8-bit ones with a scale per row.
//
// With norms on both sides of a block these kernels are bound by how many instructions a value takes as much as by HBM (8192 x 4096, both
// norms, to 8 bits: 40 a value and 59 us with THREADS read from the launch and every access checked). So THREADS is known at
// compile time, which leaves one address per operand and row, only the last unit of a thread can lie past the end of the row, what an
// operand does to the row is asked once per row, and arithmetic takes two values at a time.
//
// ALIGNED: rows start on 16 bytes and hold whole units. Otherwise units are cut where the 16-byte boundaries of the row's memory lie,
// so that its elements still move 16 bytes at a time (all of the [rows, n] operands of a call lie alike, the host sees to it): the
// first unit lacks its first `skew` elements, the last one its end, which are read along and left out, and written element by element. Vectors that rows share,
// and 8-bit results, whose rows start on 16 bytes, then lie off the units: two loads and a shift of the words, or a way through shared
// memory. Element by element throughout, 8192 x 1001 with both norms took 33 us (25.7 so), 8192 x 5001 to
// 8 bits 226 (102).
#pragma once
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "common.h"
#include "epilogue.cuh"
#include "ptx.cuh"
#include "rules.h"

namespace b200ait {

constexpr int kTeamMaxThreads = 1024;
constexpr int kTeamWarpsPerBlock = 4;  // rows of a block where a warp takes a row

template <int THREADS>
constexpr int kTeamBlock = THREADS == 32 ? 32 * kTeamWarpsPerBlock : THREADS;

// Eight elements of a unit that reaches over an end of the memory [lo, hi). (Inlined at every load it filled the instruction cache.)
static __device__ __noinline__ uint4 load_elements(const uint16_t* at, const uint16_t* lo, const uint16_t* hi) {
  uint32_t e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = at + j >= lo && at + j < hi ? at[j] : 0u;
  return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}
// The elements from .. to - 1 of a unit, one by one
static __device__ __noinline__ void store_elements(uint16_t* at, uint4 v, int from, int to) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j >= from && j < to) at[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
}

// A reduction needs one barrier: each has words of its own (`slot`), so no thread can overwrite what another still reads.
template <int CNT, int THREADS, bool ALIGNED>
struct RowTeam {
  static constexpr bool kBlock = THREADS > 32;
  uint32_t (*words)[32];  // [slots][warps], shared
  int tid, units, n, skew;

  // `row`: where the row starts in one of the operands that lie alike
  __device__ __forceinline__ RowTeam(uint32_t (*w)[32], int columns, const void* row)
      : words(w), tid(kBlock ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x & 31)), n(columns),
        skew(ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 1) & 7) {
    units = (n + skew + 7) >> 3;
  }
  static __device__ __forceinline__ long long row() {
    return kBlock ? static_cast<long long>(blockIdx.x)
                  : static_cast<long long>(blockIdx.x) * kTeamWarpsPerBlock + (threadIdx.x >> 5);
  }
  __device__ __forceinline__ int unit(int i) const { return tid + i * THREADS; }
  // (of aligned rows the host takes as few units a thread as the row allows)
  __device__ __forceinline__ bool has(int i) const { return (ALIGNED && i < CNT - 1) || unit(i) < units; }
  // element of the row that unit i starts with (negative for the first one of a skewed row), and which of its 8 are the row's
  __device__ __forceinline__ int first(int i) const { return unit(i) * 8 - skew; }
  __device__ __forceinline__ int from(int i) const { return max(0, -first(i)); }
  __device__ __forceinline__ int to(int i) const { return min(8, n - first(i)); }
  __device__ __forceinline__ bool whole(int i) const { return ALIGNED || (first(i) >= 0 && first(i) + 8 <= n); }

  __device__ __forceinline__ float sum(float v, int slot) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (kBlock) {
      if ((tid & 31) == 0) words[slot][tid >> 5] = __float_as_uint(v);
      __syncthreads();
      v = (tid & 31) < THREADS / 32 ? __uint_as_float(words[slot][tid & 31]) : 0.f;
#pragma unroll
      for (int o = THREADS / 64; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if constexpr (THREADS < 1024) v = __shfl_sync(0xffffffffu, v, 0);
    }
    return v;
  }
  // the largest of unsigned words
  __device__ __forceinline__ uint32_t most(uint32_t v, int slot) const {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (kBlock) {
      if ((tid & 31) == 0) words[slot][tid >> 5] = v;
      __syncthreads();
      v = __reduce_max_sync(0xffffffffu, (tid & 31) < THREADS / 32 ? words[slot][tid & 31] : 0u);
    }
    return v;
  }

  // Unit i of a row of an operand whose memory starts at `lo` and ends at `hi`. What is not the row's holds anything (clear_rest): a unit
  // that reaches over the row's ends takes its neighbours' elements along, which are the operand's own for an `inner` row (inner_rows).
  __device__ __forceinline__ uint4 load(const uint16_t* row, bool inner, const uint16_t* lo, const uint16_t* hi, int i) const {
    if (!has(i)) return make_uint4(0, 0, 0, 0);
    const uint16_t* at = row - skew + unit(i) * 8;
    if (ALIGNED || inner || whole(i)) return ld_stream(reinterpret_cast<const uint4*>(at));
    return load_elements(at, lo, hi);
  }
  // The same elements of a row that may lie at another place of 16 bytes than the team's: the two pieces that hold them, shifted by
  // words and by half a word.
  template <bool STREAM>
  __device__ __forceinline__ uint4 load_off(const uint16_t* row, int i) const {
    if (!has(i)) return make_uint4(0, 0, 0, 0);
    auto fetch = [](const uint16_t* at) {
      return STREAM ? ld_stream(reinterpret_cast<const uint4*>(at)) : *reinterpret_cast<const uint4*>(at);
    };
    const uint16_t* at = row + first(i);
    if (ALIGNED) return fetch(at);
    if (first(i) < 8 || first(i) + 16 > n) return load_elements(at, row, row + n);
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(at) >> 1) & 7;
    const uint4 a = fetch(at - off), b = fetch(at - off + 8);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (off & 4) {
#pragma unroll
      for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
    }
    if (off & 2) {
#pragma unroll
      for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
    }
    if (off & 1) {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // zeros for what is not the row's
  __device__ __forceinline__ void clear_rest(float* v, int i) const {
    if (ALIGNED ? has(i) : has(i) && whole(i)) return;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (!has(i) || j < from(i) || j >= to(i)) v[j] = 0.f;
  }
  template <bool BF16>
  __device__ __forceinline__ void store(uint16_t* row, int i, const float* v) const {
    if (!has(i)) return;
    const uint4 packed = pack8<BF16>(v);
    if (whole(i)) {
      reinterpret_cast<uint4*>(row - skew)[unit(i)] = packed;
      return;
    }
    store_elements(row + first(i), packed, from(i), to(i));
  }
  // The row as 8-bit values into one that starts on 8 bytes; every thread of the team calls it. The units of a skewed row lie off
  // those 8 bytes: they go through shared memory (`staged`), where a thread takes its 8 bytes out of the two units that hold them.
  static constexpr int kStagedBytes = ALIGNED ? 8 : CNT * THREADS * 8 + 8;
  __device__ __forceinline__ void store_bytes(int8_t* row, const uint2 (&b)[CNT], uint2* staged) const {
    if constexpr (ALIGNED) {
#pragma unroll
      for (int i = 0; i < CNT; ++i)
        if (has(i)) reinterpret_cast<uint2*>(row)[unit(i)] = b[i];
    } else {
#pragma unroll
      for (int i = 0; i < CNT; ++i) staged[unit(i)] = b[i];
      if constexpr (kBlock) {
        __syncthreads();
      } else {
        __syncwarp();
      }
      const int shift = 8 * skew;
#pragma unroll
      for (int i = 0; i < CNT; ++i) {
        const int g = unit(i), left = n - 8 * g;
        if (left <= 0) continue;
        const uint2 lo = staged[g], hi = staged[g + 1];  // (what is behind the last unit is not used)
        uint64_t v = (static_cast<uint64_t>(lo.y) << 32 | lo.x) >> shift;
        if (skew != 0) v |= (static_cast<uint64_t>(hi.y) << 32 | hi.x) << (64 - shift);
        if (left >= 8) {
          reinterpret_cast<uint64_t*>(row)[g] = v;
        } else {
          for (int j = 0; j < left; ++j) row[8 * g + j] = static_cast<int8_t>(v >> (8 * j));
        }
      }
    }
  }
};

// Arithmetic two values at a time
template <int N, class F>
__device__ __forceinline__ void by_pairs(float* v, F&& f) {  // v[j], v[j + 1] = f(pair, j)
#pragma unroll
  for (int j = 0; j < N; j += 2) unpack2(f(pack2(v[j], v[j + 1]), j), v[j], v[j + 1]);
}

// ------------------------------------------------------------------------------------------------ 8-bit values
// q = round(127 v / amax), ties to even, with amax the largest |v| of the row; scale = amax / 127.
//
// The quotient is formed so that for 16-bit v its rounding is that of the exact quotient: r0 = v * (127 / amax) is a step or so of
// fp32 off; its remainder 127 v - r0 * amax is exact in one FMA (127 v has at most 18 bits), and r0 + remainder / amax is then the
// nearest fp32 to the quotient. 127 v / amax is a tie only where it is one exactly, and away from ties it keeps more than 2^-20 of its
// own size from them (both mantissas have at most 11 bits), eight steps of fp32. Adding 1.5 * 2^23 rounds to a whole number, ties to
// even, and leaves it in the low bits. Five packed instructions for two values; a division would take eight for each.
//
// The largest |v| is looked for without flushing values under 2^-126 to zero, as the compiler's arithmetic here would, and in such a way
// that NaN comes out on top; across threads it is compared as an integer (the bits of a magnitude are ordered as it is).
struct RowScale {
  float scale;                // what one step of q is worth
  float prescale, amax, inv, back;  // amax after prescaling, 127 / amax, 1 / amax
  bool flat;                  // all q are 0: a row of zeros (scale 0), or one with an infinity or NaN in it (scale NaN)
};
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
// the bits of the larger of `most` and every |v|
template <int N>
__device__ __forceinline__ void take_magnitudes(uint32_t& most, const float* v) {
  float m = __uint_as_float(most);
#pragma unroll
  for (int j = 0; j < N; j += 2)
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[j]), "f"(v[N == 1 ? j : j + 1]));
  most = __float_as_uint(m);
}

// two values as whole numbers, in the low bytes of the words
__device__ __forceinline__ void quantize_pair(const RowScale& s, float v0, float v1, uint32_t& b0, uint32_t& b1) {
  if (s.prescale != 1.f) v0 = mul_exact(v0, s.prescale), v1 = mul_exact(v1, s.prescale);
  const uint64_t x = pack2(v0, v1), r0 = mul2(x, pack2(s.inv, s.inv));
  const uint64_t rest = fma2(r0, pack2(-s.amax, -s.amax), mul2(x, pack2(127.f, 127.f)));
  float m0, m1;
  unpack2(add2(fma2(rest, pack2(s.back, s.back), r0), pack2(12582912.f, 12582912.f)), m0, m1);
  b0 = s.flat ? 0u : __float_as_uint(m0), b1 = s.flat ? 0u : __float_as_uint(m1);
}
__device__ __forceinline__ uint2 quantize_unit(const RowScale& s, const float* v) {
  uint32_t b[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) quantize_pair(s, v[j], v[j + 1], b[j], b[j + 1]);
  auto word = [&](int j) { return __byte_perm(__byte_perm(b[j], b[j + 1], 0x0040), __byte_perm(b[j + 2], b[j + 3], 0x0040), 0x5410); };
  return make_uint2(word(0), word(4));
}
__device__ __forceinline__ int8_t quantize_value(const RowScale& s, float v) {
  uint32_t b, unused;
  quantize_pair(s, v, 0.f, b, unused);
  return static_cast<int8_t>(b);
}

// ------------------------------------------------------------------------------------------------ host
// How a row of n elements is laid over threads: `cnt` units each; 0: the row is too long and is walked. Many rows are a matter of bytes in
// flight and of lanes without a unit: up to four units a thread, five where that halves the threads, and six up to 128 of them. us, four at most and
// so: residual_norm of 16384 x 1280 with both norms 37.6, 33.2, plain 34.4, 28.8, of 4096 x 5120 42.3, 37.1 and 38.4, 29.6, of 13648 x 1536
// (six) 34.5, 32.7 and 31.7, 28.4; quantize_rows of 16384 x 1280 18.4, 11.3, gated 20.4, 17.0, of 1024 x 20480 21.5, 15.6; but six of 256 threads,
// 1704 x 12288 to 8 bits 31.4, 32.8. Skewed rows take registers: up to three. Up to `few_rows` rows are a matter of latency, and a thread
// takes no more than `few` units.
struct TeamShape {
  int cnt, threads;
  bool aligned;
};
constexpr TeamShape team_shape_of(long long units, bool aligned, bool few_rows, int few) {
  if (units > (aligned ? 4 : 3) * kTeamMaxThreads) return TeamShape{0, kTeamMaxThreads, aligned};
  const bool spread = few_rows && units <= few * kTeamMaxThreads;
  int threads = 32;
  while (threads * (spread ? few : !aligned || threads > 512 ? 4 : threads > 128 ? 5 : 6) < units) threads *= 2;
  if (!aligned && threads * 3 < units) threads *= 2;
  return TeamShape{static_cast<int>((units + threads - 1) / threads), threads, aligned};
}
inline TeamShape team_shape(long long rows, long long n, bool aligned, long long few_rows, int few) {
  return team_shape_of(aligned ? n / 8 : (n + 14) / 8, aligned, rows <= few_rows, few);
}
// Does a row of any length come to this shape? (The steps between shapes lie at whole 32 units.)
constexpr bool team_shape_is_taken(int cnt, int threads, bool aligned, int few) {
  for (int units = 32; units <= 4 * kTeamMaxThreads; units += 32)
    for (int i = 0; i < 2; ++i) {
      const TeamShape t = team_shape_of(units, aligned, i != 0, few);
      if (t.cnt == cnt && t.threads == threads) return true;
    }
  return false;
}
// Do these operands of rows at a pitch of whole elements lie alike: at the same place of 16 bytes in every row?
inline bool lie_alike(std::initializer_list<const void*> operands) {
  const void* one = nullptr;
  for (const void* p : operands) {
    if (p == nullptr) continue;
    if (one != nullptr && ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(one)) & 15u) != 0) return false;
    one = p;
  }
  return true;
}
inline bool multiple_of(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Calls `launch` with (CNT, THREADS, ALIGNED) as compile-time numbers.
template <int FEW, class F>
inline void for_team_shape(const TeamShape& t, F&& launch) {
  switch (t.cnt * 10000 + t.threads + (t.aligned ? 0 : 1)) {
#define B200AIT_TEAM(CNT, THREADS, ALIGNED)                                                                                                    \
  case (CNT) * 10000 + (THREADS) + ((ALIGNED) ? 0 : 1):                                                                                        \
    if constexpr (team_shape_is_taken(CNT, THREADS, ALIGNED, FEW))                                                                             \
      return launch(std::integral_constant<int, CNT>{}, std::integral_constant<int, THREADS>{}, std::integral_constant<bool, ALIGNED>{});      \
    break;
#define B200AIT_TEAMS(THREADS)                                                                                                                 \
  B200AIT_TEAM(1, THREADS, true) B200AIT_TEAM(2, THREADS, true) B200AIT_TEAM(3, THREADS, true) B200AIT_TEAM(4, THREADS, true)                  \
  B200AIT_TEAM(5, THREADS, true) B200AIT_TEAM(6, THREADS, true)                                                                                \
  B200AIT_TEAM(1, THREADS, false) B200AIT_TEAM(2, THREADS, false) B200AIT_TEAM(3, THREADS, false)
    B200AIT_TEAMS(32) B200AIT_TEAMS(64) B200AIT_TEAMS(128) B200AIT_TEAMS(256) B200AIT_TEAMS(512) B200AIT_TEAMS(1024)
#undef B200AIT_TEAMS
#undef B200AIT_TEAM
  }
  throw Error("no kernel for rows of this length");
}

}  // namespace b200ait
