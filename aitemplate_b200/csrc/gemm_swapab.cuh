// Device code and launch of the weight-streaming tensor-core GEMM (see gemm.cu for its planner and gemm_kernel.cuh for what it
// shares with the tile kernels). Included by gemm.cu and by gemm_swapab_i8.cu, which instantiate it.
#pragma once
#include "gemm_kernel.cuh"

namespace b200ait {

// ------------------------------------------------------------------------------------------------
// Weight-streaming tensor-core kernel with the operands swapped: Y^T = W X^T.
// The run time of a GEMM with few rows of X is the time to read W once. Here the rows of W sit on the 128 MMA rows
// and the rows of X are the MMA's N (MX = 16 .. 256), so a CTA consumes 16 KB of weights per four MMAs, and W is
// partitioned so that every byte is read by exactly one CTA per group of MX rows of X: a cluster of R = 2, 4 or 8 CTAs
// owns a slab of 128 weight rows, rank r streams share r of K through a TMA ring, and the ranks hand each other
// their 128 x MX fp32 partial sums through the cluster's shared-memory window (a reduce-scatter: every rank finishes
// MX / R rows of X). No global workspace, no second pass (the 128 x 256 tiles + split-K + reduce kernel this
// replaces ran at 0.54 of the copy rate for M <= 32). More than 256 rows of X are taken in groups of 256.
//   warp 0: TMA producer   warp 1: MMA issuer   warps 2-5: epilogue (TMEM lane = weight row = output column)
constexpr int kSwapThreads = 192;
constexpr int kSwapMaxM = 256;
template <int MX, int R, int H>
struct SwapCfg {
  static_assert(R == 1 || R == 2 || R == 4 || R == 8, "cluster size");
  static constexpr int kPart = MX / R;              // rows of X each rank finishes ...
  static constexpr int kSub = kPart / H;            // ... in H passes of kSub rows (what bounds the exchange buffers)
  static_assert(H >= 1 && kSub * H == kPart && kSub >= 8, "a rank finishes at least 8 rows per pass");
  static constexpr int kWBytes = 128 * kBK * 2;     // 16 KB: 128 weight rows x 64 k
  static constexpr int kXBytes = MX * kBK * 2;      // MX rows of X x 64 k
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kSlotBytes = 128 * kSub * 4;                // [kSub rows of X][128 weight rows] fp32
  static constexpr int kPartialBytes = (R - 1) * kSlotBytes;       // one slot per peer: its sums for this rank's rows
  static constexpr int kTileBytes = kSlotBytes;                    // the finished tile, [kSub][128]
  static constexpr int kFit = (227 * 1024 - 256 - kPartialBytes - kTileBytes) / kStageBytes;
  static constexpr int kStages = kFit < 8 ? kFit : 8;  // 144 to 192 KB in flight
  static constexpr int kAccCols = MX < 32 ? 32 : MX;  // TMEM columns of one accumulator
  static constexpr int kTmemCols = 2 * kAccCols;
  static constexpr int kSmemBytes = kStages * kStageBytes + kPartialBytes + kTileBytes + 256;
  static_assert(kStages >= 3 && kSmemBytes <= 227 * 1024, "swapped-operand kernel: shared memory");
};

template <int N>
__device__ __forceinline__ void tmem_ld_chunk(uint32_t taddr, uint32_t (&r)[N]) {
  static_assert(N == 8 || N == 16 || N == 32, "TMEM load width");
  if constexpr (N == 8) {
    tmem_ld_32x32b_x8(taddr, r);
  } else if constexpr (N == 16) {
    tmem_ld_32x32b_x16(taddr, r);
  } else {
    tmem_ld_32x32b_x32(taddr, r);
  }
}

// I8: operands of signed 8-bit integers (gemm_kernel.cuh). The ranks exchange 32-bit integer sums; the columns' scales are
// applied where a rank adds them up (a thread then holds one column), the rows' where the tile goes out.
template <bool BF16, int MX, int R, int H, bool I8 = false>
__global__ void __launch_bounds__(kSwapThreads, 1)
gemm_swapab_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x,
                   const GemmParams p, const int num_slabs, const int num_groups) {
  using Cfg = SwapCfg<MX, R, H>;
  constexpr int kBKE = kBKOf<I8>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const bool misaligned = (smem_u32(smem) & 1023u) != 0u;
  if (misaligned && threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, kDevBadSmemAlignment);
  float* partial = reinterpret_cast<float*>(smem + Cfg::kStages * Cfg::kStageBytes);  // [R - 1][kSub / 4][128][4], a slot per peer
  float* tile = reinterpret_cast<float*>(smem + Cfg::kStages * Cfg::kStageBytes + Cfg::kPartialBytes);  // [kSub][128]
  uint64_t* full_bar =
      reinterpret_cast<uint64_t*>(smem + Cfg::kStages * Cfg::kStageBytes + Cfg::kPartialBytes + Cfg::kTileBytes);
  uint64_t* empty_bar = full_bar + Cfg::kStages;
  uint64_t* acc_full = empty_bar + Cfg::kStages;   // [2]
  uint64_t* acc_empty = acc_full + 2;             // [2]
  uint64_t* partial_ready = acc_empty + 2;        // every peer's partial sums are in `partial` (counts their bytes)
  uint64_t* partial_taken = partial_ready + 1;    // [2] every peer has read the sums it was sent (even / odd passes)
  uint64_t* drain_bar = partial_taken + 2;
  uint64_t* tile_summed = drain_bar + 1;          // every thread has put its sums into `tile`
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tile_summed + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * Cfg::kStages + 9) * 8 + 8 <= 256, "barrier area too small");

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int walker = blockIdx.x / R, num_walkers = gridDim.x / R;
  // a unit of work: one slab of 128 weight rows against one group of MX rows of X (consecutive units share the slab,
  // so the clusters that run them side by side fetch its weights from HBM once)
  const int my_units = misaligned ? 0 : num_slabs * num_groups;
  // this rank's share of the k-blocks (the host sends no problem with fewer k-blocks than ranks)
  const int kb_total = (p.K + kBKE - 1) / kBKE;
  // split evenly, so that no rank is left without a k-block (its accumulator would never be written)
  const int kb0 = rank * kb_total / R, kb1 = (rank + 1) * kb_total / R;

  // Set-up, kept short because a small problem's whole run is a few microseconds: the lanes of warp 0 initialise one
  // barrier each while warp 1 allocates tensor memory, and the opening cluster barrier is arrived at without a release
  // (the initialisations are published by fence.mbarrier_init; a releasing arrive alone was measured at 0.5 us). Only the
  // epilogue warps touch the peers, so only they wait for the cluster here: the producer goes on to its loads as soon as its
  // barriers stand, the MMA issuer once tensor memory is there too, and both wait for the cluster after their work.
  constexpr int kSetupBar = 1;
  if (warp == 0) {
    // barriers in the order they lie in shared memory: full[kStages], empty[kStages], acc_full[2], acc_empty[2],
    // partial_ready, partial_taken[2], drain_bar, tile_summed
    constexpr int kBars = 2 * Cfg::kStages + 9;
    for (int i = lane; i < kBars; i += 32) {
      const int j = i - 2 * Cfg::kStages;  // index among the barriers after the ring's
      // every epilogue thread arrives at acc_empty and tile_summed, every peer's at partial_taken, one thread elsewhere
      const uint32_t count = (j == 2 || j == 3 || j == 8) ? 128u : (j == 5 || j == 6) ? 128u * (R > 1 ? R - 1 : 1) : 1u;
      mbar_init(&full_bar[i], count);
    }
    if (lane == 0) *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();  // the loads below credit barriers that other lanes have initialised
    __syncwarp();
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);  // two accumulators
    grid_release();
    tmem_relinquish();
  }
  tc_fence_before();
  cluster_arrive_relaxed();
  if (warp == 0) {
    named_bar_arrive(kSetupBar, kSwapThreads);
  } else {
    named_bar_sync(kSetupBar, kSwapThreads);
    if (warp != 1) cluster_wait();  // the peers' barriers are initialised before anything signals them
  }
  tc_fence_after();
  grid_wait();
  bool epi_arrived = false;  // this thread has arrived at the closing cluster barrier

  if (warp == 0) {
    // TMA producer. Every CTA reads the same rows of X: walking the k-blocks from a different starting point in every
    // cluster keeps the CTAs from asking L2 for the same lines of X at the same moment.
    const uint32_t lead = elect_one();
    const uint32_t smem0 = smem_u32(smem), full0 = smem_u32(full_bar);
    const int nkb = kb1 - kb0;
    int stage = 0;
    uint32_t phase = 0;
    bool first = true;  // the first pass over the ring: every stage is free
    bool ok = true;
    for (int unit = walker; ok && unit < my_units; unit += num_walkers) {
      const int slab = unit / num_groups, grp = unit - slab * num_groups;
      // (by slab, not by unit: every group of X rows adds its k-blocks up in the same order, so a row's result does not
      // depend on the group it falls into)
      const int rot = nkb > 0 ? static_cast<int>((static_cast<unsigned>(slab) * 11u) % static_cast<unsigned>(nkb)) : 0;
      for (int i = 0; i < nkb; ++i) {
        const int kb = kb0 + (i + rot >= nkb ? i + rot - nkb : i + rot);
        if (!first) ok = mbar_wait_warp(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, kDevWaitEmptyTimeout);
        if (!ok) break;
        const uint32_t sw = smem0 + static_cast<uint32_t>(stage) * Cfg::kStageBytes, bar = full0 + static_cast<uint32_t>(stage) * 8u;
        mbar_arrive_expect_tx_warp(&full_bar[stage], Cfg::kStageBytes, lead);
        tma_load_3d_warp(sw, &tma_w, bar, kb * kBKE, slab * 128, 0, lead);
        tma_load_3d_warp(sw + Cfg::kWBytes, &tma_x, bar, kb * kBKE, grp * MX, 0, lead);
        if (++stage == Cfg::kStages) {
          stage = 0;
          phase ^= 1u;
          first = false;
        }
      }
    }
    if (!ok) {
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) {
      }
    }
    __syncwarp();
    cluster_wait();
  } else if (warp == 1) {
    constexpr uint32_t idesc = I8 ? umma_idesc_i8(128, MX) : umma_idesc_f16(128, MX, BF16, false, false);
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t lead = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int unit = walker; ok && unit < my_units; unit += num_walkers) {
      ok = mbar_wait_warp(&acc_empty[acc], acc_phase ^ 1u, abort_flag, p.status, kDevWaitAccEmptyTimeout);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * Cfg::kAccCols);
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait_warp(&full_bar[stage], phase, abort_flag, p.status, kDevWaitFullTimeout);
        if (!ok) break;
        tc_fence_after();
        const uint32_t w_addr = smem_u32(smem + stage * Cfg::kStageBytes);
        const uint32_t w_lo = umma_smem_desc_sw128_lo(w_addr, 16), x_lo = umma_smem_desc_sw128_lo(w_addr + Cfg::kWBytes, 16);
#pragma unroll
        for (int k = 0; k < kBK / 16; ++k) {
          if constexpr (I8) {
            umma_i8_ss_warp(d_tmem, w_lo + k * (32 >> 4), x_lo + k * (32 >> 4), idesc, (kb > kb0 || k != 0) ? 1u : 0u, lead);
          } else {
            umma_f16_ss_warp(d_tmem, w_lo + k * (32 >> 4), x_lo + k * (32 >> 4), idesc, (kb > kb0 || k != 0) ? 1u : 0u, lead);
          }
        }
        umma_commit_warp(&empty_bar[stage], lead);
        if (++stage == Cfg::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      umma_commit_warp(&acc_full[acc], lead);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    if (!ok) {
      umma_commit_warp(drain_bar, lead);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(drain_bar, 0) && globaltimer_ns() - t0 < 1000000ull) {
      }
    }
    __syncwarp();
    cluster_wait();
  } else {
    const uint32_t tmem_base = *tmem_slot;
    // The MX rows of X are cut into H x R blocks of kSub rows; in pass h rank r finishes block h * R + r: it keeps
    // that block of its own sums and sends each peer q the block h * R + q (slot "sender" of q's `partial`, four rows
    // of X per 16-byte store: a warp's store covers 512 consecutive bytes). The stores are asynchronous and credit their bytes to the receiver's
    // `partial_ready`: nobody waits for a store to land except the thread that needs the data. Then the rank adds
    // what its peers sent into `tile` and writes its rows out. (H > 1 only bounds the buffers: 256 rows of X would
    // otherwise need 128 KB of them.)
    constexpr int kSub = Cfg::kSub;
    constexpr int kChunk = kSub < 32 ? kSub : 32;  // TMEM columns per load
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // weight row inside the slab == TMEM lane
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int et = static_cast<int>(threadIdx.x) - 64;  // 0..127 over the four epilogue warps
    int acc = 0;
    uint32_t acc_phase = 0;
    // Passes done so far: `tile_summed` changes phase once per pass. The peers' "taken" signals of pass s go to
    // partial_taken[s & 1]: a rank that has no rows in a pass runs through it without waiting for anybody's sums, so
    // its signals of pass s + 1 can be complete before a slow thread here has looked at those of pass s. With one
    // barrier that thread would then wait on a parity that has come round again; with two, a barrier is reused only
    // for pass s + 2, which no peer can finish before every thread here has signalled pass s + 1.
    int seq = 0;
    uint32_t ready_phase = 0;  // `partial_ready` only changes phase in the passes in which this rank has rows
    bool ok = true;
    for (int unit = walker; ok && unit < my_units; unit += num_walkers) {
      const bool last_slab = unit + num_walkers >= my_units;
      const int slab = unit / num_groups;
      const int row_base = (unit - slab * num_groups) * MX;  // first row of X of this unit's group
      const int m_here = p.M - row_base < MX ? p.M - row_base : MX;
      // The tile goes out row by row: a thread takes 8 consecutive columns (one 16-byte store), 16 threads one
      // row of the slab. A thread keeps the same columns for every row, so it fetches their bias once, early.
      const int col0 = slab * 128 + (et & 15) * 8;
      const bool vec = p.vec_ok && col0 + 8 <= p.N;
      float bias_v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (vec && p.bias != nullptr)
        unpack8<BF16>(*reinterpret_cast<const uint4*>(static_cast<const typename Elem16<BF16>::T*>(p.bias) + col0), bias_v);
      // this thread's column of the slab while it adds up sums, and the factor of a row while the tile goes out
      const float col_scale = I8 && slab * 128 + row < p.N ? p.col_scale[slab * 128 + row] : 0.f;
      auto row_factor = [&](int r) { return I8 ? p.row_scale[r] : p.alpha; };
      auto scaled = [](float v, float factor, float bias) { return I8 ? scale_row_i8(v, factor, bias) : v * factor + bias; };
      ok = mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.status, kDevWaitAccFullTimeout);
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_addr = tmem_base + lane_addr + static_cast<uint32_t>(acc * Cfg::kAccCols);
#pragma unroll 1
      for (int pass = 0; ok && pass < H; ++pass, ++seq) {
      const bool last = last_slab && pass == H - 1;
      const int my_row0 = (pass * R + rank) * kSub;
      const int my_rows = m_here - my_row0 < 0 ? 0 : (m_here - my_row0 < kSub ? m_here - my_row0 : kSub);
      const int out_row0 = row_base + my_row0;  // where this rank's block starts in the output
      // what the peers will send for this pass (a rank with no valid row of X is sent nothing and waits for nothing)
      if (R > 1 && et == 0 && my_rows > 0) mbar_arrive_expect_tx(partial_ready, (R - 1) * Cfg::kSlotBytes);
      // the peers must have read what this CTA sent for the previous pass before it is overwritten
      if (R > 1 && seq > 0)
        ok = mbar_wait_cluster(&partial_taken[(seq - 1) & 1], ((seq - 1) >> 1) & 1, abort_flag, p.status,
                               kDevWaitOtherTimeout);
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const int q_row0 = (pass * R + q) * kSub;
        if (q == rank || m_here <= q_row0) continue;
        const int slot = rank < q ? rank : rank - 1;  // where this rank's sums go in rank q's buffer
        const uint32_t dst = mapa_shared(smem_u32(partial), static_cast<uint32_t>(q)) +
                             static_cast<uint32_t>((slot * kSub * 128 + row * 4) * 4);
        const uint32_t dst_bar = mapa_shared(smem_u32(partial_ready), static_cast<uint32_t>(q));
#pragma unroll
        for (int c = 0; c < kSub / kChunk; ++c) {
          uint32_t v[kChunk];
          tmem_ld_chunk<kChunk>(t_addr + static_cast<uint32_t>(q_row0 + c * kChunk), v);
          tmem_ld_wait();
          if (ok) {
#pragma unroll
            for (int j = 0; j < kChunk; j += 4)
              st_async_cluster_v4(dst + static_cast<uint32_t>((c * kChunk + j) * 128 * 4), v[j], v[j + 1], v[j + 2], v[j + 3],
                                  dst_bar);
          }
        }
      }
      // After its last send a thread touches no peer again: the cluster-wide barrier that keeps every CTA alive
      // until then is arrived at here and waited for at the very end, when it has long completed.
      if (last) {
        cluster_arrive_relaxed();
        epi_arrived = true;
      }
      if (ok && my_rows > 0) {
        if constexpr (R > 1) {
          ok = mbar_wait_cluster(partial_ready, ready_phase, abort_flag, p.status, kDevWaitOtherTimeout);
          ready_phase ^= 1u;
        }
#pragma unroll
        for (int c = 0; c < kSub / kChunk; ++c) {
          uint32_t v[kChunk];
          tmem_ld_chunk<kChunk>(t_addr + static_cast<uint32_t>(my_row0 + c * kChunk), v);
          tmem_ld_wait();
          if (ok) {
            // The K shares are added in the order of their ranks whichever rank does the adding, so a row's result
            // does not depend on which rank finishes it (= on its position in X). All loads of the chunk come before
            // its first store: the compiler may not move a load of `partial` over a store to `tile` by itself.
            if constexpr (I8) {
              int sum[kChunk];
#pragma unroll
              for (int j = 0; j < kChunk; ++j) sum[j] = static_cast<int>(v[j]);
#pragma unroll
              for (int slot = 0; slot < R - 1; ++slot) {
#pragma unroll
                for (int j = 0; j < kChunk; j += 4) {
                  const int4 term = *reinterpret_cast<const int4*>(partial + ((slot * kSub + c * kChunk + j) * 128 + row * 4));
                  sum[j] += term.x, sum[j + 1] += term.y, sum[j + 2] += term.z, sum[j + 3] += term.w;
                }
              }
#pragma unroll
              for (int j = 0; j < kChunk; ++j) tile[(c * kChunk + j) * 128 + row] = scale_column_i8(sum[j], col_scale);
            } else {
              float sum[kChunk];
#pragma unroll
            for (int j = 0; j < kChunk; j += 4) {
#pragma unroll
              for (int q = 0; q < R; ++q) {
                const int slot = q < rank ? q : q - 1;  // where rank q's sums sit in this rank's buffer
                const float4 term =
                    q == rank ? make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), __uint_as_float(v[j + 2]),
                                            __uint_as_float(v[j + 3]))
                              : *reinterpret_cast<const float4*>(partial + ((slot * kSub + c * kChunk + j) * 128 + row * 4));
                sum[j] = q == 0 ? term.x : sum[j] + term.x;
                sum[j + 1] = q == 0 ? term.y : sum[j + 1] + term.y;
                sum[j + 2] = q == 0 ? term.z : sum[j + 2] + term.z;
                sum[j + 3] = q == 0 ? term.w : sum[j + 3] + term.w;
              }
            }
#pragma unroll
            for (int j = 0; j < kChunk; ++j) tile[(c * kChunk + j) * 128 + row] = sum[j];
            }
          }
        }
      }
      if (pass == H - 1) {  // the accumulator has been read for the last time
        tc_fence_before();
        mbar_arrive(&acc_empty[acc]);
      }
      if (ok) {
        mbar_arrive(tile_summed);
        ok = mbar_wait(tile_summed, seq & 1, abort_flag, p.status, kDevWaitOtherTimeout);
      }
      if (ok) {
        const int code = p.epilogue;
        // bias + one activation [+ one added residual [+ relu]] into a row-major output: the short store loop
        const bool add_d0 = epi_b1(code) == kBinaryAdd;
        const bool simple = vec && (epi_b1(code) == kBinaryNone || add_d0) && epi_b2(code) == kBinaryNone &&
                            (epi_u2(code) == kUnaryIdentity || (add_d0 && epi_u2(code) == kUnaryRelu)) &&
                            p.store_mode == 0;
        // An activation that is more than a max runs first, in place on this thread's own elements of the tile, a row
        // per trip of a rolled loop, so that the store loops below carry no activation code but relu. (This code runs
        // once or twice per launch, from a cold instruction cache: with the activations dispatched inside the 32-wide
        // store loop, 3072 x 768 at M = 128 with tanh took 4.7 us longer than with bias alone, 8192 x 8192 9.2 us.)
        const bool pre = vec && epi_u1(code) != kUnaryIdentity && epi_u1(code) != kUnaryRelu;
        if (pre) {
          const int u1 = epi_u1(code);
#pragma unroll 1
          for (int j = et >> 4; j < my_rows; j += 8) {
            float* src = tile + j * 128 + (et & 15) * 8;
            const float factor = row_factor(out_row0 + j);
            const float4 a0 = *reinterpret_cast<const float4*>(src), a1 = *reinterpret_cast<const float4*>(src + 4);
            float w[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = scaled(w[e], factor, bias_v[e]);
            apply_unary_vec_of<I8>(u1, w);
            *reinterpret_cast<float4*>(src) = make_float4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<float4*>(src + 4) = make_float4(w[4], w[5], w[6], w[7]);
          }
        }
        if (simple) {
          // four rows (j, j + 8, j + 16, j + 24) per trip, all of a trip's shared-memory loads first; no per-row
          // dispatch on the epilogue code
          using T = typename Elem16<BF16>::T;
          const bool relu = epi_u1(code) == kUnaryRelu, relu_after = epi_u2(code) == kUnaryRelu;
          T* out0 = static_cast<T*>(p.out) + col0;
          const T* res0 = static_cast<const T*>(p.d0) + col0;
          for (int j = et >> 4; j < my_rows; j += 32) {
            float o[4][8], factor[4];
            uint4 r0[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const int jj = j + 8 * t < my_rows ? j + 8 * t : j;
              factor[t] = row_factor(out_row0 + jj);
              if (add_d0) r0[t] = *reinterpret_cast<const uint4*>(res0 + static_cast<long long>(out_row0 + jj) * p.ldd);
              const float* src = tile + jj * 128 + (et & 15) * 8;
              const float4 a0 = *reinterpret_cast<const float4*>(src), a1 = *reinterpret_cast<const float4*>(src + 4);
              o[t][0] = a0.x, o[t][1] = a0.y, o[t][2] = a0.z, o[t][3] = a0.w;
              o[t][4] = a1.x, o[t][5] = a1.y, o[t][6] = a1.z, o[t][7] = a1.w;
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              if (j + 8 * t < my_rows) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const float y = pre ? o[t][e] : scaled(o[t][e], factor[t], bias_v[e]);
                  o[t][e] = relu ? fmaxf(y, 0.f) : y;  // identity keeps a NaN a NaN
                }
                if (add_d0) {
                  float f[8];
                  unpack8<BF16>(r0[t], f);
#pragma unroll
                  for (int e = 0; e < 8; ++e) o[t][e] = relu_after ? fmaxf(o[t][e] + f[e], 0.f) : o[t][e] + f[e];
                }
                *reinterpret_cast<uint4*>(out0 + static_cast<long long>(out_row0 + j + 8 * t) * p.ldc) = pack8<BF16>(o[t]);
              }
            }
          }
        }
        if (!simple && vec) {
          // Any epilogue: four rows per trip again. A trip's shared-memory loads and residual loads all go out
          // before the first is used, and each activation is dispatched once per trip, over the 32 values.
          using T = typename Elem16<BF16>::T;
          const int u1 = epi_u1(code), b1 = epi_b1(code), b2 = epi_b2(code), u2 = epi_u2(code);
          T* out0 = static_cast<T*>(p.out) + col_offset(p, col0);
          for (int j = et >> 4; j < my_rows; j += 32) {
            float o[32], factor[4];
            uint4 r0[4], r1[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const int jj = j + 8 * t < my_rows ? j + 8 * t : j;
              factor[t] = row_factor(out_row0 + jj);
              const float* src = tile + jj * 128 + (et & 15) * 8;
              const float4 a0 = *reinterpret_cast<const float4*>(src), a1 = *reinterpret_cast<const float4*>(src + 4);
              o[t * 8 + 0] = a0.x, o[t * 8 + 1] = a0.y, o[t * 8 + 2] = a0.z, o[t * 8 + 3] = a0.w;
              o[t * 8 + 4] = a1.x, o[t * 8 + 5] = a1.y, o[t * 8 + 6] = a1.z, o[t * 8 + 7] = a1.w;
              const long long d_at = static_cast<long long>(out_row0 + jj) * p.ldd + col0;
              if (b1 != kBinaryNone) r0[t] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.d0) + d_at);
              if (b2 != kBinaryNone) r1[t] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.d1) + d_at);
            }
            if (!pre) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float y = scaled(o[i], factor[i >> 3], bias_v[i & 7]);
                o[i] = u1 == kUnaryRelu ? fmaxf(y, 0.f) : y;
              }
            }
            if (b1 != kBinaryNone) {
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                float f[8];
                unpack8<BF16>(r0[t], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[t * 8 + e] = (b1 == kBinaryAdd) ? o[t * 8 + e] + f[e] : o[t * 8 + e] * f[e];
              }
            }
            if (b2 != kBinaryNone) {
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                float f[8];
                unpack8<BF16>(r1[t], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[t * 8 + e] = (b2 == kBinaryAdd) ? o[t * 8 + e] + f[e] : o[t * 8 + e] * f[e];
              }
            }
            apply_unary_vec_of<I8>(u2, o);
#pragma unroll
            for (int t = 0; t < 4; ++t)
              if (j + 8 * t < my_rows)
                *reinterpret_cast<uint4*>(out0 + row_offset(p, out_row0 + j + 8 * t)) = pack8<BF16>(&o[t * 8]);
          }
        }
        if (!vec) {
          // columns whose 16-byte accesses are not legal (a ragged last slab, an odd row pitch): element by element
          for (int j = et >> 4; j < my_rows; j += 8) {
            const float* src = tile + j * 128 + (et & 15) * 8;
#pragma unroll 1
            for (int e = 0; e < 8; ++e)
              if (col0 + e < p.N) {
                if constexpr (I8) {
                  epilogue_scalar_store_i8<BF16>(p, src[e], row_factor(out_row0 + j), out_row0 + j, col0 + e);
                } else {
                  epilogue_scalar_store<BF16>(p, src[e], 0, out_row0 + j, col0 + e);
                }
              }
          }
        }
        // This thread is done reading `partial`: the peers may send the next pass's sums. (Its reads have returned -
        // their values went into `tile` - so the signal needs no release. A rank without rows signals all the same:
        // the senders count every peer.)
        if (R > 1 && !last) {
#pragma unroll
          for (int q = 0; q < R; ++q)
            if (q != rank)
              mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&partial_taken[seq & 1]), static_cast<uint32_t>(q)));
        }
      }
      }  // passes
      if (last_slab) break;
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }

  // Every thread arrives at the cluster-wide barrier exactly once: the epilogue threads did after their last send
  // (unless a wait ran out first), everybody else does here.
  if (!epi_arrived) cluster_arrive_relaxed();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, Cfg::kTmemCols);
  }
  cluster_wait();  // no CTA leaves while a peer can still write to it or signal it
}

// One walker per cluster the GPU can hold at once (clusters do not straddle GPCs, so this can be fewer than SMs / R):
// a cluster left for a second wave would start when the first is already done streaming.
template <bool BF16, int MX, int R, int H, bool I8 = false>
static int swapab_resident_clusters() {
  using Cfg = SwapCfg<MX, R, H>;
  static std::atomic<uint64_t> configured{0};
  static std::atomic<int> resident{0};
  int clusters = resident.load(std::memory_order_relaxed);
  if (clusters == 0) {
    auto* kernel = &gemm_swapab_kernel<BF16, MX, R, H, I8>;
    opt_in_smem_once(configured, reinterpret_cast<const void*>(kernel), Cfg::kSmemBytes);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(R * (sm_count() / R)));
    cfg.blockDim = dim3(kSwapThreads);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = R;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    B200AIT_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
    B200AIT_REQUIRE(clusters > 0, "gemm: the weight-streaming kernel's cluster does not fit this GPU");
    resident.store(clusters, std::memory_order_relaxed);
  }
  return clusters;
}

template <bool BF16, int MX, int R, int H, bool I8 = false>
static void launch_swapab(const CUtensorMap& tw, const CUtensorMap& tx, const GemmParams& p, int num_slabs,
                          int num_groups, cudaStream_t stream) {
  using Cfg = SwapCfg<MX, R, H>;
  const int walkers = swapab_resident_clusters<BF16, MX, R, H, I8>();  // also opts the kernel in to its shared memory
  launch_early(&gemm_swapab_kernel<BF16, MX, R, H, I8>, dim3(static_cast<unsigned>(R * std::min(num_slabs * num_groups, walkers))),
               kSwapThreads, Cfg::kSmemBytes, stream, true, R, tw, tx, p, num_slabs, num_groups);
}

// The instantiations: MX rows of X per group, K split R ways, exchange in H passes.
#define B200AIT_FOR_EACH_SWAP_KERNEL(X)                                                                  \
  X(16, 2, 1) X(32, 2, 1) X(64, 2, 1) X(128, 2, 1) X(256, 2, 2) X(32, 4, 1) X(64, 4, 1) X(128, 4, 1)     \
  X(256, 4, 2) X(64, 8, 1) X(128, 8, 1) X(256, 8, 2)

// 8-bit operands; defined in gemm_swapab_i8.cu.
template <int MX, int R, int H>
void launch_swapab_i8(bool bf16, const CUtensorMap& tw, const CUtensorMap& tx, const GemmParams& p, int num_slabs,
                      int num_groups, cudaStream_t stream);

}  // namespace b200ait
