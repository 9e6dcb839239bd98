// The FP8 product for many rows where the scales are 8-bit exponents: the tensor core multiplies them in (tcgen05.mma kind::mxf8f6f4
// with block scales), so a tile's whole K range is summed in one accumulator and nothing is handed over per K block.
//
// The instruction takes one exponent per row of A and of B and 32 elements of K.  Here a scale covers 128 (and, for weights, 128
// rows), so the four MMAs of a K block use the same one: an operand's scales of four K blocks are the four bytes of one 32-bit
// column of tensor memory, and the instruction descriptor says which byte counts.  The scales of 128 rows are 4 columns (row r in
// lane r % 32 of column r / 32, the same in each of the four quarters of the lanes), those of the tile's 256 features 8.
//
// CTAS = 2: a pair of CTAs shares a tile of 256 rows and 256 features.  Each loads its 128 rows of X and 128 of the 256 weight
// rows; the MMA (cta_group::2, issued by the first CTA) reads both halves of the weights and leaves each CTA's 128 rows of sums in
// its own tensor memory.  Per K block a CTA so moves 32 KiB into shared memory and 32 KiB out of it in 512 cycles of MMAs; a lone CTA
// with 128 x 256 moves 48 + 48, and the 128 bytes a cycle that shared memory gives then bound it at 768 cycles (measured 789).
//
//   producer   one thread per CTA: TMA of the CTA's operands, counted on the first CTA's barrier
//   scales     four warps per CTA (a quarter of the lanes each): 12 words per lane and four K blocks, tcgen05.st
//   issuer     one thread of the first CTA
//   epilogue   eight warps per CTA: a row and 128 columns per thread; they empty the accumulator into registers, hand it back (the
//              next tile's MMAs wait for that alone), then round and store
#pragma once
#include "fp8_common.cuh"

namespace sk {

// ---------------------------------------------------------------- instructions
// D[tmem] (+)= (A * 2^sa)[smem] * (B * 2^sb)[smem]^T, e4m3 operands, scales in tensor memory, K = 32 per instruction.
template <int CTAS>
__device__ __forceinline__ void umma_f8_scaled(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa_tmem,
                                               uint32_t sb_tmem, uint32_t accumulate) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa_tmem), "r"(sb_tmem), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa_tmem), "r"(sb_tmem), "r"(accumulate)
        : "memory");
}
// Instruction descriptor, kind::mxf8f6f4: [4,6) byte of B's scale, [7,10) / [10,13) A / B format (0 = e4m3), [17,23) N >> 3,
// 23 scale format (1 = e8m0), [27,29) M >> 7, [29,31) byte of A's scale.
__host__ __device__ constexpr uint32_t make_idesc_scaled(int mma_m, int mma_n) {
  return (static_cast<uint32_t>(mma_n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(mma_m >> 7) << 27);
}
__device__ __forceinline__ uint32_t scale_bytes_in_idesc(uint32_t byte) { return (byte << 4) | (byte << 29); }

template <int CTAS>
__device__ __forceinline__ void commit_to(uint32_t bar) {        // arrives on the barrier (of both CTAs of a pair) once the MMAs so far are complete
  if constexpr (CTAS == 1)
    umma_commit(bar);
  else
    asm volatile(
        "{\n\t.reg .b16 m;\n\t"
        "mov.b16 m, 3;\n\t"
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(bar)
        : "memory");
}
// One arrival on a barrier of the pair's first CTA.
template <int CTAS>
__device__ __forceinline__ void arrive_first(uint32_t bar) {
  if constexpr (CTAS == 1)
    mbar_arrive(bar);
  else
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(map_to_cta(bar, 0)) : "memory");
}
// TMA load into this CTA's memory whose bytes are counted on the barrier `bar` (a shared::cluster address of either CTA of the pair).
template <int CTAS>
__device__ __forceinline__ void tma_load_counted(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CTAS == 1)
    tma_load_2d(dst, map, x, y, bar);
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x4(uint32_t taddr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}
__device__ __forceinline__ void tmem_st_32x8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <int CTAS, bool SILU>
struct Fp8ScaledTraits {
  static constexpr int kRows = 128 * CTAS;          // of the tile
  static constexpr int kStages = CTAS == 1 ? 4 : 6;
  static constexpr int kWBytes = CTAS == 1 ? 2 * kFp8TileBytes : kFp8TileBytes;
  static constexpr int kStageBytes = kFp8TileBytes + kWBytes;
  static constexpr int kSlots = 4;                  // groups of four K blocks whose scales are held
  static constexpr int kScaleCol0 = 256, kSlotCols = 16;   // tensor memory: 256 columns of sums, then the scales (4 of X, 8 of W, per slot)
  static constexpr int kOffBar = kStages * kStageBytes;
  static constexpr int kNumBars = 2 * kStages + 2 * kSlots + 3;
  static constexpr int kOffMisc = (kOffBar + kNumBars * 8 + 15) / 16 * 16;
  static constexpr int kOffAmax = kOffMisc + 16;    // SILU: [2 warpgroups][128 rows]
  static constexpr int kOffTable = kOffAmax + (SILU ? 2 * 128 * 4 : 8 * kTurnBytes);      // (else the warps' corners)
  static constexpr int kThreads = 512;
  // Registers: 128 a thread at launch; the epilogue holds 128 sums.
  static constexpr int kEpilogueRegs = 184, kOtherRegs = 72;
  static_assert(256 * kEpilogueRegs + 256 * kOtherRegs <= kThreads * 128, "a larger sum would wait forever");
  static constexpr int dynamic_bytes(int experts) { return kOffTable + group_table_bytes(experts) + 1024; }
};
static_assert(Fp8ScaledTraits<1, false>::dynamic_bytes(kFp8MaxExperts) <= 232448 && Fp8ScaledTraits<2, false>::dynamic_bytes(kFp8MaxExperts) <= 232448,
              "shared memory of a CTA");
static_assert(2 * 128 * 4 <= 8 * kTurnBytes, "(with the SiLU epilogue less)");

template <int CTAS, bool SILU>
__global__ void __launch_bounds__(512, 1)
fp8_scaled_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Fp8Params p) {
  using T = Fp8ScaledTraits<CTAS, SILU>;
  constexpr int S = T::kStages, kRows = T::kRows;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(smem);
  const uint32_t bar_full = base + T::kOffBar;      // [S] first CTA: the copies of a K block (of both CTAs) have landed
  const uint32_t bar_done = bar_full + 8 * S;       // [S] the MMAs that read a stage are complete (in both CTAs)
  const uint32_t bar_scales = bar_done + 8 * S;     // [kSlots] first CTA: the scales (of both CTAs) are in tensor memory
  const uint32_t bar_scales_free = bar_scales + 8 * T::kSlots;   // [kSlots] the MMAs that use them are complete (in both CTAs)
  const uint32_t bar_sum = bar_scales_free + 8 * T::kSlots;      // the tile's sums are complete (in both CTAs)
  const uint32_t bar_free = bar_sum + 8;            // first CTA: the sums have been read (by both CTAs)
  const uint32_t bar_drain = bar_free + 8;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + T::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + T::kOffMisc + 4);
  const WaitCtx ctx{abort_flag, p.status, p.wait_limit};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 1 ? 0 : static_cast<int>(cluster_ctarank());
  int* table = reinterpret_cast<int*>(smem + T::kOffTable);
  const GroupTable groups{table, table + p.experts + 1};

  grid_dep_launch_dependents();
  if (threadIdx.x == 384) {
    for (int i = 0; i < S; ++i) {
      mbar_init(bar_full + 8 * i, 1);
      mbar_init(bar_done + 8 * i, 1);
    }
    for (int i = 0; i < T::kSlots; ++i) {
      mbar_init(bar_scales + 8 * i, 4 * CTAS);
      mbar_init(bar_scales_free + 8 * i, 1);
    }
    mbar_init(bar_sum, 1);
    mbar_init(bar_free, 8 * CTAS);
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&tmap_w);
    prefetch_tensormap(&tmap_x);
  }
  if (warp == 13) {
    if constexpr (CTAS == 1) {
      tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
      tmem_relinquish();
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t*>(tmem_slot))), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  if (p.offsets != nullptr && warp == 0) {
    if (!p.early_weights) grid_dep_wait();
    build_group_table<kRows>(groups, p, lane);
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync_all();      // both CTAs' barriers exist before anything arrives on them
  tcgen05_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const int total = fp8_total_tiles<kRows>(groups, p);
  const int tile0 = static_cast<int>(blockIdx.x) / CTAS, step = static_cast<int>(gridDim.x) / CTAS;
  const int groups_of_four = (p.k_blocks + 3) >> 2;

  if (warp >= 8) {
    setmaxnreg_dec<T::kOtherRegs>();
    if (warp == 12) {
      // ------------------------------------------------------------ producer: one thread
      if (elect_one()) {
        int stage = 0;
        uint32_t phase = 1;                           // (the first round of stages is free)
        bool ok = true;
        const uint32_t counted = CTAS == 1 ? bar_full : map_to_cta(bar_full, 0);
        grid_dep_wait();
        for (int tile = tile0; tile < total && ok; tile += step) {
          const Fp8Tile t = fp8_tile_at<kRows>(tile, groups, p);
          // CTAS = 2: each CTA loads one of the tile's two boxes of weight rows
          const int w0 = t.expert * p.w_rows + t.n * (SILU ? 128 : 256), w1 = w0 + (SILU ? p.up_row0 : 128);
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            ok = wait_bounded_relaxed(bar_done + 8 * stage, phase, ctx, kStProducerEmpty, 40);
            if (!ok) break;
            if (kb != p.skip_block) {
              const uint32_t full = counted + 8 * stage, dst = base + stage * T::kStageBytes;
              if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * stage, T::kStageBytes * CTAS);
              tma_load_counted<CTAS>(dst, &tmap_x, kb * kFp8Block, t.row0 + rank * 128, full);
              tma_load_counted<CTAS>(dst + kFp8TileBytes, &tmap_w, kb * kFp8Block, rank == 0 ? w0 : w1, full);
              if constexpr (CTAS == 1) tma_load_counted<CTAS>(dst + 2 * kFp8TileBytes, &tmap_w, kb * kFp8Block, w1, full);
            }
            if (++stage == S) { stage = 0; phase ^= 1; }
          }
        }
        // A pair's second CTA leaves only when the first one's arrivals on its barriers have all landed: the sums' barrier, which the epilogue waits
        // for, says nothing of the others'.
        if constexpr (CTAS == 2)
          for (int i = 0; i < S && ok; ++i)
            ok = wait_bounded_relaxed(bar_done + 8 * ((stage + i) % S), stage + i < S ? phase : phase ^ 1, ctx, kStProducerEmpty, 40);
        if (!ok) {
          // Gave up: no copy may be in flight into this CTA's memory when it exits.  The first CTA watches the barriers that count
          // them, and the second, which cannot, waits far longer than a copy takes; it leaves after the first in any case.
          const long long t0 = clock64();
          if (rank == 0) {
            for (int i = 0; i < S; ++i)
              while (!mbar_try_wait(bar_full + 8 * ((stage + i) % S), stage + i < S ? phase : phase ^ 1))
                if (clock64() - t0 > ctx.limit) { atomicCAS(p.status, 0, kStDrain); break; }
          } else {
            while (clock64() - t0 < 1000000) {}
          }
        }
      }
      __syncwarp();
    } else if (warp == 13) {
      // ------------------------------------------------------------ MMA issuer: one thread of the first CTA
      if (rank == 0 && elect_one()) {
        constexpr uint32_t idesc = make_idesc_scaled(kRows, 256);
        const uint64_t desc0 = make_kmajor_sw128_desc(base);
        int stage = 0, slot = 0;
        uint32_t full_phase = 0, scales_phase = 0, free_phase = 1;      // (the accumulator is free at first)
        bool ok = true;
        grid_dep_wait();
        for (int tile = tile0; tile < total && ok; tile += step) {
          ok = wait_bounded(bar_free, free_phase, ctx, kStMmaAccEmpty);
          if (!ok) break;
          free_phase ^= 1;
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            const int q = kb & 3;
            if (q == 0) ok = wait_bounded(bar_scales + 8 * slot, scales_phase, ctx, kStEpilogueScales);
            ok = ok && wait_bounded(bar_full + 8 * stage, full_phase, ctx, kStMmaLdFull);
            if (!ok) break;
            tcgen05_fence_after_sync();
            const uint64_t a = desc0 + static_cast<uint64_t>((stage * T::kStageBytes) >> 4);
            const uint64_t b = a + static_cast<uint64_t>(kFp8TileBytes >> 4);
            const uint32_t sa = tmem + T::kScaleCol0 + slot * T::kSlotCols, sb = sa + 4;
            const uint32_t id = idesc | scale_bytes_in_idesc(q);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f8_scaled<CTAS>(tmem, a + static_cast<uint64_t>(2 * k), b + static_cast<uint64_t>(2 * k), id, sa, sb, kb > 0 || k > 0);
            commit_to<CTAS>(bar_done + 8 * stage);
            if (q == 3 || kb + 1 == p.k_blocks) {
              commit_to<CTAS>(bar_scales_free + 8 * slot);
              if (++slot == T::kSlots) { slot = 0; scales_phase ^= 1; }
            }
            if (++stage == S) { stage = 0; full_phase ^= 1; }
          }
          if (ok) commit_to<CTAS>(bar_sum);
        }
        if (!ok) {                                    // gave up: wait for the MMAs that still read shared memory
          commit_to<CTAS>(bar_drain);
          const long long t0 = clock64();
          while (!mbar_try_wait(bar_drain, 0))
            if (clock64() - t0 > ctx.limit) { atomicCAS(p.status, 0, kStDrain); break; }
        }
      }
      __syncwarp();
    } else if (warp < 12) {
      // ------------------------------------------------------------ scales: lane l holds those of rows l, l + 32, ... of X and W
      const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + T::kScaleCol0;
      int slot = 0;
      uint32_t phase = 1;
      bool ok = true;
      grid_dep_wait();
      for (int tile = tile0; tile < total && ok; tile += step) {
        const Fp8Tile t = fp8_tile_at<kRows>(tile, groups, p);
        // the two weight blocks of the 256 features (a second one past the end reads the first)
        const int n_block = SILU ? t.n : 2 * t.n;
        const int second = SILU ? p.up_block0 : (n_block + 1) * 128 < p.N ? 1 : 0;
        const long long ws0 = (t.expert * p.scale_rows + n_block) * p.k_blocks, ws1 = ws0 + second * static_cast<long long>(p.k_blocks);
        uint32_t x[4], w[2];
        auto fetch = [&](int kb) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = rank * 128 + lane + 32 * i;
            x[i] = load_exponents4(p.x_scale, static_cast<long long>(t.row0 + (row < t.rows ? row : 0)) * p.xs_row + kb * p.xs_blk, p.xs_blk, p.k_blocks - kb,
                      p.x_scale_groups);
          }
          w[0] = load_exponents4(p.w_scale, ws0 + kb, 1, p.k_blocks - kb, p.w_scale_groups);
          w[1] = load_exponents4(p.w_scale, ws1 + kb, 1, p.k_blocks - kb, p.w_scale_groups);
        };
        fetch(0);
        for (int g = 0; g < groups_of_four; ++g) {
          ok = wait_bounded_relaxed(bar_scales_free + 8 * slot, phase, ctx, kStProducerEmpty, 40);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tcgen05_fence_after_sync();
          const uint32_t sa[4] = {x[0], x[1], x[2], x[3]};
          const uint32_t sb[8] = {w[0], w[0], w[0], w[0], w[1], w[1], w[1], w[1]};
          tmem_st_32x4(t_lane + slot * T::kSlotCols, sa);
          tmem_st_32x8(t_lane + slot * T::kSlotCols + 4, sb);
          tmem_st_wait();
          tcgen05_fence_before_sync();
          __syncwarp();
          if (lane == 0) arrive_first<CTAS>(bar_scales + 8 * slot);
          if (g + 1 < groups_of_four) fetch(4 * g + 4);      // (scales read byte by byte are waited for: nobody else should)
          if (++slot == T::kSlots) { slot = 0; phase ^= 1; }
        }
      }
      if constexpr (CTAS == 2)                        // (see the producer)
        for (int i = 0; i < T::kSlots && ok; ++i) {
          ok = wait_bounded_relaxed(bar_scales_free + 8 * slot, phase, ctx, kStProducerEmpty, 40);
          ok = __all_sync(0xffffffffu, ok);
          if (++slot == T::kSlots) { slot = 0; phase ^= 1; }
        }
      __syncwarp();
    }
  } else {
    setmaxnreg_inc<T::kEpilogueRegs>();
    // ------------------------------------------------------------ epilogue: lane = row, columns = features
    const int wg = warp >> 2;
    const int row = (warp & 3) * 32 + lane;         // of this CTA's half of the tile
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    uint32_t phase = 0;
    bool ok = true;
    grid_dep_wait();
    for (int tile = tile0; tile < total && ok; tile += step) {
      const Fp8Tile t = fp8_tile_at<kRows>(tile, groups, p);
      const bool live = rank * 128 + row < t.rows;
      ok = wait_bounded_relaxed(bar_sum, phase, ctx, kStEpilogueAccFull, 100);
      ok = __all_sync(0xffffffffu, ok);
      phase ^= 1;
      uint32_t v[4][32];
      if (ok) {
        tcgen05_fence_after_sync();
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_lane + (SILU ? (c >> 1) * 128 + wg * 64 + (c & 1) * 32 : wg * 128 + c * 32), v[c]);
        tmem_ld_wait();
        tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_first<CTAS>(bar_free);
      }
      // (the warps of the SiLU epilogue meet below: none may be waited for that has given up)
      if constexpr (SILU) ok = named_barrier_all(1, 256, ok);
      if (!ok) break;
      const long long m = t.row0 + rank * 128 + row;
      if constexpr (SILU) {
        float* part = reinterpret_cast<float*>(smem + T::kOffAmax);
        const int n0 = t.n * 128 + wg * 64;
        float h[64];
        uint32_t a = 0;
#pragma unroll
        for (int j = 0; j < 64; ++j) {              // a feature past the end counts as zero in its block's maximum
          h[j] = n0 + j < p.N ? silu_times(__uint_as_float(v[j >> 5][j & 31]), __uint_as_float(v[2 + (j >> 5)][j & 31])) : 0.f;
          a = max(a, __float_as_uint(h[j]) & 0x7fffffffu);
        }
        part[wg * 128 + row] = __uint_as_float(a);
        named_barrier_sync(1, 256);
        a = max(a, __float_as_uint(part[(wg ^ 1) * 128 + row]));
        named_barrier_sync(1, 256);                 // (read before the next tile's are written)
        if (live) {
          const bool bad = not_finite_bits(a);
          const int e = bad ? 0 : fp8_block_exponent(a);
          const float inv = pow2f(-e);
          uint8_t* dst = static_cast<uint8_t*>(p.out) + m * p.ld_out + n0;
#pragma unroll
          for (int c = 0; c < 2; ++c) store_codes32(dst + 32 * c, p.N - n0 - 32 * c, inv, bad, [&](int j) { return h[32 * c + j]; });
          if (wg == 0) store_scale<true>(p.h_scale, m * p.hs_row + t.n * p.hs_blk, e, bad);
        }
      } else if (p.out_f32) {
        const int n0 = t.n * 256 + wg * 128;
        float* dst = static_cast<float*>(p.out) + m * p.ld_out + n0;
        if (live) {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            store_row16_f32(dst + 16 * c, p.N - n0 - 16 * c, [&](int j) { return __uint_as_float(v[c >> 1][16 * (c & 1) + j]); });
        }
      } else if (p.out_bytes == 2) {
        const int n0 = t.n * 256 + wg * 128, first = rank * 128 + (warp & 3) * 32;
        store_rows_turned(static_cast<uint16_t*>(p.out) + (t.row0 + first) * p.ld_out + n0, p.ld_out, min(32, t.rows - first), p.N - n0,
                          smem + T::kOffAmax + warp * kTurnBytes, lane, p.out_bf16, [&](int j) { return __uint_as_float(v[j >> 5][j & 31]); });
      } else if (live) {
        const int n0 = t.n * 256 + wg * 128;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + m * p.ld_out + n0;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          store_row16(dst + 16 * c, p.N - n0 - 16 * c, p.out_bytes, p.out_bf16,
                      [&](int j) { return __uint_as_float(v[c >> 1][16 * (c & 1) + j]); });
      }
    }
    __syncwarp();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync_all();      // (neither CTA leaves while the other may still arrive on its barriers)
  if (warp == 13) {
    tcgen05_fence_after_sync();
    if constexpr (CTAS == 1)
      tmem_dealloc(tmem, 512);
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace sk
