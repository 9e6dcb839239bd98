// The FP8 product for few rows where the scales are 8-bit exponents: weights' features on the tensor memory's lanes, TOK rows of X on
// its columns (16 or 32; with the SiLU epilogue 16), the scales multiplied in by the tensor core (fp8_scaled.cuh says how they lie).
//
// With few rows a product is a stream of weights out of HBM.  A K block is 16 KiB of weights and TOK x 128 B of activations, and all
// that happens to it is a copy, four MMAs and a commit: what the kernel for 32-bit scales does per K block in its epilogue -- 700
// cycles for one CTA, which held a projection of 4096 features and 16 rows to 44 GB/s per CTA -- is gone, and the stream is as fast as the ring
// is deep: 16 x 18944 x K, a tile per SM, takes 3.4 us and then 6.2 TB/s.  (One SM draws 80 GB/s at most.)  The ring takes what shared
// memory there is: where all CTAs (or all clusters of a split) run at once with an SM each, all of it for one CTA, else half.
//
// A tile's K range can be split over a cluster: every CTA pushes its sums into the CTA that owns the row (remote stores), one cluster
// barrier, then the owner adds them in rank order, so the result does not depend on timing.
//
// SILU: the tile holds 128 gate features and the 128 up features beside them (two accumulators); the epilogue forms SiLU(gate) * up in
// fp32 and quantises it: 128 features of a row are just one block of the next product, so its maximum is one reduction over the CTA's lanes.
#pragma once
#include "fp8_scaled.cuh"

namespace sk {

template <int TOK, bool SILU>
struct Fp8ScaledNarrowTraits {
  static constexpr int kW = SILU ? 2 : 1;
  static constexpr int kStageBytes = kW * kFp8TileBytes + TOK * kFp8Block;
  static constexpr int kMaxStages = 12;
  static constexpr int kSlots = 4;
  static constexpr int kSlotCols = kW * 4 + 4;      // 4 columns of scales per weight tile, and 4 for X (rows past 32 are not there)
  static constexpr int kSums = 2;                   // accumulator sets: the next tile's MMAs run while one is read
  static constexpr int kScaleCol0 = kSums * kW * TOK;
  static constexpr int kTmemCols = 128;
  static_assert(TOK <= 32 && kScaleCol0 + kSlots * kSlotCols <= kTmemCols, "tensor memory");
  // behind the ring (whose depth is the launch's): barriers, then the reduction buffer or the group table
  static constexpr int kNumBars = 2 * kMaxStages + 2 * kSlots + 2 * kSums + 1;
  static constexpr int kOffAmax = (kNumBars * 8 + 16 + 15) / 16 * 16;           // SILU: [4 warps][TOK]
  static constexpr int kOffTail = kOffAmax + (SILU ? 4 * TOK * 4 : 0);
  static constexpr int kRedBytes = TOK * 128 * 4;
  static constexpr int kThreads = 320;
  static constexpr int fixed_bytes(int split, int experts) {
    return 1024 + kOffTail + (split > 1 ? kRedBytes : 0) + group_table_bytes(experts);
  }
};

template <int TOK, bool SILU>
__global__ void __launch_bounds__(320, 2)
fp8_scaled_narrow_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Fp8Params p) {
  using T = Fp8ScaledNarrowTraits<TOK, SILU>;
  constexpr int kW = T::kW;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(smem);
  const int S = p.stages;
  uint8_t* behind = smem + S * T::kStageBytes;
  const uint32_t bar_full = smem_u32(behind);                    // [S] the copies of a K block have landed
  const uint32_t bar_done = bar_full + 8 * T::kMaxStages;        // [S] the MMAs that read a stage are complete
  const uint32_t bar_scales = bar_done + 8 * T::kMaxStages;      // [kSlots] the scales of four K blocks are in tensor memory
  const uint32_t bar_scales_free = bar_scales + 8 * T::kSlots;   // [kSlots] the MMAs that use them are complete
  const uint32_t bar_sum = bar_scales_free + 8 * T::kSlots;      // [kSums] a tile's sums are complete
  const uint32_t bar_free = bar_sum + 8 * T::kSums;              // [kSums] they have been read
  const uint32_t bar_drain = bar_free + 8 * T::kSums;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(behind + T::kNumBars * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(behind + T::kNumBars * 8 + 4);
  const WaitCtx ctx{abort_flag, p.status, p.wait_limit};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int rank = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  uint8_t* tail = behind + T::kOffTail;
  float* red = reinterpret_cast<float*>(tail);
  int* table = reinterpret_cast<int*>(tail + (split > 1 ? T::kRedBytes : 0));
  const GroupTable groups{table, table + p.experts + 1};

  grid_dep_launch_dependents();
  if (threadIdx.x == 256) {
    for (int i = 0; i < S; ++i) {
      mbar_init(bar_full + 8 * i, 1);
      mbar_init(bar_done + 8 * i, 1);
    }
    for (int i = 0; i < T::kSlots; ++i) {
      mbar_init(bar_scales + 8 * i, 4);
      mbar_init(bar_scales_free + 8 * i, 1);
    }
    for (int i = 0; i < T::kSums; ++i) {
      mbar_init(bar_sum + 8 * i, 1);
      mbar_init(bar_free + 8 * i, 4);
    }
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&tmap_w);
    prefetch_tensormap(&tmap_x);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), T::kTmemCols);
    tmem_relinquish();
  }
  if (p.offsets != nullptr && warp == 0) {
    if (!p.early_weights) grid_dep_wait();
    build_group_table<TOK>(groups, p, lane);
  }
  tcgen05_fence_before_sync();
  if (split > 1) cluster_sync_all(); else __syncthreads();       // (peers push into this CTA's memory only once it runs)
  tcgen05_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  const int total = fp8_total_tiles<TOK>(groups, p);
  const int tile0 = static_cast<int>(blockIdx.x) / split, step = static_cast<int>(gridDim.x) / split;
  // this CTA's share of the K blocks of a tile
  const int kb_begin = p.k_blocks * rank / split, kb_end = p.k_blocks * (rank + 1) / split;

  if (warp == 8) {
    // ------------------------------------------------------------ producer: one thread
    if (elect_one()) {
      int stage = 0, early = 0, issued = 0;          // (issued counts up to `early` only)
      uint32_t phase = 1;                           // (the first round of stages is free)
      bool ok = true;
      if (p.early_weights && tile0 < total) {       // (weights that no kernel still in flight writes)
        const Fp8Tile t = fp8_tile_at<TOK>(tile0, groups, p);
        early = min(S, kb_end - kb_begin);
        for (int i = 0; i < early; ++i) {
          if (kb_begin + i == p.skip_block) continue;
          mbar_arrive_expect_tx(bar_full + 8 * i, T::kStageBytes);
          for (int w = 0; w < kW; ++w)
            tma_load_2d(base + i * T::kStageBytes + w * kFp8TileBytes, &tmap_w, (kb_begin + i) * kFp8Block,
                        t.expert * p.w_rows + t.n * 128 + w * p.up_row0, bar_full + 8 * i);
        }
      }
      grid_dep_wait();
      for (int tile = tile0; tile < total && ok; tile += step) {
        const Fp8Tile t = fp8_tile_at<TOK>(tile, groups, p);
        const int w_row = t.expert * p.w_rows + t.n * 128;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          ok = wait_bounded_relaxed(bar_done + 8 * stage, phase, ctx, kStProducerEmpty, 40);
          if (!ok) break;
          if (kb != p.skip_block) {
            const uint32_t full = bar_full + 8 * stage, dst = base + stage * T::kStageBytes;
            if (issued >= early) {
              mbar_arrive_expect_tx(full, T::kStageBytes);
              for (int w = 0; w < kW; ++w)
                tma_load_2d(dst + w * kFp8TileBytes, &tmap_w, kb * kFp8Block, w_row + w * p.up_row0, full);
            }
            tma_load_2d(dst + kW * kFp8TileBytes, &tmap_x, kb * kFp8Block, t.row0, full);
          }
          if (issued < early) ++issued;
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) {                                    // gave up: no copy may be in flight into this CTA's memory when it exits
        const long long t0 = clock64();
        for (int i = 0; i < S; ++i)
          while (!mbar_try_wait(bar_full + 8 * ((stage + i) % S), stage + i < S ? phase : phase ^ 1))
            if (clock64() - t0 > ctx.limit) { atomicCAS(p.status, 0, kStDrain); break; }
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer: one thread
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_scaled(128, TOK);
      const uint64_t desc0 = make_kmajor_sw128_desc(base);
      int stage = 0, slot = 0, set = 0;
      uint32_t full_phase = 0, scales_phase = 0, free_phase = 1;      // (the first round of accumulators is free)
      bool ok = true;
      grid_dep_wait();
      for (int tile = tile0; tile < total && ok; tile += step) {
        ok = wait_bounded(bar_free + 8 * set, free_phase, ctx, kStMmaAccEmpty);
        if (!ok) break;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          const int q = (kb - kb_begin) & 3;
          if (q == 0) ok = wait_bounded(bar_scales + 8 * slot, scales_phase, ctx, kStEpilogueScales);
          ok = ok && wait_bounded(bar_full + 8 * stage, full_phase, ctx, kStMmaLdFull);
          if (!ok) break;
          tcgen05_fence_after_sync();
          const uint64_t a = desc0 + static_cast<uint64_t>((stage * T::kStageBytes) >> 4);
          const uint64_t b = a + static_cast<uint64_t>((kW * kFp8TileBytes) >> 4);
          const uint32_t scales = tmem + T::kScaleCol0 + slot * T::kSlotCols;
          const uint32_t id = idesc | scale_bytes_in_idesc(q);
#pragma unroll
          for (int w = 0; w < kW; ++w)
#pragma unroll
            for (int k = 0; k < 4; ++k)              // 32 bytes along K inside the swizzled row: +2 in the address field
              umma_f8_scaled<1>(tmem + (set * kW + w) * TOK, a + static_cast<uint64_t>(w * (kFp8TileBytes >> 4) + 2 * k),
                                b + static_cast<uint64_t>(2 * k), id, scales + 4 * w, scales + 4 * kW, kb > kb_begin || k > 0);
          umma_commit(bar_done + 8 * stage);
          if (q == 3 || kb + 1 == kb_end) {
            umma_commit(bar_scales_free + 8 * slot);
            if (++slot == T::kSlots) { slot = 0; scales_phase ^= 1; }
          }
          if (++stage == S) { stage = 0; full_phase ^= 1; }
        }
        if (ok) umma_commit(bar_sum + 8 * set);
        if (++set == T::kSums) { set = 0; free_phase ^= 1; }
      }
      if (!ok) {                                    // gave up: wait for the MMAs that still read shared memory
        umma_commit(bar_drain);
        const long long t0 = clock64();
        while (!mbar_try_wait(bar_drain, 0))
          if (clock64() - t0 > ctx.limit) { atomicCAS(p.status, 0, kStDrain); break; }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------ scales: lane l holds that of row l of X; W's tile has one
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + T::kScaleCol0;
    int slot = 0;
    uint32_t phase = 1;
    bool ok = true;
    grid_dep_wait();
    for (int tile = tile0; tile < total && ok; tile += step) {
      const Fp8Tile t = fp8_tile_at<TOK>(tile, groups, p);
      const long long ws0 = (t.expert * p.scale_rows + t.n) * p.k_blocks;
      // groups of four are counted from this CTA's first block, which need not lie on a multiple of four
      const bool whole_w = p.w_scale_groups && (kb_begin & 3) == 0, whole_x = p.x_scale_groups && (kb_begin & 3) == 0;
      uint32_t x, w[kW];
      auto fetch = [&](int kb) {
        x = load_exponents4(p.x_scale, static_cast<long long>(t.row0 + (lane < t.rows ? lane : 0)) * p.xs_row + kb * p.xs_blk, p.xs_blk, kb_end - kb, whole_x);
#pragma unroll
        for (int i = 0; i < kW; ++i) w[i] = load_exponents4(p.w_scale, ws0 + static_cast<long long>(i * p.up_block0) * p.k_blocks + kb, 1, kb_end - kb, whole_w);
      };
      if (kb_begin < kb_end) fetch(kb_begin);
      for (int kb = kb_begin; kb < kb_end; kb += 4) {
        ok = wait_bounded_relaxed(bar_scales_free + 8 * slot, phase, ctx, kStProducerEmpty, 40);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tcgen05_fence_after_sync();
        const uint32_t at = t_lane + slot * T::kSlotCols;
#pragma unroll
        for (int i = 0; i < kW; ++i) {
          const uint32_t sa[4] = {w[i], w[i], w[i], w[i]};
          tmem_st_32x4(at + 4 * i, sa);
        }
        const uint32_t sb[4] = {x, x, x, x};
        tmem_st_32x4(at + 4 * kW, sb);
        tmem_st_wait();
        tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_scales + 8 * slot);
        if (kb + 4 < kb_end) fetch(kb + 4);         // (scales read byte by byte are waited for: nobody else should)
        if (++slot == T::kSlots) { slot = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue: lane = feature, columns = rows of X
    const int feature = warp * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    int set = 0;
    uint32_t phase = 0;
    bool ok = true;
    grid_dep_wait();
    for (int tile = tile0; tile < total && ok; tile += step) {
      const Fp8Tile t = fp8_tile_at<TOK>(tile, groups, p);
      uint32_t v[kW][TOK];
      ok = wait_bounded_relaxed(bar_sum + 8 * set, phase, ctx, kStEpilogueAccFull, 20);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tcgen05_fence_after_sync();
#pragma unroll
        for (int w = 0; w < kW; ++w) {
          const uint32_t at = t_lane + (set * kW + w) * TOK;
          if constexpr (TOK == 32) tmem_ld_32x32(at, v[w]); else tmem_ld_32x16(at, v[w]);
        }
        tmem_ld_wait();
        tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_free + 8 * set);
      }
      if (++set == T::kSums) { set = 0; phase ^= 1; }
      // (the warps of the SiLU epilogue meet below: none may be waited for that has given up)
      if constexpr (SILU) ok = named_barrier_all(1, 128, ok);
      if (!ok) break;
      const int n = t.n * 128 + feature;
      auto sum = [&](int w, int j) { return __uint_as_float(v[w][j]); };
      if constexpr (SILU) {
        // a feature past the end counts as zero in its block's maximum
        float* part = reinterpret_cast<float*>(behind + T::kOffAmax);
        const bool live = n < p.N;
        float h[TOK];
#pragma unroll
        for (int j = 0; j < TOK; ++j) {
          if (j >= t.rows) break;                   // (most groups have a few rows)
          h[j] = live ? silu_times(sum(0, j), sum(1, j)) : 0.f;
          uint32_t a = __float_as_uint(h[j]) & 0x7fffffffu;      // (ordered like the values; NaN above all)
          a = __reduce_max_sync(0xffffffffu, a);
          if (lane == 0) part[warp * TOK + j] = __uint_as_float(a);
        }
        named_barrier_sync(1, 128);
        uint8_t* out = static_cast<uint8_t*>(p.out);
#pragma unroll
        for (int j = 0; j < TOK; ++j) {
          if (j < t.rows) {
            const uint32_t a = max(max(__float_as_uint(part[j]), __float_as_uint(part[TOK + j])),
                                   max(__float_as_uint(part[2 * TOK + j]), __float_as_uint(part[3 * TOK + j])));
            const bool bad = not_finite_bits(a);
            const int e = bad ? 0 : fp8_block_exponent(a);
            const long long m = t.row0 + j;
            if (live) out[m * p.ld_out + n] = bad ? 0x7f : static_cast<uint8_t>(e4m3x2(h[j] * pow2f(-e), 0.f) & 0xff);
            if (feature == 0) store_scale<true>(p.h_scale, m * p.hs_row + t.n * p.hs_blk, e, bad);
          }
        }
        named_barrier_sync(1, 128);                 // (the maxima are read before the next tile's are written)
      } else if (split > 1) {
        // CTA r of the cluster owns rows r * per .. of the tile (per is a power of two)
        const int shift = __ffs(TOK / split) - 1;
        const uint32_t red_at = smem_u32(red) + static_cast<uint32_t>((rank << shift) * 128 + feature) * 4;
#pragma unroll
        for (int j = 0; j < TOK; ++j)
          st_dsmem_f32(map_to_cta(red_at + static_cast<uint32_t>(j & ((1 << shift) - 1)) * 512, j >> shift), sum(0, j));
      } else if (n < p.N && p.out_f32) {
        float* out = static_cast<float*>(p.out) + static_cast<long long>(t.row0) * p.ld_out + n;
#pragma unroll
        for (int j = 0; j < TOK; ++j)
          if (j < t.rows) out[j * p.ld_out] = sum(0, j);
      } else if (n < p.N) {
        uint16_t* out = static_cast<uint16_t*>(p.out) + static_cast<long long>(t.row0) * p.ld_out + n;
#pragma unroll
        for (int j = 0; j < TOK; ++j)
          if (j < t.rows) out[j * p.ld_out] = round_out(sum(0, j), p.out_bf16);
      }
    }
    __syncwarp();
  }
  if (split > 1) {                                  // (split launches: one tile per cluster, never the SiLU epilogue)
    cluster_sync_all();
    if (warp < 4 && tile0 < total && !*abort_flag) {
      const Fp8Tile t = fp8_tile_at<TOK>(tile0, groups, p);
      const int n = t.n * 128 + warp * 32 + lane, per = TOK / split, last = min(per, t.rows - rank * per);
      const float* from = red + warp * 32 + lane;
      uint16_t* out = static_cast<uint16_t*>(p.out) + static_cast<long long>(t.row0 + rank * per) * p.ld_out + n;
      for (int j = 0; j < last; ++j) {
        float sum = from[j * 128];
        for (int r = 1; r < split; ++r) sum += from[(r * per + j) * 128];
        if (n < p.N) out[j * p.ld_out] = round_out(sum, p.out_bf16);
      }
    }
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    tcgen05_fence_after_sync();
    tmem_dealloc(tmem, T::kTmemCols);
  }
}

}  // namespace sk
