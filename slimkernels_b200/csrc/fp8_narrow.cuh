// The FP8 product for few rows and 32-bit scales: y = X W^T with the weights' 128 features on the tensor memory's lanes and 16 rows of X on its
// columns.
//
// With few rows a product is a stream of weights: every weight byte is used once per row tile, the tensor core has next to nothing
// to do, and HBM bounds the time.  So a CTA is a ring of K blocks on their way (16 KiB of weights and 2 KiB of activations each, two CTAs to an SM,
// 90 KiB in flight each), one thread that issues four MMAs per K block, and four epilogue warps that take a block's 128 x 16 partial sums out of
// tensor memory, scale them (the row scales come as broadcast loads from a warp's own corner of shared memory, four K blocks at a time and one
// group ahead) and add them up in registers.  One commit per K block serves the producer and the epilogue.  A CTA so gets through a K block in about 700
// cycles, 44 GB/s; 16 x 22016 x 4096 takes 18.7 us (4.9 TB/s), 16 x 4096 x 4096 in four splits 9.6 us.
//
// A tile's K range can be split over a cluster: every CTA pushes its sums into the CTA that owns the row (remote stores), one cluster
// barrier, then the owner adds them in rank order, so the result does not depend on timing.
//
// SILU: the tile holds 128 gate features and the 128 up features beside them; the epilogue forms SiLU(gate) * up in fp32 and
// quantises it: 128 features of a row are just one block of the next product, so its maximum is one reduction over the CTA's lanes.
#pragma once
#include "fp8_common.cuh"

namespace sk {

template <bool SILU>
struct Fp8NarrowTraits {
  static constexpr int TOK = 16;                                // rows per tile
  static constexpr int kW = SILU ? 2 : 1;                       // weight tiles per K block
  static constexpr int kXBytes = TOK * kFp8Block;
  static constexpr int kStageBytes = kW * kFp8TileBytes + kXBytes;
  static constexpr int kStages = SILU ? 3 : 5;                  // two CTAs to an SM
  static constexpr int kTmemCols = 256;
  static constexpr int kBufs = kTmemCols / (kW * TOK) > 8 ? 8 : kTmemCols / (kW * TOK);   // accumulator buffers
  static constexpr int kRing = kStages > kBufs ? kStages : kBufs;   // "block done" barriers: see the kernel
  static constexpr int kScaleBytes = 4 * kW * 4 * TOK * 4;      // [warp][weight tile][4 K blocks][TOK] floats
  static constexpr int kOffScale = kStages * kStageBytes;
  static constexpr int kOffBar = kOffScale + kScaleBytes;
  static constexpr int kNumBars = kStages + kRing + kBufs + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kOffAmax = kOffMisc + 16;                // SILU: [4 warps][TOK]
  static constexpr int kOffTail = ((kOffAmax + (SILU ? 4 * TOK * 4 : 0) + 15) / 16) * 16;   // reduction buffer, or the group table
  static constexpr int kRedBytes = TOK * 128 * 4;
  static constexpr int kThreads = 192;
  static constexpr int dynamic_bytes(int split, int experts) {
    return kOffTail + (split > 1 ? kRedBytes : 0) + group_table_bytes(experts) + 1024;
  }
};

template <bool SILU>
__global__ void __launch_bounds__(192, 2)
fp8_narrow_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Fp8Params p) {
  using T = Fp8NarrowTraits<SILU>;
  constexpr int TOK = T::TOK;
  constexpr int S = T::kStages, B = T::kBufs, R = T::kRing, kW = T::kW;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(smem);
  const uint32_t bar_full = base + T::kOffBar;      // [S] the copies of a K block have landed
  // [R] the MMAs of K block j have completed, j mod R.  The producer (which waits for block j before it refills its stage) and the
  // epilogue (before it reads its accumulators) watch the same barrier; with R >= S and R >= B neither can be overtaken by the phase
  // after next, because block j + R needs the stage of block j + R - S and the accumulators of block j + R - B.
  const uint32_t bar_done = bar_full + 8 * S;
  const uint32_t bar_free = bar_done + 8 * R;       // [B] the epilogue has read the accumulators
  const uint32_t bar_drain = bar_free + 8 * B;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + T::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + T::kOffMisc + 4);
  const WaitCtx ctx{abort_flag, p.status, p.wait_limit};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int rank = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  uint8_t* tail = smem + T::kOffTail;
  float* red = reinterpret_cast<float*>(tail);
  int* table = reinterpret_cast<int*>(tail + (split > 1 ? T::kRedBytes : 0));
  const GroupTable groups{table, table + p.experts + 1};

  grid_dep_launch_dependents();
  if (threadIdx.x == 128) {
    for (int i = 0; i < S; ++i) mbar_init(bar_full + 8 * i, 1);
    for (int i = 0; i < R; ++i) mbar_init(bar_done + 8 * i, 1);
    for (int i = 0; i < B; ++i) mbar_init(bar_free + 8 * i, 4);
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&tmap_w);
    prefetch_tensormap(&tmap_x);
  }
  if (warp == 5) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), T::kTmemCols);
    tmem_relinquish();
  }
  if (p.offsets != nullptr && warp == 0) {
    if (!p.early_weights) grid_dep_wait();
    build_group_table<TOK>(groups, p, lane);
  }
  tcgen05_fence_before_sync();
  if (split > 1) cluster_sync_all(); else __syncthreads();      // (peers push into this CTA's memory only once it runs)
  tcgen05_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  const int total = fp8_total_tiles<TOK>(groups, p);
  const int tile0 = static_cast<int>(blockIdx.x) / split, step = static_cast<int>(gridDim.x) / split;
  // this CTA's share of the K blocks of a tile
  const int kb_begin = p.k_blocks * rank / split, kb_end = p.k_blocks * (rank + 1) / split;

  if (warp == 4) {
    // ------------------------------------------------------------ producer: one thread
    if (elect_one()) {
      long long issued = 0;
      int stage = 0, early = 0;
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
          if (issued >= S) {
            const long long j = issued - S;
            ok = wait_bounded_relaxed(bar_done + 8 * static_cast<int>(j % R), static_cast<int>(j / R) & 1, ctx, kStProducerEmpty, 40);
            if (!ok) break;
          }
          if (kb != p.skip_block) {
            const uint32_t full = bar_full + 8 * stage, dst = base + stage * T::kStageBytes;
            if (issued >= early) {
              mbar_arrive_expect_tx(full, T::kStageBytes);
              for (int w = 0; w < kW; ++w)
                tma_load_2d(dst + w * kFp8TileBytes, &tmap_w, kb * kFp8Block, w_row + w * p.up_row0, full);
            }
            tma_load_2d(dst + kW * kFp8TileBytes, &tmap_x, kb * kFp8Block, t.row0, full);
          }
          ++issued;
          if (++stage == S) stage = 0;
        }
      }
      if (!ok) {                                    // gave up: no copy may be in flight into this CTA's memory when it exits
        const long long t0 = clock64();
        for (long long i = issued > S ? issued - S : 0; i < issued; ++i)
          while (!mbar_try_wait(bar_full + 8 * static_cast<int>(i % S), static_cast<int>(i / S) & 1))
            if (clock64() - t0 > ctx.limit) { atomicCAS(p.status, 0, kStDrain); break; }
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issuer: one thread
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_e4m3(128, TOK);
      const uint64_t desc0 = make_kmajor_sw128_desc(base);
      int stage = 0, buf = 0, ring = 0;
      uint32_t full_phase = 0, free_phase = 1;      // (the first round of buffers is free)
      bool ok = true;
      grid_dep_wait();
      for (int tile = tile0; tile < total && ok; tile += step)
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          ok = wait_bounded(bar_full + 8 * stage, full_phase, ctx, kStMmaLdFull) &&
               wait_bounded(bar_free + 8 * buf, free_phase, ctx, kStMmaAccEmpty);
          if (!ok) break;
          tcgen05_fence_after_sync();
          const uint64_t a = desc0 + static_cast<uint64_t>((stage * T::kStageBytes) >> 4);
          const uint64_t b = a + static_cast<uint64_t>((kW * kFp8TileBytes) >> 4);
#pragma unroll
          for (int w = 0; w < kW; ++w)
#pragma unroll
            for (int k = 0; k < 4; ++k)              // 32 bytes along K inside the swizzled row: +2 in the address field
              umma_f8(tmem + buf * (kW * TOK) + w * TOK, a + static_cast<uint64_t>(w * (kFp8TileBytes >> 4) + 2 * k),
                      b + static_cast<uint64_t>(2 * k), idesc, k > 0);
          umma_commit(bar_done + 8 * ring);
          if (++stage == S) { stage = 0; full_phase ^= 1; }
          if (++buf == B) { buf = 0; free_phase ^= 1; }
          if (++ring == R) ring = 0;
        }
      if (!ok) {                                    // gave up: wait for the MMAs that still read shared memory
        umma_commit(bar_drain);
        const long long t0 = clock64();
        while (!mbar_try_wait(bar_drain, 0))
          if (clock64() - t0 > ctx.limit) { atomicCAS(p.status, 0, kStDrain); break; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue: lane = feature, columns = rows of X
    constexpr int kPer = TOK / 8;                   // scales that a lane fetches per four K blocks
    float* slot = reinterpret_cast<float*>(smem + T::kOffScale) + warp * (kW * 4 * TOK);
    const int feature = warp * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    int buf = 0, ring = 0;
    uint32_t done_phase = 0;
    bool ok = true;
    grid_dep_wait();
    for (int tile = tile0; tile < total && ok; tile += step) {
      const Fp8Tile t = fp8_tile_at<TOK>(tile, groups, p);
      const long long ws0 = (t.expert * p.scale_rows + t.n) * p.k_blocks;
      float xv[kPer], wv[kW][kPer];
      auto fetch = [&](int kb0) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int idx = lane + 32 * i, kb = kb0 + idx / TOK, tok = idx % TOK;
          const bool on = kb < kb_end && tok < t.rows;
          xv[i] = on ? ld_global_f32(static_cast<const float*>(p.x_scale) + static_cast<long long>(t.row0 + tok) * p.xs_row + kb * p.xs_blk) : 0.f;
#pragma unroll
          for (int w = 0; w < kW; ++w)
            wv[w][i] = on ? ld_global_f32(static_cast<const float*>(p.w_scale) + ws0 + static_cast<long long>(w * p.up_block0) * p.k_blocks + kb) : 0.f;
        }
      };
      float acc[kW][TOK];
#pragma unroll
      for (int w = 0; w < kW; ++w)
#pragma unroll
        for (int j = 0; j < TOK; ++j) acc[w][j] = 0.f;
      fetch(kb_begin);
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        const int q = (kb - kb_begin) & 3;
        if (q == 0) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int w = 0; w < kW; ++w) slot[w * 4 * TOK + lane + 32 * i] = xv[i] * wv[w][i];
          __syncwarp();
          fetch(kb + 4);
        }
        ok = wait_bounded(bar_done + 8 * ring, done_phase, ctx, kStEpilogueAccFull);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tcgen05_fence_after_sync();
#pragma unroll
        for (int w = 0; w < kW; ++w) {
          uint32_t v[TOK];
          tmem_ld_32x16(t_lane + buf * (kW * TOK) + w * TOK, v);
          tmem_ld_wait();
          if (w == kW - 1) {                        // the last read of this buffer
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_free + 8 * buf);
          }
          const float4* s4 = reinterpret_cast<const float4*>(slot + w * 4 * TOK + q * TOK);
#pragma unroll
          for (int j = 0; j < TOK; j += 4) {
            const float4 s = s4[j / 4];
            acc[w][j] = fmaf(__uint_as_float(v[j]), s.x, acc[w][j]);
            acc[w][j + 1] = fmaf(__uint_as_float(v[j + 1]), s.y, acc[w][j + 1]);
            acc[w][j + 2] = fmaf(__uint_as_float(v[j + 2]), s.z, acc[w][j + 2]);
            acc[w][j + 3] = fmaf(__uint_as_float(v[j + 3]), s.w, acc[w][j + 3]);
          }
        }
        if (++buf == B) buf = 0;
        if (++ring == R) { ring = 0; done_phase ^= 1; }
      }
      // (the warps of the SiLU epilogue meet below: none may be waited for that has given up)
      if constexpr (SILU) ok = named_barrier_all(1, 128, ok);
      if (!ok) break;
      const int n = t.n * 128 + feature;
      if constexpr (SILU) {
        // a feature past the end counts as zero in its block's maximum
        float* part = reinterpret_cast<float*>(smem + T::kOffAmax);
        const bool live = n < p.N;
#pragma unroll
        for (int j = 0; j < TOK; ++j) {
          if (j >= t.rows) break;
          acc[0][j] = live ? silu_times(acc[0][j], acc[1][j]) : 0.f;
          uint32_t a = __float_as_uint(acc[0][j]) & 0x7fffffffu;      // (ordered like the values; NaN above all)
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
            if (live) out[m * p.ld_out + n] = bad ? 0x7f : static_cast<uint8_t>(e4m3x2(acc[0][j] * pow2f(-e), 0.f) & 0xff);
            if (feature == 0) store_scale<false>(p.h_scale, m * p.hs_row + t.n * p.hs_blk, e, bad);
          }
        }
        named_barrier_sync(1, 128);                 // (the maxima are read before the next tile's are written)
      } else if (split > 1) {
        // CTA r of the cluster owns rows r * per .. of the tile (per is a power of two)
        const int shift = __ffs(TOK / split) - 1;
        const uint32_t red_at = smem_u32(red) + static_cast<uint32_t>((rank << shift) * 128 + feature) * 4;
#pragma unroll
        for (int j = 0; j < TOK; ++j)
          st_dsmem_f32(map_to_cta(red_at + static_cast<uint32_t>(j & ((1 << shift) - 1)) * 512, j >> shift), acc[0][j]);
      } else if (n < p.N && p.out_f32) {
        float* out = static_cast<float*>(p.out) + static_cast<long long>(t.row0) * p.ld_out + n;
#pragma unroll
        for (int j = 0; j < TOK; ++j)
          if (j < t.rows) out[j * p.ld_out] = acc[0][j];
      } else if (n < p.N) {
        uint16_t* out = static_cast<uint16_t*>(p.out) + static_cast<long long>(t.row0) * p.ld_out + n;
#pragma unroll
        for (int j = 0; j < TOK; ++j)
          if (j < t.rows) out[j * p.ld_out] = round_out(acc[0][j], p.out_bf16);
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
  if (warp == 5) {
    tcgen05_fence_after_sync();
    tmem_dealloc(tmem, T::kTmemCols);
  }
}

}  // namespace sk
