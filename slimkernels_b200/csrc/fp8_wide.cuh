// The FP8 product for many rows: 128 rows of X on the tensor memory's lanes, 256 features on its columns.
//
// With rows on the lanes the scale of a K block's partial sums is one number per thread and weight block (the row's scale times the
// block's), so the epilogue is one FFMA per value; with features on the lanes every column has its own scale, a load more per four.  256
// columns instead of 128 halve the bytes of X that a MMA reads again.
//
// Two accumulators of 256 columns fill the tensor memory: the MMAs of one K block run while eight warps drain the other.
//   producer   one thread: TMA of 128 x 128 B of X and two boxes of 128 x 128 B of W per K block, four stages of 48 KiB
//   issuer     one thread: four MMAs of 128 x 256 x 32 per K block and one commit, which serves the producer and the epilogue
//   epilogue   two warpgroups, each a row per thread and 128 of the 256 columns, fp32 sums in registers
// The CTAs stay and walk the tiles; the operands of the next tile are on their way while a tile is written.
//
// What bounds it: 4096 x 8192 x 8192 takes 309 us (1780 TFLOP/s; 260 before the power settles), about 1050 cycles a K block.  The MMAs are 512 of
// them, shared memory (48 KiB in by TMA, 48 KiB out to the tensor core, 128 B a cycle) makes that 768.  The 128 FFMAs of each epilogue thread add
// 200 to 250 wherever they stand, with operands of zeros (no power limit) as well: 223 us, 180 without them, 176 without the loads of the sums, too.
// Measured and not kept: pairs of CTAs (shared memory then takes 512: 253 against 257 us, ragged groups up to 40 % slower), accumulators in four halves
// with barriers of their own (2 % faster here, up to 13 % slower with 16 K blocks), two warps that multiply the scales, results through shared memory,
// sixteen epilogue warps, the next block's columns loaded ahead, a second issuer (nothing), two FFMAs an instruction (spills).  With 8-bit
// scales none of this is needed (fp8_scaled.cuh).
//
// SILU: the columns are 128 gate features and the 128 up features beside them, and a thread takes 64 of either, so that SiLU(gate) * up
// and its quantisation (one block of the next product per row) stay in registers but for the two halves' maxima.
#pragma once
#include "fp8_common.cuh"

namespace sk {

template <bool SILU>
struct Fp8WideTraits {
  static constexpr int kStages = 4, kBufs = 2;
  static constexpr int kRing = kStages;             // "block done" barriers: R >= S and R >= B, as in the narrow kernel
  static constexpr int kStageBytes = 3 * kFp8TileBytes;
  static constexpr int kOffBar = kStages * kStageBytes;
  static constexpr int kNumBars = kStages + kRing + kBufs + 1;
  static constexpr int kOffMisc = (kOffBar + kNumBars * 8 + 15) / 16 * 16;
  static constexpr int kSlots = 3;                  // groups of four K blocks whose scales are held or on their way
  static constexpr int kOffXScale = kOffMisc + 16;  // [kSlots][256 epilogue threads][4]
  static constexpr int kOffWScale = kOffXScale + kSlots * 256 * 16;      // [kSlots][8 warps][2 weight blocks][4]
  static constexpr int kOffAmax = kOffWScale + kSlots * 8 * 32;          // SILU: [2 warpgroups][128 rows]
  static constexpr int kOffTable = kOffAmax + (SILU ? 2 * 128 * 4 : 8 * kTurnBytes);      // (else the warps' corners)
  static constexpr int kThreads = 384;             // two epilogue warpgroups, one for the producer and the issuer
  // Registers: 168 a thread at launch; the epilogue's 128 sums and 32 loaded values take more, the other roles less.
  static constexpr int kEpilogueRegs = 232, kOtherRegs = 40;
  static_assert(256 * kEpilogueRegs + 128 * kOtherRegs <= kThreads * 168, "a larger sum would wait forever");
  static constexpr int dynamic_bytes(int experts) { return kOffTable + group_table_bytes(experts) + 1024; }
};
static_assert(Fp8WideTraits<true>::dynamic_bytes(kFp8MaxExperts) <= 232448 && Fp8WideTraits<false>::dynamic_bytes(kFp8MaxExperts) <= 232448,
              "shared memory of a CTA");

template <bool SILU>
__global__ void __launch_bounds__(384, 1)
fp8_wide_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Fp8Params p) {
  using T = Fp8WideTraits<SILU>;
  constexpr int S = T::kStages, B = T::kBufs, R = T::kRing;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(smem);
  const uint32_t bar_full = base + T::kOffBar, bar_done = bar_full + 8 * S, bar_free = bar_done + 8 * R, bar_drain = bar_free + 8 * B;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + T::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + T::kOffMisc + 4);
  const WaitCtx ctx{abort_flag, p.status, p.wait_limit};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* table = reinterpret_cast<int*>(smem + T::kOffTable);
  const GroupTable groups{table, table + p.experts + 1};

  grid_dep_launch_dependents();
  if (threadIdx.x == 256) {
    for (int i = 0; i < S; ++i) mbar_init(bar_full + 8 * i, 1);
    for (int i = 0; i < R; ++i) mbar_init(bar_done + 8 * i, 1);
    for (int i = 0; i < B; ++i) mbar_init(bar_free + 8 * i, 8);
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&tmap_w);
    prefetch_tensormap(&tmap_x);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    tmem_relinquish();
  }
  if (p.offsets != nullptr && warp == 0) {
    if (!p.early_weights) grid_dep_wait();
    build_group_table<128>(groups, p, lane);
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const int total = fp8_total_tiles<128>(groups, p);
  const int up_rows = SILU ? p.up_row0 : 128;       // from a tile's first weight box to its second

  if (warp >= 8) {
    setmaxnreg_dec<T::kOtherRegs>();
    if (warp == 8) {
      // ------------------------------------------------------------ producer: one thread
      if (elect_one()) {
        long long issued = 0;
        int stage = 0, ring = 0;
        uint32_t phase = 1;                           // (the first round of stages is free)
        bool ok = true;
        grid_dep_wait();
        for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
          const Fp8Tile t = fp8_tile_at<128>(tile, groups, p);
          const int w_row = t.expert * p.w_rows + t.n * (SILU ? 128 : 256);
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            ok = wait_bounded_relaxed(bar_done + 8 * ring, phase, ctx, kStProducerEmpty, 40);
            if (!ok) break;
            if (kb != p.skip_block) {
              const uint32_t full = bar_full + 8 * stage, dst = base + stage * T::kStageBytes;
              mbar_arrive_expect_tx(full, T::kStageBytes);
              tma_load_2d(dst, &tmap_x, kb * kFp8Block, t.row0, full);
              tma_load_2d(dst + kFp8TileBytes, &tmap_w, kb * kFp8Block, w_row, full);
              tma_load_2d(dst + 2 * kFp8TileBytes, &tmap_w, kb * kFp8Block, w_row + up_rows, full);
            }
            ++issued;
            if (++stage == S) stage = 0;
            if (++ring == R) { ring = 0; phase ^= 1; }
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
    } else if (warp == 9) {
      // ------------------------------------------------------------ MMA issuer: one thread
      if (elect_one()) {
        constexpr uint32_t idesc = make_idesc_e4m3(128, 256);
        const uint64_t desc0 = make_kmajor_sw128_desc(base);
        int stage = 0, buf = 0, ring = 0;
        uint32_t full_phase = 0, free_phase = 1;
        bool ok = true;
        grid_dep_wait();
        for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x)
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            ok = wait_bounded_two(bar_full + 8 * stage, full_phase, bar_free + 8 * buf, free_phase, ctx, kStMmaLdFull, kStMmaAccEmpty);
            if (!ok) break;
            tcgen05_fence_after_sync();
            const uint64_t a = desc0 + static_cast<uint64_t>((stage * T::kStageBytes) >> 4);
            const uint64_t b = a + static_cast<uint64_t>(kFp8TileBytes >> 4);      // (the two boxes lie one behind the other)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f8(tmem + buf * 256, a + static_cast<uint64_t>(2 * k), b + static_cast<uint64_t>(2 * k), idesc, k > 0);
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
    }
  } else {
    setmaxnreg_inc<T::kEpilogueRegs>();
    // ------------------------------------------------------------ epilogue: lane = row, columns = features
    const int wg = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    int buf = 0, ring = 0;
    uint32_t done_phase = 0;
    const uint32_t xs_slot = base + T::kOffXScale + threadIdx.x * 16, ws_slot = base + T::kOffWScale + warp * 32;
    bool ok = true;
    grid_dep_wait();
    for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
      const Fp8Tile t = fp8_tile_at<128>(tile, groups, p);
      const bool live = row < t.rows;
      // Scales come four K blocks at a time, two groups ahead, as asynchronous copies into shared memory that only this thread (a row's) or
      // warp (the weight blocks') reads.  (As plain loads, one group ahead, they cost the epilogue a stall of 900 cycles every four K blocks,
      // although nothing used them: a warp's few scoreboards are shared with the barriers' answers.)
      const float* x_scale = static_cast<const float*>(p.x_scale) + static_cast<long long>(t.row0 + (live ? row : 0)) * p.xs_row;
      // the weight blocks that this warp's columns need: one (its 128 columns; past the end any), or the gate's and the up projection's
      const int n_block = SILU ? t.n : (2 * t.n + wg) * 128 < p.N ? 2 * t.n + wg : 2 * t.n;
      const float* w_scale = static_cast<const float*>(p.w_scale) + (t.expert * p.scale_rows + n_block) * p.k_blocks;
      const float* up_scale = w_scale + static_cast<long long>(p.up_block0) * p.k_blocks;
      auto fetch = [&](int g) {                     // the scales of blocks 4 g .. 4 g + 3, as far as they exist
        const int slot = g % T::kSlots, kb = 4 * g;
        if (kb < p.k_blocks) {
          copy_scales4(xs_slot + slot * (256 * 16), x_scale + kb * p.xs_blk, p.xs_blk, p.k_blocks - kb, p.x_scale_groups);
          if (lane == 0) copy_scales4(ws_slot + slot * (8 * 32), w_scale + kb, 1, p.k_blocks - kb, p.w_scale_groups);
          if (SILU && lane == 1) copy_scales4(ws_slot + slot * (8 * 32) + 16, up_scale + kb, 1, p.k_blocks - kb, p.w_scale_groups);
        }
        cp_async_commit();
      };
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.f;
      fetch(0);
      fetch(1);
      for (int kb0 = 0; kb0 < p.k_blocks && ok; kb0 += 4) {
        const int slot = (kb0 >> 2) % T::kSlots;
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        const float4 x4 = lds_f32x4(xs_slot + slot * (256 * 16)), w4 = lds_f32x4(ws_slot + slot * (8 * 32));
        const float4 u4 = SILU ? lds_f32x4(ws_slot + slot * (8 * 32) + 16) : w4;
        const float s0[4] = {x4.x * w4.x, x4.y * w4.y, x4.z * w4.z, x4.w * w4.w};
        const float s1[4] = {x4.x * u4.x, x4.y * u4.y, x4.z * u4.z, x4.w * u4.w};
        __syncwarp();                               // (read by all lanes before the slot is written again)
        fetch((kb0 >> 2) + 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (kb0 + i >= p.k_blocks) break;
          ok = wait_bounded(bar_done + 8 * ring, done_phase, ctx, kStEpilogueAccFull);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tcgen05_fence_after_sync();
          const uint32_t from = t_lane + buf * 256 + (SILU ? wg * 64 : wg * 128);
          uint32_t v[2][32];
          auto load = [&](int c) { tmem_ld_32x32(from + (SILU ? (c >> 1) * 128 + (c & 1) * 32 : c * 32), v[c & 1]); };
          auto add = [&](int c) {
            const float f = SILU && c >= 2 ? s1[i] : s0[i];
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[32 * c + j] = fmaf(__uint_as_float(v[c & 1][j]), f, acc[32 * c + j]);
          };
          // 64 columns at a time: the second half's loads go out between the first half's sums.  (Handing the buffer back before the second
          // half is added is 2 % slower, 316 us instead of 309 on 4096 x 8192 x 8192.)
          load(0);
          load(1);
          tmem_ld_wait();
          add(0);
          load(2);
          add(1);
          load(3);
          tmem_ld_wait();
          add(2);
          add(3);
          tcgen05_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_free + 8 * buf);
          if (++buf == B) buf = 0;
          if (++ring == R) { ring = 0; done_phase ^= 1; }
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      // (the warps of the SiLU epilogue meet below: none may be waited for that has given up)
      if constexpr (SILU) ok = named_barrier_all(1, 256, ok);
      if (!ok) break;
      const long long m = t.row0 + row;
      if constexpr (SILU) {
        float* part = reinterpret_cast<float*>(smem + T::kOffAmax);
        const int n0 = t.n * 128 + wg * 64;
        uint32_t a = 0;
#pragma unroll
        for (int j = 0; j < 64; ++j) {              // a feature past the end counts as zero in its block's maximum
          acc[j] = n0 + j < p.N ? silu_times(acc[j], acc[64 + j]) : 0.f;
          a = max(a, __float_as_uint(acc[j]) & 0x7fffffffu);
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
          for (int c = 0; c < 2; ++c) store_codes32(dst + 32 * c, p.N - n0 - 32 * c, inv, bad, [&](int j) { return acc[32 * c + j]; });
          if (wg == 0) store_scale<false>(p.h_scale, m * p.hs_row + t.n * p.hs_blk, e, bad);
        }
      } else if (p.out_f32) {
        const int n0 = t.n * 256 + wg * 128;
        float* dst = static_cast<float*>(p.out) + m * p.ld_out + n0;
        if (live) {
#pragma unroll
          for (int c = 0; c < 8; ++c) store_row16_f32(dst + 16 * c, p.N - n0 - 16 * c, [&](int j) { return acc[16 * c + j]; });
        }
      } else if (p.out_bytes == 2) {
        const int n0 = t.n * 256 + wg * 128, first = (warp & 3) * 32;
        store_rows_turned(static_cast<uint16_t*>(p.out) + (t.row0 + first) * p.ld_out + n0, p.ld_out, min(32, t.rows - first), p.N - n0,
                          smem + T::kOffAmax + warp * kTurnBytes, lane, p.out_bf16, [&](int j) { return acc[j]; });
      } else if (live) {
        const int n0 = t.n * 256 + wg * 128;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + m * p.ld_out + n0;
#pragma unroll
        for (int c = 0; c < 8; ++c) store_row16(dst + 16 * c, p.N - n0 - 16 * c, p.out_bytes, p.out_bf16, [&](int j) { return acc[16 * c + j]; });
      }
    }
    __syncwarp();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    tcgen05_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace sk
