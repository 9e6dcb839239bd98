// What the FP8 kernels share: the operands of a product, scales in either form, and the row groups of a product by expert.
//
// A tensor is held as e4m3 codes and one scale per block of 128 along K (activations: per row; weights: per 128 rows):
//   out[m, n] = round( sum_b xs[m, b] * ws[n / 128, b] * P_b[m, n] ),   P_b = sum over the 128 k of block b of xq[m, k] * wq[n, k]
// P_b comes from tcgen05.mma kind::f8f6f4 in fp32 (products of two e4m3 values are exact); the scales are applied in fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx_sm100.cuh"
#include "waits.cuh"

namespace sk {

constexpr int kFp8Block = 128;          // elements along K, and weight rows, per scale
constexpr int kFp8TileBytes = 128 * 128;  // 128 rows of one K block
constexpr int kFp8MaxExperts = 1024;

struct Fp8Params {
  const void* x_scale;                  // element (m, b) at m * xs_row + b * xs_blk
  long long xs_row, xs_blk;
  const void* w_scale;                  // [experts][scale_rows][k_blocks] contiguous
  long long scale_rows;                 // blocks of 128 rows per expert (gate and up together)
  const int* offsets;                   // [experts + 1] first rows of the groups, or nullptr: one group of all rows
  int experts;
  int w_rows;                           // weight rows per expert
  void* out;                            // [M, ld_out] half / bf16 / fp32; with the SiLU epilogue: e4m3 codes
  long long ld_out;
  void* h_scale;                        // SiLU epilogue: the codes' scales, element (m, b) at m * hs_row + b * hs_blk
  long long hs_row, hs_blk;
  int M, N;                             // N: features of `out`
  int k_blocks;
  int n_tiles;                          // feature tiles of this kernel's width
  int up_row0;                          // SiLU epilogue: the up projection's first row / scale block within an expert
  int up_block0;
  int out_bf16;
  int out_f32;                          // the result is kept in fp32 (the expert layers' second product; rows on 64 bytes)
  int x_scale_groups, w_scale_groups;   // the scales of four K blocks may be loaded at once (side by side and aligned)
  int out_bytes;                        // what the rows of the result start on: 32, 16 or 2 bytes
  int early_weights;                    // the weights may be read before the previous kernel is complete
  int stages;                           // depth of the ring (kernels whose launch decides it)
  int split;                            // CTAs of a cluster that share the K range of a tile
  int skip_block;                       // failure-path test hook: this K block's copies are left out (-1: off)
  long long wait_limit;
  int* status;
};

// The 8-bit scales of up to four K blocks from element i on, `left` of which exist, in the bytes of a word.
__device__ __forceinline__ uint32_t load_exponents4(const void* base, long long i, long long step, int left, bool whole) {
  const uint8_t* p = static_cast<const uint8_t*>(base) + i;
  uint32_t w = 0;
  if (whole && left >= 4) {
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(w) : "l"(p) : "memory");
    return w;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) {
      uint32_t b;
      asm volatile("ld.global.u8 %0, [%1];" : "=r"(b) : "l"(p + j * step) : "memory");
      w |= b << (8 * j);
    }
  return w;
}
// Asynchronous copies of the 32-bit scales of up to four K blocks to 16 bytes of shared memory.
__device__ __forceinline__ void copy_scales4(uint32_t to, const float* from, long long step, int left, bool whole) {
  if (whole && left >= 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4 * j), "l"(from + j * step) : "memory");
}

// The exponent e of a block's scale 2^e: the smallest with amax <= 448 * 2^e, from amax's bits (448 = 1.75 * 2^8); 0 for an
// all-zero block, never below -126, so that the scale is a normal float.
__device__ __forceinline__ int fp8_block_exponent(uint32_t amax_bits) {
  if (amax_bits == 0) return 0;
  const int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -126);
}
__device__ __forceinline__ bool not_finite_bits(uint32_t abs_bits) { return abs_bits >= 0x7f800000u; }
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }   // -126 <= e <= 127

// Two values, times 2^-e (exact above the subnormals), as e4m3 (nearest, ties to even).  The caller has seen to it that nothing
// exceeds 448.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Stores a block's scale.
template <bool E8M0>
__device__ __forceinline__ void store_scale(void* base, long long i, int e, bool bad) {
  if constexpr (E8M0)
    static_cast<uint8_t*>(base)[i] = static_cast<uint8_t>(bad ? 255 : e + 127);
  else
    static_cast<float*>(base)[i] = bad ? __uint_as_float(0x7fc00000u) : pow2f(e);
}

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 operands, fp32 accumulators, K = 32 per instruction.
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor, kind::f8f6f4: [4,6) D format (1 = fp32), [7,10) / [10,13) A / B format (0 = e4m3), K-major both,
// [17,23) N >> 3, [24,29) M >> 4.
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int mma_m, int mma_n) {
  return (1u << 4) | (static_cast<uint32_t>(mma_n >> 3) << 17) | (static_cast<uint32_t>(mma_m >> 4) << 24);
}

// ---------------------------------------------------------------- rows by expert
// Table in shared memory: start[0 .. experts], the groups' first rows (cut to [0, M] and made non-decreasing, so that whatever
// the caller's offsets hold nothing outside the operands is touched), and first[0 .. experts], the number of row tiles in front
// of a group.  Built by warp 0.
struct GroupTable {
  int* start;
  int* first;
};
__host__ __device__ constexpr int group_table_bytes(int experts) { return 2 * (experts + 1) * 4; }

__device__ __forceinline__ float lds_f32(uint32_t addr) {   // stays where it is
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 lds_f32x4(uint32_t addr) {   // 16-byte aligned; stays where it is
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int ld_global_int(const int* p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

template <int ROWS>
__device__ __forceinline__ void build_group_table(const GroupTable& t, const Fp8Params& p, int lane) {
  int row = 0, tiles = 0;               // carried from one batch of 32 experts to the next
  row = min(max(ld_global_int(p.offsets), 0), p.M);
  for (int e0 = 0; e0 < p.experts; e0 += 32) {
    const int e = e0 + lane;
    int end = e < p.experts ? min(max(ld_global_int(p.offsets + e + 1), 0), p.M) : 0;
    end = max(end, row);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end = max(end, up);
    }
    int begin = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) begin = row;
    const int mine = e < p.experts ? (end - begin + ROWS - 1) / ROWS : 0;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (e < p.experts) {
      t.start[e] = begin;
      t.first[e] = tiles + incl - mine;
    }
    row = __shfl_sync(0xffffffffu, end, 31);
    tiles += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) {
    t.start[p.experts] = row;
    t.first[p.experts] = tiles;
  }
}

// Tiles are numbered group by group; inside a group in bands of kBandTiles row tiles, feature tile by feature tile inside a band,
// so that the CTAs in flight share weights and activations in L2.
constexpr int kBandTiles = 32;
struct Fp8Tile {
  int expert, row0, rows, n;            // rows: how many of the tile's rows belong to the group
};
template <int ROWS>
__device__ __forceinline__ int fp8_total_tiles(const GroupTable& t, const Fp8Params& p) {
  return (p.offsets ? t.first[p.experts] : (p.M + ROWS - 1) / ROWS) * p.n_tiles;
}
template <int ROWS>
__device__ __forceinline__ Fp8Tile fp8_tile_at(int tile, const GroupTable& t, const Fp8Params& p) {
  int e = 0, lo = 0, hi = p.M, mt = (p.M + ROWS - 1) / ROWS;
  if (p.offsets) {
    const int rt = tile / p.n_tiles;    // (row tiles in front of it, in whole groups)
    int a = 0, b = p.experts;           // the group with first[e] <= rt < first[e + 1]
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (t.first[m] <= rt) a = m; else b = m;
    }
    e = a;
    lo = t.start[e];
    hi = t.start[e + 1];
    mt = t.first[e + 1] - t.first[e];
    tile -= t.first[e] * p.n_tiles;
  }
  const int band = tile / (kBandTiles * p.n_tiles);
  const int in_band = tile - band * kBandTiles * p.n_tiles;
  const int width = min(kBandTiles, mt - band * kBandTiles);
  Fp8Tile r;
  r.expert = e;
  r.n = in_band / width;
  r.row0 = lo + (band * kBandTiles + in_band - r.n * width) * ROWS;
  r.rows = min(ROWS, hi - r.row0);
  return r;
}

__device__ __forceinline__ uint32_t pack_out(float a, float b, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint16_t round_out(float a, bool bf16) {
  if (bf16) return __bfloat16_as_ushort(__float2bfloat16_rn(a));
  return __half_as_ushort(__float2half_rn(a));
}
// 32 bytes at once, 32-byte aligned: a whole sector.  (A warp's lanes write rows of their own, so a store touches 32 lines whatever its
// width; in 16-byte pieces the 64 KiB of a 128 x 256 tile took 6900 cycles.)
__device__ __forceinline__ void st_global_v8(void* dst, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
               "r"(w[6]), "r"(w[7])
               : "memory");
}
// 16 neighbouring results of a row, of which those in front of `left` exist.  bytes: what the row's pieces of 16 start on, 32, 16 or less.
template <class Value>
__device__ __forceinline__ void store_row16(uint16_t* dst, int left, int bytes, bool bf16, Value&& value) {
  if (bytes >= 16 && left >= 16) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = pack_out(value(2 * j), value(2 * j + 1), bf16);
    if (bytes == 32) {
      st_global_v8(dst, w);
    } else {
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(dst + 8) = make_uint4(w[4], w[5], w[6], w[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < left) dst[j] = round_out(value(j), bf16);
  }
}
// The same in fp32; rows and pieces start on 64 bytes.
template <class Value>
__device__ __forceinline__ void store_row16_f32(float* dst, int left, Value&& value) {
  if (left >= 16) {
#pragma unroll
    for (int h = 0; h < 16; h += 8) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(value(h + j));
      st_global_v8(dst + h, w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < left) dst[j] = value(j);
  }
}
// 128 columns of a warp's 32 rows, one a lane, whose pieces start on 2 bytes only (an odd pitch).  As they lie, 16-bit stores would touch 32 lines
// each; so the warp turns 16 columns at a time round in its corner of shared memory (kTurnBytes) and a store covers a piece of two rows.
// dst: the first row; `rows` and `left`: rows and columns that exist.
constexpr int kTurnPitch = 36, kTurnBytes = 32 * kTurnPitch;
template <class Value>
__device__ __forceinline__ void store_rows_turned(uint16_t* dst, long long ld, int rows, int left, uint8_t* corner, int lane, bool bf16, Value&& value) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    if (16 * c >= left) break;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<uint32_t*>(corner + lane * kTurnPitch + 4 * j) = pack_out(value(16 * c + 2 * j), value(16 * c + 2 * j + 1), bf16);
    __syncwarp();
    const int col = lane & 15;
    if (16 * c + col < left) {
#pragma unroll 4
      for (int r = lane >> 4; r < rows; r += 2)
        dst[r * ld + 16 * c + col] = *reinterpret_cast<const uint16_t*>(corner + r * kTurnPitch + 2 * col);
    }
  }
}
// 32 neighbouring codes of a row (rows start on 32 bytes), values times inv.
template <class Value>
__device__ __forceinline__ void store_codes32(uint8_t* dst, int left, float inv, bool bad, Value&& value) {
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    w[j] = bad ? 0x7f7f7f7fu : e4m3x2(value(4 * j) * inv, value(4 * j + 1) * inv) | (e4m3x2(value(4 * j + 2) * inv, value(4 * j + 3) * inv) << 16);
  if (left >= 32) {
    st_global_v8(dst, w);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < left) dst[j] = static_cast<uint8_t>(w[j >> 2] >> (8 * (j & 3)));
  }
}

// Named barrier of some warps that also tells whether `ok` holds in all of their threads.
__device__ __forceinline__ bool named_barrier_all(int id, int nthreads, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "bar.red.and.pred q, %1, %2, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(nthreads), "r"(static_cast<uint32_t>(ok))
      : "memory");
  return r != 0;
}

// SiLU(g) * u in fp32 with the library's exponential and an IEEE division.
__device__ __forceinline__ float silu_times(float g, float u) { return g / (1.f + expf(-g)) * u; }

}  // namespace sk
