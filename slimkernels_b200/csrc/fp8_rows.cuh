// Row kernels around the FP8 products: the quantiser of activations (in place or into the rows of an expert's group), the weight
// preparation, the router, and the weighted sum of the experts' results.  All are passes over their data that HBM (large calls) or
// the launch (small ones) bounds.
#pragma once
#include "fp8_common.cuh"

namespace sk {

// Elements of an activation or weight tensor: 0 fp16, 1 bf16, 2 fp32.
template <int TYPE>
__device__ __forceinline__ float load_element(const void* p, long long i) {
  if constexpr (TYPE == 2) return ld_global_f32(static_cast<const float*>(p) + i);
  unsigned short v;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(static_cast<const uint16_t*>(p) + i) : "memory");
  if constexpr (TYPE == 1) return __uint_as_float(static_cast<uint32_t>(v) << 16);
  return __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ uint4 ld_global_v4(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
// Eight consecutive elements, 16-byte aligned.
template <int TYPE>
__device__ __forceinline__ void load_eight(const void* p, long long i, float (&f)[8]) {
  if constexpr (TYPE == 2) {
    const uint4 a = ld_global_v4(static_cast<const float*>(p) + i), b = ld_global_v4(static_cast<const float*>(p) + i + 4);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
  } else {
    const uint4 a = ld_global_v4(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (TYPE == 1) {
        f[2 * j] = __uint_as_float(w[j] << 16);
        f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        f[2 * j] = v.x;
        f[2 * j + 1] = v.y;
      }
    }
  }
}

// Eight of a block's 128 values in each of 16 neighbouring lanes -> their codes, the block's exponent and whether it holds a value that is not
// finite (then the codes are NaN).
__device__ __forceinline__ uint2 quantise_eight(const float (&f)[8], int* exponent, bool* not_finite) {
  uint32_t a = 0;                                   // bits of |x|: ordered like the values, infinity and NaN above all
#pragma unroll
  for (int j = 0; j < 8; ++j) a = max(a, __float_as_uint(f[j]) & 0x7fffffffu);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  const bool bad = not_finite_bits(a);
  const int e = bad ? 0 : fp8_block_exponent(a);
  const float inv = pow2f(-e);
  uint2 code;
  code.x = e4m3x2(f[0] * inv, f[1] * inv) | (e4m3x2(f[2] * inv, f[3] * inv) << 16);
  code.y = e4m3x2(f[4] * inv, f[5] * inv) | (e4m3x2(f[6] * inv, f[7] * inv) << 16);
  if (bad) code = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
  *exponent = e;
  *not_finite = bad;
  return code;
}

// x [M, K] -> codes [M, ld_q] and scales, one per row and block of 128 (the rule is fp8_block_exponent's; a block with a value that
// is not finite has a NaN scale and NaN codes).  Blocks do not depend on one another: 16 lanes hold one, eight elements each.
// rows != nullptr: row t is written to the rows rows[t * choices .. t * choices + choices - 1] of the result instead, which orders tokens by expert
// on the way.  Places outside [0, places) are nobody's.
template <int TYPE, bool E8M0, bool VECTOR>
__global__ void __launch_bounds__(256)
fp8_quantize_kernel(const void* x, long long ld_x, long long M, int K, uint8_t* q, long long ld_q, void* scale, long long s_row,
                    long long s_blk, const int* rows, int choices, int places) {
  // The next kernel may start only when every CTA of this one has passed the wait: what it then reads early (weights, offsets) was
  // complete before this kernel's inputs were.  So the trigger has to stay behind the wait (the products' stand in front of theirs).
  grid_dep_wait();
  grid_dep_launch_dependents();
  // A CTA takes 16 neighbouring blocks (blockIdx.y) of every gridDim.x-th row, two rows a turn; a row's destinations come with its values, one
  // per lane.
  const int l16 = threadIdx.x & 15, b = blockIdx.y * 16 + (threadIdx.x >> 4), k0 = b * kFp8Block + l16 * 8;
  const bool mine = k0 - l16 * 8 < K;               // (past the row's last block: only along for the shuffles)
  struct Row {
    long long m;
    int place;
    float f[8];
  };
  const auto load = [&](long long m) {
    Row u;
    u.m = m < M && mine ? m : -1;
    u.place = rows != nullptr && u.m >= 0 && l16 < choices ? ld_global_int(rows + m * choices + l16) : -1;
    if (VECTOR && u.m >= 0 && k0 + 8 <= K) {
      load_eight<TYPE>(x, m * ld_x + k0, u.f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) u.f[j] = u.m >= 0 && k0 + j < K ? load_element<TYPE>(x, m * ld_x + k0 + j) : 0.f;
    }
    return u;
  };
  const auto store = [&](const Row& u) {
    int e;
    bool bad;
    const uint2 code = quantise_eight(u.f, &e, &bad);
    for (int c = 0; c < choices; ++c) {
      long long r = u.m;
      if (rows != nullptr) {
        r = __shfl_sync(0xffffffffu, u.place, c & 15, 16);
        if (c >= 16) r = u.m >= 0 ? ld_global_int(rows + u.m * choices + c) : -1;
      }
      if (r < 0 || (rows != nullptr && r >= places)) continue;
      uint8_t* dst = q + r * ld_q + k0;
      if (k0 + 8 <= K) {                            // (ld_q is a multiple of 16)
        *reinterpret_cast<uint2*>(dst) = code;
      } else {
        const uint32_t w[2] = {code.x, code.y};
        for (int j = 0; j < 8 && k0 + j < K; ++j) dst[j] = static_cast<uint8_t>(w[j >> 2] >> (8 * (j & 3)));
      }
      if (l16 == 0) store_scale<E8M0>(scale, r * s_row + b * s_blk, e, bad);
    }
  };
  for (long long m = blockIdx.x; m < M; m += 2 * gridDim.x) {
    const Row u0 = load(m), u1 = load(m + gridDim.x);
    store(u0);
    store(u1);
  }
}

// w [rows, K] -> codes and one scale per 128 x 128 block; a CTA takes one block.  blockIdx.y counts matrices of w_rows rows whose
// blocks start anew.
template <int TYPE, bool E8M0>
__global__ void __launch_bounds__(256)
fp8_prepare_weight_kernel(const void* w, long long ld_w, long long matrix, int N, int K, uint8_t* q, long long ld_q, long long q_matrix,
                          void* scale) {
  __shared__ uint32_t red[8];
  const int kb = (K + kFp8Block - 1) / kFp8Block, nb = (N + kFp8Block - 1) / kFp8Block;
  const int b = blockIdx.x % kb, r = blockIdx.x / kb;
  const long long in = blockIdx.y * matrix, out = blockIdx.y * q_matrix;
  const int col = b * kFp8Block + (threadIdx.x & 31) * 4, row0 = r * kFp8Block + (threadIdx.x >> 5);
  float f[16][4];
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = row0 + 8 * i, k = col + j;
      f[i][j] = n < N && k < K ? load_element<TYPE>(w, in + n * ld_w + k) : 0.f;
      a = max(a, __float_as_uint(f[i][j]) & 0x7fffffffu);
    }
  a = __reduce_max_sync(0xffffffffu, a);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, red[i]);
  const bool bad = not_finite_bits(a);
  const int e = bad ? 0 : fp8_block_exponent(a);
  const float inv = pow2f(-e);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int n = row0 + 8 * i;
    if (n >= N || col >= K) continue;
    uint32_t code = e4m3x2(f[i][0] * inv, f[i][1] * inv) | (e4m3x2(f[i][2] * inv, f[i][3] * inv) << 16);
    if (bad) code = 0x7f7f7f7fu;
    uint8_t* dst = q + out + n * ld_q + col;
    if (col + 4 <= K) {                             // (ld_q is a multiple of 16)
      *reinterpret_cast<uint32_t*>(dst) = code;
    } else {
      for (int j = 0; j < 4 && col + j < K; ++j) dst[j] = static_cast<uint8_t>(code >> (8 * j));
    }
  }
  if (threadIdx.x == 0) store_scale<E8M0>(scale, (static_cast<long long>(blockIdx.y) * nb + r) * kb + b, e, bad);
}

// out[t, :] = round( sum over j of weights[t, j] * y[rows[t, j], :] ), in the order of j; choices with rows outside [0, T * choices) count nothing.
// y is fp32, as the second product leaves it: the result is rounded once, and an expert's result past fp16's range is no infinity in a sum
// within it.  HBM bounds the pass: 16384 rows of 4096 to 4096 tokens 53 us (300 MB, 5.7 TB/s).
template <bool BF16, bool VECTOR>
__global__ void __launch_bounds__(256)
fp8_combine_kernel(const float* y, long long ld_y, const int* rows, const float* weights, int choices, int T, int H, uint16_t* out,
                   long long ld_out) {
  grid_dep_wait();
  grid_dep_launch_dependents();
  constexpr int kPer = VECTOR ? 8 : 1;
  const int per_row = (H + kPer - 1) / kPer;
  const long long total = static_cast<long long>(T) * per_row;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long t = i / per_row;
    const int h = static_cast<int>(i - t * per_row) * kPer;
    float acc[8] = {};
    for (int j = 0; j < choices; ++j) {
      const int r = ld_global_int(rows + t * choices + j);
      if (r < 0 || r >= T * choices) continue;
      const float w = ld_global_f32(weights + t * choices + j);
      if constexpr (VECTOR) {
        float f[8];
        load_eight<2>(y, r * ld_y + h, f);
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = fmaf(w, f[c], acc[c]);
      } else {
        acc[0] = fmaf(w, load_element<2>(y, r * ld_y + h), acc[0]);
      }
    }
    uint16_t* dst = out + t * ld_out + h;
    if constexpr (VECTOR) {
      uint4 v;
      v.x = pack_out(acc[0], acc[1], BF16);
      v.y = pack_out(acc[2], acc[3], BF16);
      v.z = pack_out(acc[4], acc[5], BF16);
      v.w = pack_out(acc[6], acc[7], BF16);
      *reinterpret_cast<uint4*>(dst) = v;
    } else {
      *dst = round_out(acc[0], BF16);
    }
  }
}

// ---------------------------------------------------------------- router
// A CTA takes a run of tokens, a warp a run of those; everything is in the order of the choices t * k + j, so the places are those
// of a stable sort by expert and the same in every run.
//   pass 1  (TOPK: the k largest logits of each token and their weights,) how many choices each expert got from this CTA, and the place of each
//           choice among these
//   pass 2  (after pass 1 of all CTAs) the experts' first rows, added to the places
// With one CTA both are one launch.  Issue slots and latency bound all of it (8192 tokens of 256 logits are 4 MB): 32 warps to a CTA, a token's
// logits loaded while the one before it is worked on, as few instructions per choice as can be.
constexpr int kRouteWarps = 32;
struct RouteParams {
  const void* logits;                   // [T, ld]
  long long ld;
  int T, E, k, renormalize;
  int* ids;                             // [T, k] written by pass 1, or the caller's
  float* weights;                       // [T, k]
  int* rows;                            // [T, k]
  int* offsets;                         // [E + 1]
  int* counts;                          // [CTAs][E]
  int per_cta;                          // tokens
};

// Bits that order like the logits: larger is larger, NaN above all (as a maximum that propagates it has it).
__device__ __forceinline__ uint32_t ordered_bits(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);      // (-0 and 0 are one value)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered_bits(uint32_t o) {
  if (o == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// One token: lane holds the logits of experts lane, lane + 32, ...; the choice of a round is the largest left, the lowest expert among equals.
// A logit of 16 bits and its expert fit one word, so that a round is one reduction and no two words are equal:
//   bits that order like the logits | 0xffff - expert
// A lane sorts its words first; the lane that held a round's largest moves on to its next.  (Looking through its words again instead: 12.1
// against 9.7 us for 64 tokens of 256 experts.)
// 32-bit logits take a second reduction where several lanes hold the largest.  The lane that held it looks through its logits again, as it does among
// more than 512 experts.
template <int TYPE, int PER>
struct TokenLogits {
  static constexpr bool kWord = TYPE != 2;
  static constexpr bool kSorted = kWord && PER <= 16;         // (32 words take more registers than a thread has)
  uint32_t key[PER];                    // 0: none (below -infinity's)

  static __device__ __forceinline__ uint32_t order16(uint32_t b) {
    const bool nan = TYPE == 1 ? (b & 0x7fffu) > 0x7f80u : (b & 0x7fffu) > 0x7c00u;
    if (nan) return 0xffffu;
    if (b == 0x8000u) b = 0;
    return b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
  }
  // Batcher's odd-even merge sort, the largest first.
  __device__ __forceinline__ void sort() {
#pragma unroll
    for (int p = 1; p < PER; p *= 2)
#pragma unroll
      for (int d = p; d >= 1; d /= 2)
#pragma unroll
        for (int j = d % p; j + d < PER; j += 2 * d)
#pragma unroll
          for (int i = 0; i < d; ++i)
            if (i + j + d < PER && (i + j) / (2 * p) == (i + j + d) / (2 * p)) {
              const uint32_t a = key[i + j], b = key[i + j + d];
              key[i + j] = max(a, b);
              key[i + j + d] = min(a, b);
            }
  }
  static __device__ __forceinline__ float value16(uint32_t o) {
    if (o == 0xffffu) return __uint_as_float(0x7fc00000u);
    const uint32_t b = o & 0x8000u ? o & 0x7fffu : ~o & 0xffffu;
    if constexpr (TYPE == 1) return __uint_as_float(b << 16);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
  }
  static __device__ __forceinline__ float value(uint32_t k) { return kWord ? value16(k >> 16) : from_ordered_bits(k); }
  static __device__ __forceinline__ bool masked(uint32_t k) {   // -infinity
    return kWord ? (k >> 16) == (TYPE == 1 ? 0x007fu : 0x03ffu) : k == 0x007fffffu;
  }

  __device__ __forceinline__ void load(const RouteParams& p, long long t, int lane) {   // as they lie in memory, so that nothing waits yet
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      key[i] = 0;
      if (lane + 32 * i >= p.E) continue;
      if constexpr (kWord) {
        unsigned short v;
        asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(static_cast<const uint16_t*>(p.logits) + t * p.ld + lane + 32 * i) : "memory");
        key[i] = v;
      } else {
        key[i] = __float_as_uint(ld_global_f32(static_cast<const float*>(p.logits) + t * p.ld + lane + 32 * i));
      }
    }
  }
  __device__ __forceinline__ void order(const RouteParams& p, int lane) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 32 * i;
      if (e >= p.E) key[i] = 0;
      else if constexpr (kWord) key[i] = order16(key[i]) << 16 | (0xffffu - e);
      else key[i] = ordered_bits(__uint_as_float(key[i]));
    }
  }

  __device__ __forceinline__ void choose(const RouteParams& p, long long t, int lane) {
    order(p, lane);
    uint32_t first, mine = 0;                         // the largest of all, and (lane j) choice j
    int my_id = 0;
    float sum = 0.f;
    const auto total = [&](uint32_t largest) {        // of the whole softmax, while all keys are there
      const float top = value(largest);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < p.E) sum += expf(value(key[i]) - top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    };
    if constexpr (kSorted) {
      if (!p.renormalize) {
        uint32_t most = key[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) most = max(most, key[i]);
        total(__reduce_max_sync(0xffffffffu, most));
      }
      sort();
      first = 0;
      for (int j = 0; j < p.k; ++j) {
        const uint32_t winner = __reduce_max_sync(0xffffffffu, key[0]);
        if (key[0] == winner) {
#pragma unroll
          for (int i = 0; i < PER; ++i) key[i] = i + 1 < PER ? key[i + 1] : 0;
        }
        if (j == 0) first = winner;
        if (lane == j) mine = winner;
      }
      my_id = static_cast<int>(0xffffu - (mine & 0xffffu));
    } else {
      uint32_t best = 0;
      int at = 0;
      auto look = [&]() {               // the lane's own largest; 0: none left
        best = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if constexpr (kWord) best = max(best, key[i]);
          else if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
        }
      };
      look();
      first = 0;
      for (int j = 0; j < p.k; ++j) {
        const uint32_t winner = __reduce_max_sync(0xffffffffu, best);
        int e;
        if constexpr (kWord) {
          e = static_cast<int>(0xffffu - (winner & 0xffffu));
        } else {
          const uint32_t holders = __ballot_sync(0xffffffffu, best == winner);
          e = __shfl_sync(0xffffffffu, at, __ffs(holders) - 1);
          if (holders & (holders - 1)) e = static_cast<int>(__reduce_min_sync(0xffffffffu, best == winner ? static_cast<uint32_t>(at) : 0x7fffffffu));
        }
        if (j == 0) {
          first = winner;
          if (!p.renormalize) total(winner);
        }
        if ((e & 31) == lane) {
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (kWord ? key[i] == winner : lane + 32 * i == e) key[i] = 0;
          look();
        }
        if (lane == j) { mine = winner; my_id = e; }
      }
    }
    // lane j holds choice j: its weight, and the sum of all in the order of the choices
    const float w = expf(value(mine) - value(first));
    if (p.renormalize)
      for (int j = 0; j < p.k; ++j) sum += __shfl_sync(0xffffffffu, w, j);
    if (lane < p.k) {
      p.ids[t * p.k + lane] = my_id;
      // a token whose logits are all -infinity has no distribution: its weights are zero
      p.weights[t * p.k + lane] = masked(first) ? 0.f : w / sum;
    }
  }
};

struct RouteRange { long long t0, t1; };   // tokens of this warp
__device__ __forceinline__ RouteRange route_range(const RouteParams& p) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
  const long long c0 = static_cast<long long>(blockIdx.x) * p.per_cta, c1 = min(static_cast<long long>(p.T), c0 + p.per_cta);
  const int per_warp = (p.per_cta + warps - 1) / warps;
  RouteRange r;
  r.t0 = min(c1, c0 + static_cast<long long>(warp) * per_warp);
  r.t1 = min(c1, r.t0 + per_warp);
  return r;
}

// hist [warps][E]: how many choices each expert got from each warp.
template <int TYPE, int PER, bool TOPK>
__device__ __forceinline__ void route_count(const RouteParams& p, int* hist) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const RouteRange r = route_range(p);
  if constexpr (TOPK) {
    TokenLogits<TYPE, PER> now, next;
    if (r.t0 < r.t1) now.load(p, r.t0, lane);
    for (int i = threadIdx.x; i < warps * p.E; i += blockDim.x) hist[i] = 0;
    for (long long t = r.t0; t < r.t1; ++t) {
      if (PER <= 16 && t + 1 < r.t1) next.load(p, t + 1, lane);
      now.choose(p, t, lane);
      if (PER <= 16) now = next;
      else if (t + 1 < r.t1) now.load(p, t + 1, lane);      // (no registers for two tokens' logits)
    }
    __syncwarp();
  } else {
    for (int i = threadIdx.x; i < warps * p.E; i += blockDim.x) hist[i] = 0;
  }
  __syncthreads();
  for (long long i = r.t0 * p.k + lane; i < r.t1 * p.k; i += 32) {
    const int e = p.ids[i];
    if (e >= 0 && e < p.E) atomicAdd(hist + warp * p.E + e, 1);      // (integers: the order does not show)
  }
  __syncthreads();
}

// hist: on entry the warps' counts, on return each warp's next place for every expert.  base: the experts' first places of this CTA.
__device__ __forceinline__ void route_place(const RouteParams& p, int* hist, const int* base) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int at = base[e];
    for (int w0 = 0; w0 < warps; w0 += 8) {         // (eight loads at once: one after another they are a chain of round trips)
      int n[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) n[i] = w0 + i < warps ? hist[(w0 + i) * p.E + e] : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (w0 + i < warps) hist[(w0 + i) * p.E + e] = at;
        at += n[i];
      }
    }
  }
  __syncthreads();
  const RouteRange r = route_range(p);
  int* next = hist + warp * p.E;
  for (long long i0 = r.t0 * p.k; i0 < r.t1 * p.k; i0 += 32) {
    const long long i = i0 + lane;
    const int e = i < r.t1 * p.k ? p.ids[i] : -1;
    const bool on = e >= 0 && e < p.E;
    const uint32_t same = __match_any_sync(0xffffffffu, on ? e : -1);
    const int before = __popc(same & ((1u << lane) - 1u));
    const int at = on ? next[e] + before : -1;
    __syncwarp();
    if (on && before == 0) next[e] += __popc(same);
    __syncwarp();
    if (i < r.t1 * p.k) p.rows[i] = at;
  }
}

// Exclusive sums over the experts of total[] (in place -> first places); the grand total is stored behind them.  A warp scans 32 experts, then
// adds what lies in front of them (at most 32 such sums).
__device__ __forceinline__ int warp_scan(int n, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, n, o);
    if (lane >= o) n += up;
  }
  return n;
}
__device__ __forceinline__ void scan_experts(int* total, int E) {
  __shared__ int ahead[32];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, parts = (E + 31) >> 5;
  for (int g = warp; g < parts; g += warps) {
    const int e = 32 * g + lane, n = e < E ? total[e] : 0, incl = warp_scan(n, lane);
    if (e < E) total[e] = incl - n;
    if (lane == 31) ahead[g] = incl;
  }
  __syncthreads();
  const int part = lane < parts ? ahead[lane] : 0, sums = warp_scan(part, lane);
  for (int g = warp; g < parts; g += warps) {
    const int before = __shfl_sync(0xffffffffu, sums - part, g);
    if (32 * g + lane < E) total[32 * g + lane] += before;
  }
  if (threadIdx.x == 31) total[E] = sums;
  __syncthreads();
}

// Shared memory of pass 1: [warps][E] counts, [E + 1] first places.
__host__ __device__ constexpr int route_smem_bytes(int warps, int E) { return (warps * E + E + 1) * 4; }
static_assert(route_smem_bytes(kRouteWarps, kFp8MaxExperts) + 128 <= 232448, "shared memory of a CTA (128 bytes are scan_experts')");

template <int TYPE, int PER, bool TOPK, bool ONE_CTA>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_count_kernel(const RouteParams p) {
  extern __shared__ int route_smem[];
  const int warps = blockDim.x >> 5;
  int* hist = route_smem;
  int* total = hist + warps * p.E;
  grid_dep_wait();
  grid_dep_launch_dependents();
  route_count<TYPE, PER, TOPK>(p, hist);
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int n = 0;
    for (int w = 0; w < warps; ++w) n += hist[w * p.E + e];
    if constexpr (!ONE_CTA) p.counts[static_cast<long long>(blockIdx.x) * p.E + e] = n;
    total[e] = ONE_CTA ? n : 0;
  }
  __syncthreads();
  if constexpr (ONE_CTA) {
    scan_experts(total, p.E);
    for (int e = threadIdx.x; e <= p.E; e += blockDim.x) p.offsets[e] = total[e];
  }
  route_place(p, hist, total);
}

// Adds the experts' first places, and what the CTAs in front chose, to the places.
__global__ void __launch_bounds__(1024)
route_shift_kernel(const RouteParams p) {
  extern __shared__ int route_smem[];
  int* total = route_smem;              // [E + 1]
  int* base = total + p.E + 1;          // [E]
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) total[e] = base[e] = 0;
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch_dependents();
  const long long c0 = static_cast<long long>(blockIdx.x) * p.per_cta, c1 = min(static_cast<long long>(p.T), c0 + p.per_cta);
  const long long i0 = c0 * p.k + threadIdx.x;      // (a thread's first place is on its way with the counts)
  const bool on = i0 < c1 * p.k;
  const int at0 = on ? ld_global_int(p.rows + i0) : -1, e0 = on ? ld_global_int(p.ids + i0) : 0;
  // the counts of all CTAs, and of those in front of this one: as many threads per expert as there are
  const int share = max(1, static_cast<int>(blockDim.x) / p.E), ctas = static_cast<int>(gridDim.x);
  for (int i = threadIdx.x; i < share * p.E; i += blockDim.x) {
    const int e = i % p.E, part = i / p.E;
    int before = 0, all = 0;
#pragma unroll 16
    for (int c = part; c < ctas; c += share) {
      const int n = p.counts[static_cast<long long>(c) * p.E + e];
      before += c < static_cast<int>(blockIdx.x) ? n : 0;
      all += n;
    }
    atomicAdd(total + e, all);
    atomicAdd(base + e, before);
  }
  __syncthreads();
  scan_experts(total, p.E);
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) base[e] += total[e];
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= p.E; e += blockDim.x) p.offsets[e] = total[e];
  __syncthreads();
  if (at0 >= 0) p.rows[i0] = at0 + base[e0];
  for (long long i = i0 + blockDim.x; i < c1 * p.k; i += blockDim.x) {
    const int at = p.rows[i];
    if (at >= 0) p.rows[i] = at + base[p.ids[i]];
  }
}

}  // namespace sk
