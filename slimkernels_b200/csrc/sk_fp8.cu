// Launchers of the FP8 products, the router and the expert layers (C ABI: include/sk_fp8.h).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "../../include/sk_fp8.h"
#include "fp8_common.cuh"
#include "fp8_narrow.cuh"
#include "fp8_rows.cuh"
#include "fp8_scaled.cuh"
#include "fp8_scaled_narrow.cuh"
#include "fp8_wide.cuh"

namespace sk {

__device__ int g_fp8_status;            // the first wait that ran into its limit on this device, 0: none

namespace {

std::atomic<int64_t> g_options[6];

int cuda_status(cudaError_t e) {
  if (e == cudaSuccess) return SK_OK;
  (void)cudaGetLastError();
  return e == cudaErrorMemoryAllocation ? SK_ERR_OUT_OF_MEMORY : SK_ERR_CUDA;
}

struct DeviceInfo {
  int index = 0;
  int sms = 0;
  int* status = nullptr;
};
// What a launch needs to know of the current device.
int device_info(DeviceInfo* out) {
  constexpr int kMax = 64;
  static std::atomic<int> sms[kMax];
  static std::atomic<int*> words[kMax];
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return cuda_status(e);
  if (dev < 0 || dev >= kMax) return SK_ERR_UNAVAILABLE;
  if (sms[dev].load() == 0) {
    // (a first call under stream capture: looking the status word up may load the module, which a capture in global mode refuses)
    struct Relaxed {
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      Relaxed() { (void)cudaThreadExchangeStreamCaptureMode(&mode); }
      ~Relaxed() { (void)cudaThreadExchangeStreamCaptureMode(&mode); }
    } relaxed;
    int major = 0, n = 0;
    if (cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev); e != cudaSuccess) return cuda_status(e);
    if (major != 10) return SK_ERR_UNSUPPORTED_ARCH;
    if (cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev); e != cudaSuccess) return cuda_status(e);
    void* word = nullptr;
    if (cudaError_t e = cudaGetSymbolAddress(&word, g_fp8_status); e != cudaSuccess) return cuda_status(e);
    words[dev].store(static_cast<int*>(word));
    sms[dev].store(n);
  }
  out->index = dev;
  out->sms = sms[dev].load();
  out->status = words[dev].load();
  return SK_OK;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// Codes [rows, K] in boxes of 128 bytes x box_rows, 128-byte swizzle, zeros outside.
int codes_map(const void* q, int64_t rows, int64_t K, int64_t ld, int box_rows, CUtensorMap* out) {
  EncodeFn enc = encode_fn();
  if (!enc) return SK_ERR_CUDA;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  const cuuint32_t box[2] = {128u, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t unit[2] = {1u, 1u};
  return enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(q), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? SK_OK
             : SK_ERR_CUDA;
}

constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }
constexpr int64_t kIntMax = 0x7fffffff;
constexpr int kOutF32 = -1;             // beside sk_out_dtype: the expert layers' second product, whose results a weighted sum follows
bool aligned(const void* p, int64_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool aligned4(std::initializer_list<const void*> ps) {
  return std::all_of(ps.begin(), ps.end(), [](const void* p) { return aligned(p, 4); });
}
bool is_scale_type(int t) { return t == SK_SCALE_F32 || t == SK_SCALE_E8M0; }
bool is_float_type(int t) { return t >= SK_FLOAT_F16 && t <= SK_FLOAT_F32; }
bool is_out_type(int t) { return t == SK_OUT_F16 || t == SK_OUT_BF16; }
int64_t scale_bytes(int scale_type) { return scale_type == SK_SCALE_E8M0 ? 1 : 4; }

// dependent: programmatic dependent launch.  Every kernel here but the weight preparation waits (griddepcontrol.wait) before it reads what a
// kernel still in flight may write, and before it writes anything, so its set-up may run under the tail of whatever is in front of it; that saves 1 to 2
// us a launch between this library's kernels, which let their followers start early.  Products of a call with the quantiser in front of them
// (early_weights) read weights and offsets before their wait.  That is sound only because fp8_quantize_kernel lets its followers start AFTER its own
// wait: see product().  (A follower may hold tensor memory while it waits.  It cannot take any that the
// kernel in front still needs: every kernel here takes at most half of an SM's columns with half of its shared memory, or all with most of it.)
struct LaunchConfig {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  LaunchConfig(int64_t grid_x, int64_t grid_y, int threads, int64_t smem, bool dependent, int cluster, cudaStream_t stream) {
    cfg.gridDim = dim3(static_cast<unsigned>(grid_x), static_cast<unsigned>(grid_y), 1);
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 0;
    if (dependent) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
      ++cfg.numAttrs;
    }
  }
};

// Lets a kernel have so much shared memory: once per kernel and device (`done` belongs to the kernel).
template <class Kernel>
int allow_shared(Kernel kern, int bytes, const DeviceInfo& dev, std::atomic<uint64_t>& done) {
  const uint64_t bit = uint64_t(1) << dev.index;
  if (done.load(std::memory_order_acquire) & bit) return SK_OK;
  if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); e != cudaSuccess) return cuda_status(e);
  done.fetch_or(bit, std::memory_order_release);
  return SK_OK;
}

// Calls fn(std::integral_constant...) for a runtime value.
template <class F>
int with_bool(bool b, F&& fn) {
  return b ? fn(std::true_type{}) : fn(std::false_type{});
}
template <class F>
int with_type(int t, F&& fn) {
  switch (t) {
    case 0: return fn(std::integral_constant<int, 0>{});
    case 1: return fn(std::integral_constant<int, 1>{});
    default: return fn(std::integral_constant<int, 2>{});
  }
}

// ---------------------------------------------------------------- products
constexpr int kSmShared = 233472, kCtaShared = 232448;      // shared memory of an SM (1 KiB per CTA goes to the system) and of a CTA
constexpr int shared_for(int ctas) { return ctas == 1 ? kCtaShared : kSmShared / ctas - 1024; }      // what a CTA may have with so many to an SM

// How many clusters of 2, 4 or 8 CTAs, one or two CTAs to an SM, run at once.  A cluster lies within one GPC, so fewer fit than there is room for
// single CTAs: on B200's 148 SMs 33 of four and 15 of eight, with two CTAs to an SM 71 and 33.  Asked for a kernel of its own, which is never launched:
// of a kernel that takes tensor memory the occupancy calculator only counts one CTA to an SM, though two run (72 clusters of four are slower than 71 by a third).
__global__ void cluster_room_kernel() {}
int clusters_at_once(const DeviceInfo& dev, int size, int per_sm) {
  static std::atomic<int> known[64][2][4];
  std::atomic<int>& slot = known[dev.index][per_sm - 1][size == 2 ? 1 : size == 4 ? 2 : 3];
  int n = slot.load();
  if (n == 0) {
    static std::atomic<uint64_t> done;
    LaunchConfig lc(size, 1, 256, shared_for(per_sm), false, size, nullptr);
    if (allow_shared(cluster_room_kernel, kCtaShared, dev, done) != SK_OK ||
        cudaOccupancyMaxActiveClusters(&n, cluster_room_kernel, &lc.cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    slot.store(n);
  }
  return n;
}

struct Choice {
  int kernel;                           // sk_fp8_kernel
  int row_tile, feature_tile, split;
  int64_t ctas;
};

// What a product, or the products of the groups, are launched as.  Measured on B200 (us; few rows: features on the tensor memory's lanes in tiles
// of 16 or 32 rows, many: rows on the lanes, 128 a CTA or 256 a pair of CTAs).
//   One group, 8-bit scales, tile of 32 / many / pair:
//     K 4096:  64 x 12288  14.2 / 17.1 / 15.4     128 x 12288  21.3 / 17.8 / 16.2     256 x 4096  12.6 / 14.3 / 14.8     512 x 4096  20.7 / 14.7 / 15.2
//     K 8192:  64 x 8192   18.4 / 29.8 / 23.9     128 x 8192   21.9 / 30.9 / 25.1     256 x 8192  37.6 / 30.7 / 25.2
//   so few rows' kernel takes what its tiles of 32 rows hold with two CTAs to an SM, and a stream of weights (up to 32 rows) always; the pair the rest.
//   One group, 32-bit scales, K 4096, tile of 16 / many:  32 x 12288  14.8 / 23.0   64 x 12288  22.4 / 21.8   128 x 4096  12.8 / 20.8   256 x 4096  22.5 / 20.8
//   By expert, 16 experts x 4096 x 2048, 8-bit scales, rows per expert (ragged) 2 / 8 / 16 / 32 / 64 / 256 / 1024:
//     tile 16  21.7 / 26.1 / 26.8 / 31.4 / 41.9     tile 32  22.5 / 25.8 / 25.9 / 29.2 / 34.4
//     many     27.1 / 26.3 / 26.5 / 27.1 / 27.7 / 49.9 / 135.6     pair  30.1 / 31.2 / 32.1 / 33.1 / 34.3 / 48.7 / 126.4
//   (64 experts x 2048 x 2048 at 16 and 32: tile 32  47.9, 50.3, many  50.2, 51.4).  A pair's tiles of 256 rows are emptier at a group's end, which costs
//   more than its faster MMAs give up to about 512 rows (16 experts' layers of 2048 x 1024, 512 rows each: many 129, pair 145; 1024 rows 238 and 235).
//   With 32-bit scales, 2 / 16 / 32 / 64:
//     tile 16  21.9 / 27.0 / 33.4 / 47.8     many  28.7 / 29.8 / 31.0 / 31.4
//   With the SiLU epilogue, whose time goes with the tile's rows, tiles of 16 are the fastest up to 32 rows per expert (67 us a block, tiles of 32 87, many 80).
// A tile's K range is split while that makes no more CTAs than SMs and leaves a CTA eight K blocks or so: 64 x 4096 x 4096 12.9 us in one, 10.9 in four; splitting
// where the tiles fill the SMs already loses (16 x 22016 x 4096 18.8 in one, 25.2 in two; 256 x 2048 x 4096, 8-bit scales, 11.1 and 11.7).
// Beyond that, to two CTAs an SM, it is split where all clusters run at once (16 x 9216 x 16384, 72 tiles: four 35.6, two 28.5; 71 tiles 28.3) and K is long (us, a
// quarter GB of weights in turn).  From one to two:
//   32-bit scales, one row tile:   80 feature tiles  K 4096 12.7 / 12.5  6144 17.0 / 14.7    112  4096 13.6 / 14.3  6144 18.7 / 17.9
//                                  144               4096 15.2 / 17.1  6144 21.4 / 22.1  8192 27.6 / 27.0
//     where weights are read again by other row tiles:   40 x 2  4096 12.1 / 10.2    72 x 2  4096 12.6 / 12.7  6144 16.8 / 15.0    18 x 8  4096 12.1 / 10.6
//   8-bit scales:   40 x 2  8192 18.1 / 17.5    56 x 2  8192 18.2 / 18.5    72 x 2  18.5 / 21.2    36 x 4  18.3 / 17.8    18 x 8  18.3 / 17.2
//                   one row tile   80  19.0 / 18.0    96  19.5 / 20.8    112  22.5 / 22.7    144  27.2 / 27.5
//   so the more feature tiles, that is the nearer to the stream of weights, the longer K has to be, and with 8-bit scales there are too many at two fifths of the SMs.
//   From two to four, 32-bit scales, K 8192:   56  15.2 / 14.2   70  16.4 / 16.8   28 x 2  14.0 / 11.3;   8-bit scales, K 16384:   56  23.8 / 22.0   70  28.3 / 27.0
//   14 x 4  20.1 / 16.5, but K 8192   56  14.2 / 14.2.
Choice choose(int64_t M, int64_t N, int64_t K, int64_t experts, bool grouped, bool silu, bool e8m0, const DeviceInfo& dev) {
  const int sms = dev.sms;
  Choice c;
  const int64_t rows = ceil_div(M, experts);       // of a group, on average
  const int64_t blocks = ceil_div(N, 128), kb = ceil_div(K, 128);
  bool few;
  if (grouped) {
    few = rows <= (e8m0 ? 32 : 16);
    c.row_tile = rows <= 8 ? 16 : 32;
  } else {
    const int tile = e8m0 ? 32 : 16;
    few = rows <= 32 || ceil_div(rows, tile) * blocks <= 2 * sms;
    c.row_tile = rows <= 16 ? 16 : 32;
  }
  c.kernel = few ? SK_FP8_KERNEL_FEW : !e8m0 || (grouped && rows <= 512) ? SK_FP8_KERNEL_MANY : SK_FP8_KERNEL_PAIR;
  if (const int64_t forced = g_options[SK_FP8_OPT_KERNEL].load()) c.kernel = static_cast<int>(!e8m0 && forced == SK_FP8_KERNEL_PAIR ? SK_FP8_KERNEL_MANY : forced);
  few = c.kernel == SK_FP8_KERNEL_FEW;
  if (few) {
    if (const int64_t forced = g_options[SK_FP8_OPT_ROW_TILE].load()) c.row_tile = static_cast<int>(forced);
    if (silu || !e8m0) c.row_tile = 16;
    c.feature_tile = 128;
  } else {
    c.row_tile = c.kernel == SK_FP8_KERNEL_PAIR ? 256 : 128;
    c.feature_tile = silu ? 128 : 256;
  }
  const int64_t tiles = (ceil_div(M, c.row_tile) + (grouped ? std::min(experts, M) : 0)) * ceil_div(N, c.feature_tile);
  c.split = 1;
  if (!grouped && few) {
    while (c.split < 8 && tiles * c.split * 2 <= sms && kb >= c.split * 8) c.split *= 2;
    const bool streams = e8m0 ? blocks * 5 > sms * 2 : kb * 5 < blocks * 2;
    while (c.split < 8 && tiles <= clusters_at_once(dev, c.split * 2, 2) && kb >= c.split * (e8m0 ? 64 : 32) && !(c.split == 1 && streams)) c.split *= 2;
    if (const int64_t forced = g_options[SK_FP8_OPT_SPLIT_K].load()) c.split = forced <= kb ? static_cast<int>(forced) : 1;
  }
  c.ctas = tiles * c.split;
  return c;
}

template <bool SILU>
int launch_narrow(const CUtensorMap& mw, const CUtensorMap& mx, const Fp8Params& p, int64_t tiles, const DeviceInfo& dev, cudaStream_t stream) {
  using T = Fp8NarrowTraits<SILU>;
  auto kern = fp8_narrow_kernel<SILU>;
  constexpr int kMost = T::dynamic_bytes(SILU ? 1 : 8, kFp8MaxExperts);
  static_assert(kMost <= 232448 && T::dynamic_bytes(SILU ? 1 : 8, 1) <= 115712, "shared memory of a CTA");
  static std::atomic<uint64_t> done;
  if (int rc = allow_shared(kern, kMost, dev, done); rc != SK_OK) return rc;
  const int64_t grid = p.split > 1 ? tiles * p.split : std::min<int64_t>(tiles, static_cast<int64_t>(dev.sms) * 2);
  LaunchConfig lc(grid, 1, T::kThreads, T::dynamic_bytes(p.split, p.experts), true, p.split, stream);
  return cuda_status(cudaLaunchKernelEx(&lc.cfg, kern, mw, mx, p));
}

template <bool SILU>
int launch_wide(const CUtensorMap& mw, const CUtensorMap& mx, const Fp8Params& p, int64_t tiles, const DeviceInfo& dev, cudaStream_t stream) {
  using T = Fp8WideTraits<SILU>;
  auto kern = fp8_wide_kernel<SILU>;
  static std::atomic<uint64_t> done;
  if (int rc = allow_shared(kern, T::dynamic_bytes(kFp8MaxExperts), dev, done); rc != SK_OK) return rc;
  LaunchConfig lc(std::min<int64_t>(tiles, dev.sms), 1, T::kThreads, T::dynamic_bytes(p.experts), true, 1, stream);
  return cuda_status(cudaLaunchKernelEx(&lc.cfg, kern, mw, mx, p));
}

// The ring: 3 to 12 stages, for two CTAs per SM where there are more CTAs than SMs and two fit, else for one.  The clusters of a split
// count as they fit: 16 of eight CTAs with an SM each ran one after 15 others (1 x 2048 x 4096 10.5 us, 5.8 with two CTAs to an SM), 36 of four after 33 (1 x 4608
// x 4096 13.3 and 7.7).
template <int TOK, bool SILU>
int launch_scaled_narrow(const CUtensorMap& mw, const CUtensorMap& mx, Fp8Params p, int64_t tiles, const DeviceInfo& dev, cudaStream_t stream) {
  using T = Fp8ScaledNarrowTraits<TOK, SILU>;
  auto kern = fp8_scaled_narrow_kernel<TOK, SILU>;
  const int fixed = T::fixed_bytes(p.split, p.experts);
  int ctas = (p.split > 1 ? tiles > clusters_at_once(dev, p.split, 1) : tiles > dev.sms) ? 2 : 1;
  if ((shared_for(ctas) - fixed) / T::kStageBytes < 3) ctas = 1;
  p.stages = std::min(T::kMaxStages, (shared_for(ctas) - fixed) / T::kStageBytes);
  static_assert((kCtaShared - T::fixed_bytes(SILU ? 1 : 8, 1)) / T::kStageBytes >= 3 && (kCtaShared - T::fixed_bytes(1, kFp8MaxExperts)) / T::kStageBytes >= 3,
                "room for a ring");
  static std::atomic<uint64_t> done;
  if (int rc = allow_shared(kern, kCtaShared, dev, done); rc != SK_OK) return rc;
  const int64_t grid = p.split > 1 ? tiles * p.split : std::min<int64_t>(tiles, static_cast<int64_t>(dev.sms) * ctas);
  LaunchConfig lc(grid, 1, T::kThreads, fixed + p.stages * T::kStageBytes, true, p.split, stream);
  return cuda_status(cudaLaunchKernelEx(&lc.cfg, kern, mw, mx, p));
}

template <int CTAS, bool SILU>
int launch_scaled(const CUtensorMap& mw, const CUtensorMap& mx, const Fp8Params& p, int64_t tiles, const DeviceInfo& dev, cudaStream_t stream) {
  using T = Fp8ScaledTraits<CTAS, SILU>;
  auto kern = fp8_scaled_kernel<CTAS, SILU>;
  static std::atomic<uint64_t> done;
  if (int rc = allow_shared(kern, T::dynamic_bytes(kFp8MaxExperts), dev, done); rc != SK_OK) return rc;
  LaunchConfig lc(std::min<int64_t>(tiles, dev.sms / CTAS) * CTAS, 1, T::kThreads, T::dynamic_bytes(p.experts), true, CTAS, stream);
  return cuda_status(cudaLaunchKernelEx(&lc.cfg, kern, mw, mx, p));
}

template <bool SILU>
int launch_product(const Choice& c, bool e8m0, const CUtensorMap& mw, const CUtensorMap& mx, const Fp8Params& p, int64_t tiles, const DeviceInfo& dev,
                   cudaStream_t stream) {
  if (!e8m0) {
    if (c.kernel == SK_FP8_KERNEL_MANY) return launch_wide<SILU>(mw, mx, p, tiles, dev, stream);
    return launch_narrow<SILU>(mw, mx, p, tiles, dev, stream);
  }
  if (c.kernel == SK_FP8_KERNEL_MANY) return launch_scaled<1, SILU>(mw, mx, p, tiles, dev, stream);
  if (c.kernel == SK_FP8_KERNEL_PAIR) return launch_scaled<2, SILU>(mw, mx, p, tiles, dev, stream);
  if constexpr (!SILU)
    if (c.row_tile == 32) return launch_scaled_narrow<32, SILU>(mw, mx, p, tiles, dev, stream);
  return launch_scaled_narrow<16, SILU>(mw, mx, p, tiles, dev, stream);
}

// silu_out: the SiLU epilogue; w then holds 2 * experts matrices of N rows.  early_weights: this library's quantiser is in front, or a product
// of the same call with it in front.  It lets its followers start only when all kernels in front of it are complete (fp8_quantize_kernel), those
// among them that wrote the weights or the groups' offsets, so both may be read before this kernel's own wait.
int product(int64_t M, const sk_fp8_rows* x, const sk_fp8_weight* w, int scale_type, const int32_t* offsets, void* out, int64_t ld_out,
            int out_dtype, const sk_fp8_rows* silu_out, bool early_weights, cudaStream_t stream) {
  const bool silu = silu_out != nullptr;
  const int64_t experts = silu ? w->experts / 2 : w->experts;
  const int64_t N = w->N, K = w->K;
  DeviceInfo dev;
  if (int rc = device_info(&dev); rc != SK_OK) return rc;
  const Choice c = choose(M, N, K, experts, offsets != nullptr, silu, scale_type == SK_SCALE_E8M0, dev);
  Fp8Params p = {};
  p.x_scale = x->scale;
  p.xs_row = x->scale_row;
  p.xs_blk = x->scale_block;
  p.w_scale = w->scale;
  const int64_t blocks = ceil_div(N, 128);
  p.scale_rows = silu ? 2 * blocks : blocks;
  p.offsets = offsets;
  p.experts = offsets ? static_cast<int>(experts) : 1;
  p.w_rows = static_cast<int>(silu ? 2 * N : N);
  p.out = silu ? silu_out->q : out;
  p.ld_out = silu ? silu_out->ld : ld_out;
  if (silu) {
    p.h_scale = silu_out->scale;
    p.hs_row = silu_out->scale_row;
    p.hs_blk = silu_out->scale_block;
    p.up_row0 = static_cast<int>(N);
    p.up_block0 = static_cast<int>(blocks);
  }
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.k_blocks = static_cast<int>(ceil_div(K, 128));
  p.n_tiles = static_cast<int>(ceil_div(N, c.feature_tile));
  p.out_bf16 = out_dtype == SK_OUT_BF16;
  p.out_f32 = out_dtype == kOutF32;
  p.out_bytes = silu ? 32 : aligned(out, 32) && ld_out % 16 == 0 ? 32 : aligned(out, 16) && ld_out % 8 == 0 ? 16 : 2;
  const int64_t four = 4 * scale_bytes(scale_type);
  p.x_scale_groups = p.xs_blk == 1 && p.xs_row % 4 == 0 && aligned(p.x_scale, four);
  p.w_scale_groups = p.k_blocks % 4 == 0 && aligned(p.w_scale, four);
  p.early_weights = early_weights;
  p.split = c.split;
  p.skip_block = static_cast<int>(g_options[SK_FP8_OPT_TEST_SKIP_COPY].load()) - 1;
  const int64_t limit = g_options[SK_FP8_OPT_WAIT_LIMIT_CYCLES].load();
  p.wait_limit = limit > 0 ? limit : kWaitLimitCycles;
  p.status = dev.status;
  const int64_t tiles = c.ctas / c.split;
  if (tiles > kIntMax / 8) return SK_ERR_BAD_SHAPE;
  CUtensorMap mw, mx;
  if (int rc = codes_map(w->q, w->experts * N, K, w->ld, 128, &mw); rc != SK_OK) return rc;
  if (int rc = codes_map(x->q, M, K, x->ld, std::min(c.row_tile, 128), &mx); rc != SK_OK) return rc;
  return with_bool(silu, [&](auto s) {
    return launch_product<decltype(s)::value>(c, scale_type == SK_SCALE_E8M0, mw, mx, p, tiles, dev, stream);
  });
}

int check_weight(const sk_fp8_weight* w, int64_t max_experts) {
  if (!w || !w->q || !w->scale) return SK_ERR_NULL_POINTER;
  if (w->experts < 1 || w->experts > max_experts || w->N < 1 || w->K < 1 || w->ld < w->K) return SK_ERR_BAD_SHAPE;
  if (w->N > kIntMax / 256 || w->K > kIntMax / 256 || w->experts * w->N > kIntMax - 4096 || w->ld >= (int64_t(1) << 36)) return SK_ERR_BAD_SHAPE;
  if (!aligned(w->q, 16) || w->ld % 16) return SK_ERR_BAD_ALIGNMENT;
  return SK_OK;
}
int check_rows(const sk_fp8_rows* x, int64_t M, int64_t K) {
  if (!x || !x->q || !x->scale) return SK_ERR_NULL_POINTER;
  if (M < 0 || M > kIntMax - 4096 || x->ld < K || x->ld >= (int64_t(1) << 36)) return SK_ERR_BAD_SHAPE;
  if (!aligned(x->q, 16) || x->ld % 16) return SK_ERR_BAD_ALIGNMENT;
  return SK_OK;
}

int quantize(const void* x, int x_type, int64_t ld_x, int64_t M, int64_t K, const sk_fp8_rows& out, int scale_type, const int32_t* rows,
             int64_t choices, cudaStream_t stream) {
  DeviceInfo dev;
  if (int rc = device_info(&dev); rc != SK_OK) return rc;
  const int64_t parts = ceil_div(ceil_div(K, 128), 16), most = std::max<int64_t>(1, static_cast<int64_t>(dev.sms) * 8 / parts);
  if (parts > 65535) return SK_ERR_BAD_SHAPE;
  const int64_t size = x_type == SK_FLOAT_F32 ? 4 : 2;
  const bool vector = aligned(x, 16) && ld_x * size % 16 == 0;
  LaunchConfig lc(std::min(M, most), parts, 256, 0, true, 1, stream);
  return with_type(x_type, [&](auto type) {
    return with_bool(scale_type == SK_SCALE_E8M0, [&](auto e8m0) {
      return with_bool(vector, [&](auto v) {
        return cuda_status(cudaLaunchKernelEx(&lc.cfg, fp8_quantize_kernel<decltype(type)::value, decltype(e8m0)::value, decltype(v)::value>, x,
                                              static_cast<long long>(ld_x), static_cast<long long>(M), static_cast<int>(K), out.q,
                                              static_cast<long long>(out.ld), out.scale, static_cast<long long>(out.scale_row),
                                              static_cast<long long>(out.scale_block), static_cast<const int*>(rows), static_cast<int>(choices),
                                              static_cast<int>(std::min<int64_t>(M * choices, kIntMax))));
      });
    });
  });
}

// Codes and scales of [M, K] in a workspace, rows on 32 bytes.  The scales lie row by row, rows padded to four: the products read four K blocks' at once.
int64_t scale_pitch(int64_t K) { return round_up(ceil_div(K, 128), 4); }
int64_t rows_bytes(int64_t M, int64_t K, int scale_type) {
  return round_up(M * round_up(K, 32), 256) + round_up(M * scale_pitch(K) * scale_bytes(scale_type), 256);
}
sk_fp8_rows rows_in(uint8_t* at, int64_t M, int64_t K, int scale_type) {
  sk_fp8_rows r;
  r.q = at;
  r.ld = round_up(K, 32);
  r.scale = at + round_up(M * r.ld, 256);
  r.scale_row = scale_pitch(K);
  r.scale_block = 1;
  return r;
}

// ---------------------------------------------------------------- router
// Tokens per CTA: one CTA for as long as its warps have two tokens each, then enough for one CTA per SM.
int64_t route_per_cta(int64_t T, int sms) {
  if (T <= 2 * kRouteWarps) return std::max<int64_t>(T, 1);
  return std::max<int64_t>(kRouteWarps, round_up(ceil_div(T, sms), kRouteWarps));
}

template <int TYPE, bool TOPK>
int launch_route(RouteParams p, int64_t ctas, const DeviceInfo& dev, cudaStream_t stream) {
  // (as many warps as there is work for, four at least: the experts' sums are spread over all threads)
  const int warps = std::min(kRouteWarps, std::max(4, TOPK ? p.per_cta : static_cast<int>(ceil_div(static_cast<int64_t>(p.per_cta) * p.k, 32))));
  const int smem = route_smem_bytes(warps, p.E);
  const auto go = [&](auto per) -> int {
    constexpr int kPer = decltype(per)::value;
    auto kern = ctas == 1 ? route_count_kernel<TYPE, kPer, TOPK, true> : route_count_kernel<TYPE, kPer, TOPK, false>;
    // (what any call may want, not what this one does: the limit is the kernel's, and another thread may be about to launch it)
    static std::atomic<uint64_t> done[2];
    if (int rc = allow_shared(kern, route_smem_bytes(kRouteWarps, kFp8MaxExperts), dev, done[ctas == 1]); rc != SK_OK) return rc;
    LaunchConfig lc(ctas, 1, warps * 32, smem, true, 1, stream);
    if (cudaError_t e = cudaLaunchKernelEx(&lc.cfg, kern, p); e != cudaSuccess) return cuda_status(e);
    if (ctas == 1) return SK_OK;
    LaunchConfig second(ctas, 1, 1024, (2 * p.E + 1) * 4, true, 1, stream);
    return cuda_status(cudaLaunchKernelEx(&second.cfg, route_shift_kernel, p));
  };
  if constexpr (!TOPK) {
    return go(std::integral_constant<int, 1>{});
  } else {
    const int per = static_cast<int>(ceil_div(p.E, 32));
    if (per <= 1) return go(std::integral_constant<int, 1>{});
    if (per <= 2) return go(std::integral_constant<int, 2>{});
    if (per <= 4) return go(std::integral_constant<int, 4>{});
    if (per <= 8) return go(std::integral_constant<int, 8>{});
    if (per <= 16) return go(std::integral_constant<int, 16>{});
    return go(std::integral_constant<int, 32>{});
  }
}

int route(RouteParams p, int logits_type, bool topk, int64_t T, int64_t E, int64_t k, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  DeviceInfo dev;
  if (int rc = device_info(&dev); rc != SK_OK) return rc;
  p.T = static_cast<int>(T);
  p.E = static_cast<int>(E);
  p.k = static_cast<int>(k);
  p.per_cta = static_cast<int>(route_per_cta(T, dev.sms));
  const int64_t ctas = std::max<int64_t>(1, ceil_div(T, p.per_cta));
  if (ctas > 1) {
    if (!workspace) return SK_ERR_NULL_POINTER;
    if (workspace_bytes < ctas * E * 4) return SK_ERR_BAD_ARGUMENT;
    if (!aligned(workspace, 4)) return SK_ERR_BAD_ALIGNMENT;
    p.counts = static_cast<int*>(workspace);
  }
  if (!topk) return launch_route<0, false>(p, ctas, dev, stream);
  return with_type(logits_type, [&](auto type) { return launch_route<decltype(type)::value, true>(p, ctas, dev, stream); });
}

int check_route(int64_t T, int64_t E, int64_t k) {
  if (E < 1 || E > kFp8MaxExperts || k < 1 || k > std::min<int64_t>(E, 32) || T < 0 || T > kIntMax / 64) return SK_ERR_BAD_SHAPE;
  return SK_OK;
}

}  // namespace
}  // namespace sk

using namespace sk;

extern "C" {

int sk_fp8_quantize(const void* x, int x_type, int64_t ld_x, int64_t M, int64_t K, const sk_fp8_rows* out, int scale_type, sk_stream_t stream) {
  if (!x || !out) return SK_ERR_NULL_POINTER;
  if (!is_float_type(x_type) || !is_scale_type(scale_type)) return SK_ERR_BAD_ARGUMENT;
  if (K < 1 || K > kIntMax / 256 || ld_x < K) return SK_ERR_BAD_SHAPE;
  if (int rc = check_rows(out, M, K); rc != SK_OK) return rc;
  if (!aligned(x, x_type == SK_FLOAT_F32 ? 4 : 2) || (scale_type == SK_SCALE_F32 && !aligned(out->scale, 4))) return SK_ERR_BAD_ALIGNMENT;
  if (M == 0) return SK_OK;
  return quantize(x, x_type, ld_x, M, K, *out, scale_type, nullptr, 1, static_cast<cudaStream_t>(stream));
}

int sk_fp8_prepare_weight(const void* w, int w_type, int64_t ld_w, int64_t w_matrix, int64_t matrices, int64_t N, int64_t K, uint8_t* w_q,
                          int64_t ld_q, int64_t q_matrix, void* w_scale, int scale_type, sk_stream_t stream) {
  if (!w || !w_q || !w_scale) return SK_ERR_NULL_POINTER;
  if (!is_float_type(w_type) || !is_scale_type(scale_type)) return SK_ERR_BAD_ARGUMENT;
  if (N < 1 || K < 1 || N > kIntMax / 256 || K > kIntMax / 256 || matrices < 1 || matrices > 65535 || ld_w < K || ld_q < K) return SK_ERR_BAD_SHAPE;
  const int64_t blocks = ceil_div(N, 128) * ceil_div(K, 128);
  if (blocks > kIntMax) return SK_ERR_BAD_SHAPE;
  if (!aligned(w, w_type == SK_FLOAT_F32 ? 4 : 2) || !aligned(w_q, 16) || ld_q % 16 || q_matrix % 4) return SK_ERR_BAD_ALIGNMENT;
  if (scale_type == SK_SCALE_F32 && !aligned(w_scale, 4)) return SK_ERR_BAD_ALIGNMENT;
  DeviceInfo dev;
  if (int rc = device_info(&dev); rc != SK_OK) return rc;
  LaunchConfig lc(blocks, matrices, 256, 0, false, 1, static_cast<cudaStream_t>(stream));
  return with_type(w_type, [&](auto type) {
    return with_bool(scale_type == SK_SCALE_E8M0, [&](auto e8m0) {
      return cuda_status(cudaLaunchKernelEx(&lc.cfg, fp8_prepare_weight_kernel<decltype(type)::value, decltype(e8m0)::value>, w,
                                            static_cast<long long>(ld_w), static_cast<long long>(w_matrix), static_cast<int>(N), static_cast<int>(K),
                                            w_q, static_cast<long long>(ld_q), static_cast<long long>(q_matrix), w_scale));
    });
  });
}

static int check_product(int64_t M, const sk_fp8_weight* w, int scale_type, const void* out, int64_t ld_out, int out_dtype, int64_t max_experts) {
  if (int rc = check_weight(w, max_experts); rc != SK_OK) return rc;
  if (!out) return SK_ERR_NULL_POINTER;
  if (!is_scale_type(scale_type) || !is_out_type(out_dtype)) return SK_ERR_BAD_ARGUMENT;
  if (scale_type == SK_SCALE_F32 && !aligned(w->scale, 4)) return SK_ERR_BAD_ALIGNMENT;
  if (M < 0 || M > kIntMax - 4096 || ld_out < w->N) return SK_ERR_BAD_SHAPE;
  if (!aligned(out, 2)) return SK_ERR_BAD_ALIGNMENT;
  return SK_OK;
}

int sk_fp8_gemm(int64_t M, const sk_fp8_rows* x, const sk_fp8_weight* w, int scale_type, void* out, int64_t ld_out, int out_dtype, sk_stream_t stream) {
  if (int rc = check_product(M, w, scale_type, out, ld_out, out_dtype, 1); rc != SK_OK) return rc;
  if (int rc = check_rows(x, M, w->K); rc != SK_OK) return rc;
  if (scale_type == SK_SCALE_F32 && !aligned(x->scale, 4)) return SK_ERR_BAD_ALIGNMENT;
  if (M == 0) return SK_OK;
  return product(M, x, w, scale_type, nullptr, out, ld_out, out_dtype, nullptr, false, static_cast<cudaStream_t>(stream));
}

int sk_fp8_grouped_gemm(int64_t M, const sk_fp8_rows* x, const sk_fp8_weight* w, int scale_type, const int32_t* offsets, void* out, int64_t ld_out,
                        int out_dtype, sk_stream_t stream) {
  if (int rc = check_product(M, w, scale_type, out, ld_out, out_dtype, kFp8MaxExperts); rc != SK_OK) return rc;
  if (int rc = check_rows(x, M, w->K); rc != SK_OK) return rc;
  if (!offsets) return SK_ERR_NULL_POINTER;
  if (!aligned(offsets, 4) || (scale_type == SK_SCALE_F32 && !aligned(x->scale, 4))) return SK_ERR_BAD_ALIGNMENT;
  if (M == 0) return SK_OK;
  return product(M, x, w, scale_type, offsets, out, ld_out, out_dtype, nullptr, false, static_cast<cudaStream_t>(stream));
}

int64_t sk_fp8_linear_workspace_bytes(int64_t M, int64_t K, int scale_type) {
  if (M < 0 || K < 1 || !is_scale_type(scale_type)) return 0;
  return rows_bytes(M, K, scale_type);
}

int sk_fp8_linear(int64_t M, const void* x, int x_type, int64_t ld_x, const sk_fp8_weight* w, int scale_type, void* out, int64_t ld_out, int out_dtype,
                  void* workspace, int64_t workspace_bytes, sk_stream_t stream) {
  if (int rc = check_product(M, w, scale_type, out, ld_out, out_dtype, 1); rc != SK_OK) return rc;
  if (!x || !workspace) return SK_ERR_NULL_POINTER;
  if (!is_float_type(x_type) || workspace_bytes < rows_bytes(M, w->K, scale_type)) return SK_ERR_BAD_ARGUMENT;
  if (ld_x < w->K) return SK_ERR_BAD_SHAPE;
  if (!aligned(x, x_type == SK_FLOAT_F32 ? 4 : 2) || !aligned(workspace, 256)) return SK_ERR_BAD_ALIGNMENT;
  if (M == 0) return SK_OK;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const sk_fp8_rows rows = rows_in(static_cast<uint8_t*>(workspace), M, w->K, scale_type);
  if (int rc = quantize(x, x_type, ld_x, M, w->K, rows, scale_type, nullptr, 1, s); rc != SK_OK) return rc;
  return product(M, &rows, w, scale_type, nullptr, out, ld_out, out_dtype, nullptr, true, s);
}

int64_t sk_route_workspace_bytes(int64_t T, int64_t E) {
  if (check_route(T, E, 1) != SK_OK) return 0;
  // (never more CTAs than this, whatever the device)
  return T <= 2 * kRouteWarps ? 0 : std::min<int64_t>(ceil_div(T, kRouteWarps), 1024) * E * 4;
}

int sk_route_tokens(const void* logits, int logits_type, int64_t ld, int64_t T, int64_t E, int64_t k, int renormalize, int32_t* ids, float* weights,
                    int32_t* rows, int32_t* offsets, void* workspace, int64_t workspace_bytes, sk_stream_t stream) {
  if (!logits || !ids || !weights || !rows || !offsets) return SK_ERR_NULL_POINTER;
  if (!is_float_type(logits_type)) return SK_ERR_BAD_ARGUMENT;
  if (int rc = check_route(T, E, k); rc != SK_OK) return rc;
  if (ld < E) return SK_ERR_BAD_SHAPE;
  if (!aligned(logits, logits_type == SK_FLOAT_F32 ? 4 : 2) || !aligned4({ids, weights, rows, offsets})) return SK_ERR_BAD_ALIGNMENT;
  RouteParams p = {};
  p.logits = logits;
  p.ld = ld;
  p.renormalize = renormalize != 0;
  p.ids = ids;
  p.weights = weights;
  p.rows = rows;
  p.offsets = offsets;
  return route(p, logits_type, true, T, E, k, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int sk_group_by_expert(const int32_t* ids, int64_t T, int64_t k, int64_t E, int32_t* rows, int32_t* offsets, void* workspace, int64_t workspace_bytes,
                       sk_stream_t stream) {
  if (!ids || !rows || !offsets) return SK_ERR_NULL_POINTER;
  if (int rc = check_route(T, E, 1); rc != SK_OK) return rc;
  if (k < 1 || k > 1024 || T * k > kIntMax) return SK_ERR_BAD_SHAPE;
  if (!aligned4({ids, rows, offsets})) return SK_ERR_BAD_ALIGNMENT;
  RouteParams p = {};
  p.ids = const_cast<int32_t*>(ids);               // (only read)
  p.rows = rows;
  p.offsets = offsets;
  return route(p, SK_FLOAT_F32, false, T, E, k, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int64_t sk_fp8_experts_workspace_bytes(int64_t T, int64_t k, int64_t hidden, int64_t inter, int scale_type) {
  if (T < 0 || k < 1 || hidden < 1 || inter < 1 || !is_scale_type(scale_type)) return 0;
  return rows_bytes(T * k, hidden, scale_type) + rows_bytes(T * k, inter, scale_type) + round_up(T * k * round_up(hidden, 16) * 4, 256);
}

int sk_fp8_experts(int64_t T, int64_t k, const void* x, int x_type, int64_t ld_x, const int32_t* rows, const float* weights, const int32_t* offsets,
                   const sk_fp8_weight* gate_up, const sk_fp8_weight* down, int scale_type, void* out, int64_t ld_out, int out_dtype, void* workspace,
                   int64_t workspace_bytes, sk_stream_t stream) {
  if (!x || !rows || !weights || !offsets || !workspace) return SK_ERR_NULL_POINTER;
  if (int rc = check_product(T, down, scale_type, out, ld_out, out_dtype, kFp8MaxExperts); rc != SK_OK) return rc;
  if (int rc = check_weight(gate_up, 2 * kFp8MaxExperts); rc != SK_OK) return rc;
  if (scale_type == SK_SCALE_F32 && !aligned(gate_up->scale, 4)) return SK_ERR_BAD_ALIGNMENT;
  const int64_t hidden = down->N, inter = down->K, E = down->experts;
  if (gate_up->experts != 2 * E || gate_up->N != inter || gate_up->K != hidden || ld_x < hidden) return SK_ERR_BAD_SHAPE;
  if (k < 1 || k > 1024 || T * k > kIntMax - 4096) return SK_ERR_BAD_SHAPE;
  if (!is_float_type(x_type) || workspace_bytes < sk_fp8_experts_workspace_bytes(T, k, hidden, inter, scale_type)) return SK_ERR_BAD_ARGUMENT;
  if (!aligned(x, x_type == SK_FLOAT_F32 ? 4 : 2) || !aligned(workspace, 256) || !aligned4({rows, weights, offsets})) return SK_ERR_BAD_ALIGNMENT;
  if (T == 0) return SK_OK;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t R = T * k, ld_y = round_up(hidden, 16);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  const sk_fp8_rows xr = rows_in(at, R, hidden, scale_type);
  at += rows_bytes(R, hidden, scale_type);
  const sk_fp8_rows hr = rows_in(at, R, inter, scale_type);
  at += rows_bytes(R, inter, scale_type);
  if (int rc = quantize(x, x_type, ld_x, T, hidden, xr, scale_type, rows, k, s); rc != SK_OK) return rc;
  if (int rc = product(R, &xr, gate_up, scale_type, offsets, nullptr, 0, out_dtype, &hr, true, s); rc != SK_OK) return rc;
  if (int rc = product(R, &hr, down, scale_type, offsets, at, ld_y, kOutF32, nullptr, true, s); rc != SK_OK) return rc;
  DeviceInfo dev;
  if (int rc = device_info(&dev); rc != SK_OK) return rc;
  const bool vector = hidden % 8 == 0 && ld_out % 8 == 0 && aligned(out, 16);
  const int64_t units = T * (vector ? hidden / 8 : hidden);
  LaunchConfig lc(std::min<int64_t>(ceil_div(units, 256), static_cast<int64_t>(dev.sms) * 8), 1, 256, 0, true, 1, s);
  return with_bool(out_dtype == SK_OUT_BF16, [&](auto bf16) {
    return with_bool(vector, [&](auto v) {
      return cuda_status(cudaLaunchKernelEx(&lc.cfg, fp8_combine_kernel<decltype(bf16)::value, decltype(v)::value>,
                                            reinterpret_cast<const float*>(at), static_cast<long long>(ld_y), static_cast<const int*>(rows), weights,
                                            static_cast<int>(k), static_cast<int>(T), static_cast<int>(hidden), static_cast<uint16_t*>(out),
                                            static_cast<long long>(ld_out)));
    });
  });
}

int sk_fp8_last_device_status(int device, int* device_status) {
  if (device_status) *device_status = 0;
  int cur = 0;
  if (cudaError_t e = cudaGetDevice(&cur); e != cudaSuccess) return cuda_status(e);
  if (cudaError_t e = cudaSetDevice(device); e != cudaSuccess) return cuda_status(e);
  int word = 0;
  const int zero = 0;
  // (the copy alone would wait for streams that synchronise with the legacy one, and others may still run into their limit)
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&word, g_fp8_status, sizeof(int));
  // (while the word is not zero, kernels leave it as it is: nothing noted in between is lost)
  if (e == cudaSuccess && word != 0) e = cudaMemcpyToSymbol(g_fp8_status, &zero, sizeof(int));
  (void)cudaSetDevice(cur);
  if (e != cudaSuccess) return cuda_status(e);
  if (device_status) *device_status = word;
  return word == 0 ? SK_OK : SK_ERR_DEVICE_TIMEOUT;
}

int sk_fp8_query_launch(int64_t M, int64_t N, int64_t K, int64_t experts, int scale_type, int* kernel, int* row_tile, int* feature_tile, int* split, int* ctas) {
  if (M < 1 || N < 1 || K < 1 || experts < 1 || experts > kFp8MaxExperts) return SK_ERR_BAD_SHAPE;
  if (!is_scale_type(scale_type)) return SK_ERR_BAD_ARGUMENT;
  DeviceInfo dev;
  if (int rc = device_info(&dev); rc != SK_OK) return rc;
  const Choice c = choose(M, N, K, experts, experts > 1, false, scale_type == SK_SCALE_E8M0, dev);
  if (kernel) *kernel = c.kernel;
  if (row_tile) *row_tile = c.row_tile;
  if (feature_tile) *feature_tile = c.feature_tile;
  if (split) *split = c.split;
  if (ctas) *ctas = static_cast<int>(std::min<int64_t>(c.ctas, kIntMax));
  return SK_OK;
}

int sk_fp8_set_option(int key, int64_t value) {
  if (value < 0) return SK_ERR_BAD_ARGUMENT;
  switch (key) {
    case SK_FP8_OPT_ROW_TILE:
      if (value != 0 && value != 16 && value != 32) return SK_ERR_BAD_ARGUMENT;
      break;
    case SK_FP8_OPT_SPLIT_K:
      if (value != 0 && value != 1 && value != 2 && value != 4 && value != 8) return SK_ERR_BAD_ARGUMENT;
      break;
    case SK_FP8_OPT_WAIT_LIMIT_CYCLES:
      // (a wait is not given up before every copy in flight has long landed: a producer that is done does not look after its last ones)
      if (value != 0 && value < 1000000) return SK_ERR_BAD_ARGUMENT;
      break;
    case SK_FP8_OPT_KERNEL:
      if (value > SK_FP8_KERNEL_PAIR) return SK_ERR_BAD_ARGUMENT;
      break;
    case SK_FP8_OPT_TEST_SKIP_COPY:
      if (value > kIntMax) return SK_ERR_BAD_ARGUMENT;
      break;
    default: return SK_ERR_BAD_ARGUMENT;
  }
  g_options[key].store(value);
  return SK_OK;
}

}  // extern "C"
