/*
 * sk_fp8.h — C ABI of the FP8 products next to the W2A8 GEMM: 8-bit floats (e4m3) with one scale per block of 128.
 *
 *   out[m, n] = cast( sum_b x_scale[m, b] * w_scale[n / 128, b] * fp32( sum_{k in block b} x_q[m, k] * w_q[n, k] ) )
 *
 * For the layers that 2-bit weights do not suit (the output head, say) and for mixture-of-experts layers, whose products are
 * grouped by expert.  The functions live in the library of sk_w2a8.h and share its status codes and conventions: raw device
 * pointers, caller-owned buffers, leading dimensions in elements, everything asynchronous on `stream`, no allocation, no
 * exception.  They keep no plan: a call reads its operands as they are when it runs.  All pointers must belong to the current device.
 *
 * Scales are 32-bit floats or 8-bit exponents (e8m0: 2^(b - 127), 255 is NaN); both operands of a product have the same type.
 * K may be any number: the last block of a row is short.  Rows of codes start on 16 bytes (ld % 16 == 0, base 16-byte aligned).
 */
#ifndef SK_FP8_H_
#define SK_FP8_H_

#include "sk_w2a8.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum sk_scale_type { SK_SCALE_F32 = 0, SK_SCALE_E8M0 = 1 } sk_scale_type;
typedef enum sk_float_type { SK_FLOAT_F16 = 0, SK_FLOAT_BF16 = 1, SK_FLOAT_F32 = 2 } sk_float_type;

/* Activations: codes [M, K] with leading dimension ld; scale of row m and block b at scale[m * scale_row + b * scale_block]. */
typedef struct sk_fp8_rows {
  uint8_t* q;
  int64_t ld;
  void* scale;
  int64_t scale_row, scale_block;
} sk_fp8_rows;

/* Weights: `experts` matrices of [N, K] codes, one behind the other (leading dimension ld), scales
 * [experts][ceil(N / 128)][ceil(K / 128)] contiguous. */
typedef struct sk_fp8_weight {
  const uint8_t* q;
  int64_t ld;
  const void* scale;
  int64_t experts, N, K;
} sk_fp8_weight;

/* x [M, K] -> codes and scales, per row and block of 128:  a = max|x|, scale = 2^e with the smallest e such that a <= 448 * 2^e
 * (e = 0 where a = 0; e >= -126), code = x / scale rounded to nearest even.  A block with an infinity or a NaN gets a NaN scale and NaN
 * codes.  x_type: sk_float_type.  Any K, any ld_x >= K; 16-byte aligned rows are read faster. */
int sk_fp8_quantize(const void* x, int x_type, int64_t ld_x, int64_t M, int64_t K, const sk_fp8_rows* out, int scale_type,
                    sk_stream_t stream);
/* The same rule for weights: `matrices` matrices [N, K] (row pitch ld_w, w_matrix elements apart) -> codes (row pitch ld_q,
 * q_matrix apart) and one scale per 128 x 128 block, [matrices][ceil(N / 128)][ceil(K / 128)]. */
int sk_fp8_prepare_weight(const void* w, int w_type, int64_t ld_w, int64_t w_matrix, int64_t matrices, int64_t N, int64_t K,
                          uint8_t* w_q, int64_t ld_q, int64_t q_matrix, void* w_scale, int scale_type, sk_stream_t stream);

/* out [M, N] = the product above; out_dtype: sk_out_dtype.  experts must be 1. */
int sk_fp8_gemm(int64_t M, const sk_fp8_rows* x, const sk_fp8_weight* w, int scale_type, void* out, int64_t ld_out, int out_dtype,
                sk_stream_t stream);

/* A whole linear layer on float activations x [M, K]: quantise, then the product.  The codes live in a workspace of
 * sk_fp8_linear_workspace_bytes(M, K, scale_type) bytes, 256-byte aligned. */
int64_t sk_fp8_linear_workspace_bytes(int64_t M, int64_t K, int scale_type);
int sk_fp8_linear(int64_t M, const void* x, int x_type, int64_t ld_x, const sk_fp8_weight* w, int scale_type, void* out, int64_t ld_out,
                  int out_dtype, void* workspace, int64_t workspace_bytes, sk_stream_t stream);

/* Products grouped by expert: rows offsets[e] .. offsets[e + 1] - 1 of x (device memory, int32 [experts + 1], non-decreasing) times
 * expert e's matrix.  Groups may be empty; rows outside [offsets[0], offsets[experts]) of `out` are left as they were.  Offsets
 * outside [0, M] are cut to it.  experts <= 1024. */
int sk_fp8_grouped_gemm(int64_t M, const sk_fp8_rows* x, const sk_fp8_weight* w, int scale_type, const int32_t* offsets, void* out,
                        int64_t ld_out, int out_dtype, sk_stream_t stream);

/* Router: the k largest of a token's E logits (ties: the lower expert first) and softmax weights; renormalize: divided by the sum of
 * the k chosen.  rows[t, j] is the place of choice (t, j) in the order of the experts and, within an expert, of t * k + j; offsets
 * [E + 1] the experts' first places.  -infinity masks an expert (it is chosen last, with weight zero; a token with nothing else
 * gets weights of zero); NaN and +infinity give the token NaN weights.  logits [T, E], row pitch ld, sk_float_type.  E <= 1024,
 * k <= min(E, 32).  workspace: sk_route_workspace_bytes(T, E) bytes of device memory (0: none). */
int64_t sk_route_workspace_bytes(int64_t T, int64_t E);
int sk_route_tokens(const void* logits, int logits_type, int64_t ld, int64_t T, int64_t E, int64_t k, int renormalize, int32_t* ids,
                    float* weights, int32_t* rows, int32_t* offsets, void* workspace, int64_t workspace_bytes, sk_stream_t stream);
/* The places and offsets alone, for experts chosen elsewhere.  Ids outside [0, E) belong to nobody here: their rows are -1. */
int sk_group_by_expert(const int32_t* ids, int64_t T, int64_t k, int64_t E, int32_t* rows, int32_t* offsets, void* workspace,
                       int64_t workspace_bytes, sk_stream_t stream);

/* The expert layers of a mixture-of-experts block on routed tokens:
 *   y_e(x) = W_down[e] q( SiLU(gate) * up ),   [gate; up] = W_gate_up[e] q(x),   q the quantiser above,
 *   out[t] = cast( sum_j weights[t, j] * y_{expert of (t, j)}(x[t]) ),   choices with rows outside [0, T * k) count nothing.
 * gate_up: 2 * experts matrices [inter, hidden] (an expert's gate, then its up; `experts` there counts matrices), down: experts
 * matrices [hidden, inter].  y and its sum are fp32, rounded once.  x_type: fp16 or bf16 or fp32.  rows and offsets are those of
 * one routing: a place that lies in no group has no result.  The workspace is 256-byte aligned. */
int64_t sk_fp8_experts_workspace_bytes(int64_t T, int64_t k, int64_t hidden, int64_t inter, int scale_type);
int sk_fp8_experts(int64_t T, int64_t k, const void* x, int x_type, int64_t ld_x, const int32_t* rows, const float* weights,
                   const int32_t* offsets, const sk_fp8_weight* gate_up, const sk_fp8_weight* down, int scale_type, void* out,
                   int64_t ld_out, int out_dtype, void* workspace, int64_t workspace_bytes, sk_stream_t stream);

/* Waits for all work on `device`, then reads and clears the word in which a kernel of this header notes a wait that ran into its limit there;
 * non-zero maps to SK_ERR_DEVICE_TIMEOUT.  sk_device_status_string words it.  The output of such a launch is undefined. */
int sk_fp8_last_device_status(int device, int* device_status);
typedef enum sk_fp8_kernel {
  SK_FP8_KERNEL_FEW = 1,        /* few rows: features on the tensor memory's lanes, tiles of 16 or (8-bit scales) 32 rows */
  SK_FP8_KERNEL_MANY = 2,       /* many rows: 128 of them on the lanes */
  SK_FP8_KERNEL_PAIR = 3        /* the same on pairs of CTAs, 256 rows (8-bit scales) */
} sk_fp8_kernel;                /* 8-bit scales are multiplied in by the tensor core, 32-bit ones in fp32 after every K block */
/* The launch a product makes: kernel, rows per tile, features per tile, CTAs that share a tile's K range, CTAs (at most).  experts > 1:
 * a product by expert of M rows in all. */
int sk_fp8_query_launch(int64_t M, int64_t N, int64_t K, int64_t experts, int scale_type, int* kernel, int* row_tile, int* feature_tile,
                        int* split, int* ctas);

/* Testing and tuning, process-wide; 0 restores the default. */
typedef enum sk_fp8_option {
  SK_FP8_OPT_ROW_TILE = 1,          /* rows per tile of the kernel for few rows: 16 / 32 (16 where there is no 32) */
  SK_FP8_OPT_SPLIT_K = 2,           /* CTAs that share the K range of a tile (products of one group) */
  SK_FP8_OPT_WAIT_LIMIT_CYCLES = 3, /* as SK_OPT_WAIT_LIMIT_CYCLES, 10^6 at least */
  SK_FP8_OPT_TEST_SKIP_COPY = 4,    /* as SK_OPT_TEST_SKIP_COPY */
  SK_FP8_OPT_KERNEL = 5             /* sk_fp8_kernel; with 32-bit scales 3 means 2 */
} sk_fp8_option;
int sk_fp8_set_option(int key, int64_t value);

#ifdef __cplusplus
}
#endif
#endif /* SK_FP8_H_ */
