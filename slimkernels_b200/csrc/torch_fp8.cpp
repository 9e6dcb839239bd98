// The FP8 ops of namespace `slimkernels` (slimkernels_b200/torch/fp8.py): tensors into the C ABI of include/sk_fp8.h.  No kernels
// live here.  Inference only, like the W2A8 ops: nothing is recorded for a backward pass.
#include <ATen/Context.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>
#include <torch/library.h>
#include <torch/types.h>

#include <tuple>
#include <vector>

#include "../../include/sk_fp8.h"

namespace {

void check(int rc, const char* what) {
  TORCH_CHECK(rc == SK_OK, "slimkernels::", what, " failed: ", sk_status_string(rc), " (", rc, ")");
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// at::empty on like's device without a turn through the dispatcher (0.4 us each; a router call makes four), so dispatch modes do not see it.
// torch's deterministic mode, which fills new tensors, has its turn.
at::Tensor fresh(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
  const at::Context& context = at::globalContext();
  if (C10_UNLIKELY(context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory())) return at::empty(size, like.options().dtype(type));
  return at::Tensor(at::detail::empty_cuda(size, type, like.device(), c10::nullopt));
}

int float_type(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kHalf: return SK_FLOAT_F16;
    case at::kBFloat16: return SK_FLOAT_BF16;
    case at::kFloat: return SK_FLOAT_F32;
    default: TORCH_CHECK(false, what, " must be float16, bfloat16 or float32, got ", t.scalar_type());
  }
}

int out_type(at::ScalarType t) {
  TORCH_CHECK(t == at::kHalf || t == at::kBFloat16, "out_dtype must be float16 or bfloat16");
  return t == at::kBFloat16 ? SK_OUT_BF16 : SK_OUT_F16;
}

// What a product returns where the caller does not say: the activations' own 16-bit type, float16 for others.
at::ScalarType default_out(const at::Tensor& x, c10::optional<at::ScalarType> asked) {
  if (asked.has_value()) return *asked;
  return x.scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kHalf;
}

int scale_type(at::ScalarType t, const char* what) {
  TORCH_CHECK(t == at::kFloat || t == at::kFloat8_e8m0fnu, what, " must be float32 or float8_e8m0fnu, got ", t);
  return t == at::kFloat ? SK_SCALE_F32 : SK_SCALE_E8M0;
}

void same_device(const at::Tensor& a, const at::Tensor& b, const char* what) {
  TORCH_CHECK(b.is_cuda() && b.get_device() == a.get_device(), what, " must be on ", a.device(), ", it is on ", b.device());
}

// Activations as rows, unit inner stride: as they are where possible (any row pitch), else contiguous.
at::Tensor as_rows(const at::Tensor& x, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1, what, " must be a CUDA tensor [..., K]");
  at::Tensor x2 = x.dim() == 2 ? x : x.reshape({x.size(-1) == 0 ? 0 : x.numel() / x.size(-1), x.size(-1)});
  const bool plain = (x2.size(1) <= 1 || x2.stride(1) == 1) && (x2.size(0) <= 1 || x2.stride(0) >= x2.size(1));
  return plain ? x2 : x2.contiguous();
}
int64_t pitch(const at::Tensor& rows) { return rows.size(0) <= 1 ? rows.size(1) : rows.stride(0); }

at::Tensor with_leading_shape(const at::Tensor& y, const at::Tensor& x) {
  if (x.dim() == 2) return y;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = y.size(1);
  return y.reshape(shape);
}

// Codes [M, K] and their scales as the products take them.
sk_fp8_rows fp8_rows(const at::Tensor& q, const at::Tensor& scale, const char* name) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kFloat8_e4m3fn && q.dim() == 2, name, "_q must be a 2-D CUDA float8_e4m3fn tensor [M, K]");
  const int64_t M = q.size(0), K = q.size(1);
  TORCH_CHECK(K >= 1 && (K == 1 || q.stride(1) == 1), name, "_q must have unit inner stride and at least one feature");
  TORCH_CHECK(scale.dim() == 2 && scale.size(0) == M && scale.size(1) == ceil_div(K, 128), name, "_scale must have shape [M, ceil(K / 128)] = [", M,
              ", ", ceil_div(K, 128), "]");
  same_device(q, scale, "the scales");
  sk_fp8_rows r;
  r.q = static_cast<uint8_t*>(q.data_ptr());
  r.ld = M <= 1 ? round_up(K, 16) : q.stride(0);      // (the pitch of a single row is never used)
  TORCH_CHECK(r.ld >= K && r.ld % 16 == 0 && (reinterpret_cast<uintptr_t>(r.q) & 15) == 0, name,
              "_q rows must start on 16 bytes (quantize_fp8 pads them so)");
  r.scale = scale.data_ptr();
  r.scale_row = scale.stride(0);
  r.scale_block = scale.stride(1);
  return r;
}

// Weights [N, K] or [..., N, K]: the matrices lie one behind the other.
sk_fp8_weight fp8_weight(const at::Tensor& q, const at::Tensor& scale, const char* name) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kFloat8_e4m3fn && q.dim() >= 2, name, " must be a CUDA float8_e4m3fn tensor [..., N, K]");
  const int64_t N = q.size(-2), K = q.size(-1);
  TORCH_CHECK(N >= 1 && K >= 1 && q.numel() > 0, name, " must not be empty");
  TORCH_CHECK(K == 1 || q.stride(-1) == 1, name, " must have unit inner stride");
  sk_fp8_weight w;
  w.experts = q.numel() / (N * K);
  // one row pitch through all rows of all matrices
  const int64_t rows = w.experts * N;
  int64_t ld = round_up(K, 16), expect = 0;
  bool regular = true;
  for (int64_t d = q.dim() - 2, below = 1; d >= 0; below *= q.size(d), --d) {
    if (q.size(d) <= 1) continue;
    if (expect == 0) {
      ld = q.stride(d) / below;
      regular = regular && q.stride(d) == ld * below;
      expect = 1;
    } else {
      regular = regular && q.stride(d) == ld * below;
    }
  }
  TORCH_CHECK(regular && (rows <= 1 || ld >= K), name, " must be stored row by row, one matrix behind the other");
  TORCH_CHECK(ld % 16 == 0 && (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0, name,
              " rows must start on 16 bytes (prepare_weight_fp8 pads them so)");
  std::vector<int64_t> shape(q.sizes().begin(), q.sizes().end());
  shape[shape.size() - 2] = ceil_div(N, 128);
  shape[shape.size() - 1] = ceil_div(K, 128);
  TORCH_CHECK(scale.sizes() == at::IntArrayRef(shape) && scale.is_contiguous(), "the scales of ", name, " must be contiguous with shape ",
              at::IntArrayRef(shape));
  same_device(q, scale, "the scales");
  w.q = static_cast<const uint8_t*>(q.data_ptr());
  w.ld = ld;
  w.scale = scale.data_ptr();
  w.N = N;
  w.K = K;
  return w;
}

int one_scale_type(const at::Tensor& a, const at::Tensor& b) {
  const int t = scale_type(a.scalar_type(), "scales");
  TORCH_CHECK(a.scalar_type() == b.scalar_type(), "the scales of a product must have one type, got ", a.scalar_type(), " and ", b.scalar_type());
  return t;
}

// Empty codes [M, K] with rows on 16 bytes, and their scales in the order the products read fastest.
std::tuple<at::Tensor, at::Tensor> empty_rows(const at::Tensor& like, int64_t M, int64_t K, at::ScalarType scales) {
  const int64_t kb = ceil_div(K, 128);
  at::Tensor q = fresh({M, round_up(K, 16)}, at::kFloat8_e4m3fn, like).narrow(1, 0, K);
  at::Tensor s = fresh({M, round_up(kb, 4)}, scales, like).narrow(1, 0, kb);
  return {q, s};
}

std::tuple<at::Tensor, at::Tensor> quantize_fp8(const at::Tensor& x, at::ScalarType scale_dtype) {
  const int st = scale_type(scale_dtype, "scale_dtype");
  const at::Tensor x2 = as_rows(x, "x");
  const int ft = float_type(x2, "x");
  const int64_t M = x2.size(0), K = x2.size(1);
  TORCH_CHECK(K >= 1, "x must have at least one feature");
  c10::cuda::CUDAGuard guard(x2.device());
  auto [q, s] = empty_rows(x2, M, K, scale_dtype);
  if (M > 0) {
    sk_fp8_rows r{static_cast<uint8_t*>(q.data_ptr()), round_up(K, 16), s.data_ptr(), s.stride(0), s.stride(1)};
    check(sk_fp8_quantize(x2.data_ptr(), ft, pitch(x2), M, K, &r, st, at::cuda::getCurrentCUDAStream().stream()), "quantize_fp8");
  }
  if (x.dim() == 2) return {q, s};
  std::vector<int64_t> lead(x.sizes().begin(), x.sizes().end() - 1);
  if (lead.empty()) return {q.squeeze(0), s.squeeze(0)};
  return {q.unflatten(0, lead), s.unflatten(0, lead)};
}

std::tuple<at::Tensor, at::Tensor> prepare_weight_fp8(const at::Tensor& w, at::ScalarType scale_dtype) {
  const int st = scale_type(scale_dtype, "scale_dtype");
  TORCH_CHECK(w.is_cuda() && w.dim() >= 2 && w.numel() > 0, "w must be a CUDA tensor [..., N, K] that is not empty");
  const int ft = float_type(w, "w");
  const int64_t N = w.size(-2), K = w.size(-1), matrices = w.numel() / (N * K);
  TORCH_CHECK(matrices <= 65535, "too many matrices");
  const at::Tensor c = w.contiguous();
  c10::cuda::CUDAGuard guard(w.device());
  std::vector<int64_t> shape(w.sizes().begin(), w.sizes().end()), blocks = shape;
  shape.back() = round_up(K, 16);
  blocks[blocks.size() - 2] = ceil_div(N, 128);
  blocks.back() = ceil_div(K, 128);
  at::Tensor q = K % 16 ? at::zeros(shape, w.options().dtype(at::kByte)).view(at::kFloat8_e4m3fn) : at::empty(shape, w.options().dtype(at::kFloat8_e4m3fn));
  at::Tensor s = at::empty(blocks, w.options().dtype(scale_dtype));
  check(sk_fp8_prepare_weight(c.data_ptr(), ft, K, N * K, matrices, N, K, static_cast<uint8_t*>(q.data_ptr()), shape.back(), N * shape.back(),
                              s.data_ptr(), st, at::cuda::getCurrentCUDAStream().stream()),
        "prepare_weight_fp8");
  return {q.narrow(-1, 0, K), s};
}

void check_out(const at::Tensor& out, const at::Tensor& x, int64_t M, int64_t N) {
  TORCH_CHECK(out.is_cuda() && out.dim() == 2 && out.size(0) == M && out.size(1) == N && (N == 1 || out.stride(1) == 1),
              "out must be [M, N] = [", M, ", ", N, "] with unit inner stride");
  TORCH_CHECK(M <= 1 || out.stride(0) >= N, "the rows of out must not overlap");
  same_device(x, out, "out");
}

void fp8_gemm_out(const at::Tensor& x_q, const at::Tensor& x_scale, const at::Tensor& w_q, const at::Tensor& w_scale, at::Tensor& out) {
  const sk_fp8_rows x = fp8_rows(x_q, x_scale, "x");
  const sk_fp8_weight w = fp8_weight(w_q, w_scale, "w_q");
  TORCH_CHECK(w_q.dim() == 2, "w_q must have shape [N, K]");
  const int st = one_scale_type(x_scale, w_scale);
  same_device(x_q, w_q, "w_q");
  const int64_t M = x_q.size(0);
  TORCH_CHECK(w.K == x_q.size(1), "x_q has ", x_q.size(1), " features, w_q ", w.K);
  check_out(out, x_q, M, w.N);
  const int ot = out_type(out.scalar_type());
  if (M == 0) return;
  c10::cuda::CUDAGuard guard(x_q.device());
  check(sk_fp8_gemm(M, &x, &w, st, out.data_ptr(), M == 1 ? w.N : out.stride(0), ot, at::cuda::getCurrentCUDAStream().stream()), "fp8_gemm");
}

at::Tensor fp8_gemm(const at::Tensor& x_q, const at::Tensor& x_scale, const at::Tensor& w_q, const at::Tensor& w_scale, at::ScalarType out_dtype) {
  out_type(out_dtype);
  TORCH_CHECK(x_q.dim() == 2 && w_q.dim() == 2, "x_q must have shape [M, K] and w_q [N, K]");
  at::Tensor out = fresh({x_q.size(0), w_q.size(0)}, out_dtype, x_q);
  fp8_gemm_out(x_q, x_scale, w_q, w_scale, out);
  return out;
}

at::Tensor fp8_linear(const at::Tensor& x, const at::Tensor& w_q, const at::Tensor& w_scale, c10::optional<at::ScalarType> out_dtype) {
  const sk_fp8_weight w = fp8_weight(w_q, w_scale, "w_q");
  TORCH_CHECK(w_q.dim() == 2, "w_q must have shape [N, K]");
  const int st = scale_type(w_scale.scalar_type(), "w_scale");
  const at::Tensor x2 = as_rows(x, "x");
  const int ft = float_type(x2, "x");
  same_device(x2, w_q, "w_q");
  const int64_t M = x2.size(0);
  TORCH_CHECK(x2.size(1) == w.K, "x must have ", w.K, " features, got ", x2.size(1));
  const at::ScalarType dt = default_out(x, out_dtype);
  const int ot = out_type(dt);
  c10::cuda::CUDAGuard guard(x2.device());
  at::Tensor out = fresh({M, w.N}, dt, x2);
  if (M > 0) {
    const int64_t bytes = sk_fp8_linear_workspace_bytes(M, w.K, st);
    at::Tensor ws = fresh({bytes}, at::kByte, x2);     // caching allocator: 512-byte aligned
    check(sk_fp8_linear(M, x2.data_ptr(), ft, pitch(x2), &w, st, out.data_ptr(), w.N, ot, ws.data_ptr(), bytes,
                        at::cuda::getCurrentCUDAStream().stream()),
          "fp8_linear");
  }
  return with_leading_shape(out, x);
}

void check_offsets(const at::Tensor& offsets, const at::Tensor& x, int64_t E) {
  TORCH_CHECK(offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.size(0) == E + 1 && offsets.is_contiguous(),
              "offsets must be a contiguous int32 tensor [experts + 1] = [", E + 1, "]");
  same_device(x, offsets, "offsets");
}

void fp8_grouped_gemm_out(const at::Tensor& x_q, const at::Tensor& x_scale, const at::Tensor& w_q, const at::Tensor& w_scale,
                          const at::Tensor& offsets, at::Tensor& out) {
  const sk_fp8_rows x = fp8_rows(x_q, x_scale, "x");
  const sk_fp8_weight w = fp8_weight(w_q, w_scale, "w_q");
  TORCH_CHECK(w_q.dim() == 3, "w_q must have shape [experts, N, K]");
  const int st = one_scale_type(x_scale, w_scale);
  same_device(x_q, w_q, "w_q");
  check_offsets(offsets, x_q, w.experts);
  const int64_t M = x_q.size(0);
  TORCH_CHECK(w.K == x_q.size(1), "x_q has ", x_q.size(1), " features, w_q ", w.K);
  check_out(out, x_q, M, w.N);
  const int ot = out_type(out.scalar_type());
  if (M == 0) return;
  c10::cuda::CUDAGuard guard(x_q.device());
  check(sk_fp8_grouped_gemm(M, &x, &w, st, offsets.data_ptr<int>(), out.data_ptr(), M == 1 ? w.N : out.stride(0), ot,
                            at::cuda::getCurrentCUDAStream().stream()),
        "fp8_grouped_gemm");
}

at::Tensor fp8_grouped_gemm(const at::Tensor& x_q, const at::Tensor& x_scale, const at::Tensor& w_q, const at::Tensor& w_scale,
                            const at::Tensor& offsets, at::ScalarType out_dtype) {
  out_type(out_dtype);
  TORCH_CHECK(x_q.dim() == 2 && w_q.dim() == 3, "x_q must have shape [M, K] and w_q [experts, N, K]");
  at::Tensor out = fresh({x_q.size(0), w_q.size(1)}, out_dtype, x_q);
  fp8_grouped_gemm_out(x_q, x_scale, w_q, w_scale, offsets, out);
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> route_tokens(const at::Tensor& logits, int64_t k, bool renormalize) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "logits must be a CUDA tensor [T, E]");
  const int ft = float_type(logits, "logits");
  const int64_t T = logits.size(0), E = logits.size(1);
  TORCH_CHECK(E >= 1 && E <= 1024 && k >= 1 && k <= std::min<int64_t>(E, 32), "1 <= k <= min(E, 32) and E <= 1024 are wanted, got k = ", k, ", E = ", E);
  const at::Tensor l = as_rows(logits, "logits");
  c10::cuda::CUDAGuard guard(l.device());
  at::Tensor ids = fresh({T, k}, at::kInt, l), weights = fresh({T, k}, at::kFloat, l), rows = fresh({T, k}, at::kInt, l);
  at::Tensor offsets = fresh({E + 1}, at::kInt, l);
  const int64_t bytes = sk_route_workspace_bytes(T, E);
  at::Tensor ws = bytes > 0 ? fresh({bytes}, at::kByte, l) : offsets;
  // (an empty tensor has no address; nothing is read or written through these when T = 0)
  void* some = offsets.data_ptr();
  check(sk_route_tokens(T ? l.data_ptr() : some, ft, T ? pitch(l) : E, T, E, k, renormalize, static_cast<int*>(T ? ids.data_ptr() : some),
                        static_cast<float*>(T ? weights.data_ptr() : some), static_cast<int*>(T ? rows.data_ptr() : some), offsets.data_ptr<int>(),
                        ws.data_ptr(), bytes, at::cuda::getCurrentCUDAStream().stream()),
        "route_tokens");
  return {ids, weights, rows, offsets};
}

std::tuple<at::Tensor, at::Tensor> group_by_expert(const at::Tensor& ids_in, int64_t E) {
  TORCH_CHECK(ids_in.is_cuda() && ids_in.dim() == 2 && (ids_in.scalar_type() == at::kInt || ids_in.scalar_type() == at::kLong),
              "expert_ids must be a CUDA int32 or int64 tensor [T, k]");
  TORCH_CHECK(E >= 1 && E <= 1024 && ids_in.size(1) >= 1 && ids_in.size(1) <= 1024, "at most 1024 experts and 1 to 1024 choices are taken");
  c10::cuda::CUDAGuard guard(ids_in.device());
  // (64-bit ids are cut to the range that 32 bits hold, so that none wraps into a valid one)
  const at::Tensor ids = (ids_in.scalar_type() == at::kLong ? ids_in.clamp(-1, E).to(at::kInt) : ids_in).contiguous();
  const int64_t T = ids.size(0), k = ids.size(1);
  at::Tensor rows = fresh({T, k}, at::kInt, ids), offsets = fresh({E + 1}, at::kInt, ids);
  const int64_t bytes = sk_route_workspace_bytes(T, E);
  at::Tensor ws = bytes > 0 ? fresh({bytes}, at::kByte, ids) : offsets;
  void* some = offsets.data_ptr();
  check(sk_group_by_expert(static_cast<const int*>(T ? ids.data_ptr() : some), T, k, E, static_cast<int*>(T ? rows.data_ptr() : some),
                           offsets.data_ptr<int>(), ws.data_ptr(), bytes, at::cuda::getCurrentCUDAStream().stream()),
        "group_by_expert");
  return {rows, offsets};
}

at::Tensor fp8_experts(const at::Tensor& x, const at::Tensor& rows, const at::Tensor& weights, const at::Tensor& offsets, const at::Tensor& gate_up,
                       const at::Tensor& gate_up_scale, const at::Tensor& down, const at::Tensor& down_scale, c10::optional<at::ScalarType> out_dtype) {
  TORCH_CHECK(gate_up.dim() == 4 && gate_up.size(1) == 2 && down.dim() == 3, "gate_up must have shape [experts, 2, inter, hidden] and down [experts, hidden, inter]");
  const sk_fp8_weight gu = fp8_weight(gate_up, gate_up_scale, "gate_up"), dn = fp8_weight(down, down_scale, "down");
  TORCH_CHECK(gate_up.size(0) == down.size(0) && gu.N == dn.K && gu.K == dn.N, "gate_up ", gate_up.sizes(), " and down ", down.sizes(),
              " do not belong together");
  const int st = one_scale_type(gate_up_scale, down_scale);
  const at::Tensor x2 = as_rows(x, "x");
  const int ft = float_type(x2, "x");
  const int64_t T = x2.size(0);
  TORCH_CHECK(x2.size(1) == gu.K, "x must have ", gu.K, " features, got ", x2.size(1));
  same_device(x2, gate_up, "gate_up");
  same_device(x2, down, "down");
  TORCH_CHECK(rows.dim() == 2 && rows.size(0) == T && rows.size(1) >= 1 && rows.scalar_type() == at::kInt && rows.is_contiguous(),
              "rows must be a contiguous int32 tensor [tokens, k]");
  TORCH_CHECK(weights.sizes() == rows.sizes() && weights.scalar_type() == at::kFloat && weights.is_contiguous(),
              "weights must be a contiguous float32 tensor like rows");
  same_device(x2, rows, "rows");
  same_device(x2, weights, "weights");
  check_offsets(offsets, x2, dn.experts);
  const int64_t k = rows.size(1);
  const at::ScalarType dt = default_out(x, out_dtype);
  const int ot = out_type(dt);
  c10::cuda::CUDAGuard guard(x2.device());
  at::Tensor out = fresh({T, gu.K}, dt, x2);
  if (T > 0) {
    const int64_t bytes = sk_fp8_experts_workspace_bytes(T, k, gu.K, gu.N, st);
    at::Tensor ws = fresh({bytes}, at::kByte, x2);
    check(sk_fp8_experts(T, k, x2.data_ptr(), ft, pitch(x2), rows.data_ptr<int>(), weights.data_ptr<float>(), offsets.data_ptr<int>(), &gu, &dn, st,
                         out.data_ptr(), gu.K, ot, ws.data_ptr(), bytes, at::cuda::getCurrentCUDAStream().stream()),
          "fp8_experts");
  }
  return with_leading_shape(out, x);
}

int64_t fp8_device_status(int64_t device) {
  int v = 0;
  const int rc = sk_fp8_last_device_status(static_cast<int>(device), &v);
  TORCH_CHECK(rc == SK_OK || rc == SK_ERR_DEVICE_TIMEOUT, "slimkernels::fp8_device_status failed: ", sk_status_string(rc));
  return v;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(slimkernels, m) {
  m.def("quantize_fp8(Tensor x, ScalarType scale_dtype) -> (Tensor, Tensor)", &quantize_fp8);
  m.def("prepare_weight_fp8(Tensor w, ScalarType scale_dtype) -> (Tensor, Tensor)", &prepare_weight_fp8);
  m.def("fp8_gemm(Tensor x_q, Tensor x_scale, Tensor w_q, Tensor w_scale, ScalarType out_dtype) -> Tensor", &fp8_gemm);
  m.def("fp8_gemm_out(Tensor x_q, Tensor x_scale, Tensor w_q, Tensor w_scale, Tensor(a!) out) -> ()", &fp8_gemm_out);
  m.def("fp8_linear(Tensor x, Tensor w_q, Tensor w_scale, ScalarType? out_dtype=None) -> Tensor", &fp8_linear);
  m.def("fp8_grouped_gemm(Tensor x_q, Tensor x_scale, Tensor w_q, Tensor w_scale, Tensor offsets, ScalarType out_dtype) -> Tensor", &fp8_grouped_gemm);
  m.def("fp8_grouped_gemm_out(Tensor x_q, Tensor x_scale, Tensor w_q, Tensor w_scale, Tensor offsets, Tensor(a!) out) -> ()", &fp8_grouped_gemm_out);
  m.def("route_tokens(Tensor logits, int k, bool renormalize) -> (Tensor, Tensor, Tensor, Tensor)", &route_tokens);
  m.def("group_by_expert(Tensor expert_ids, int experts) -> (Tensor, Tensor)", &group_by_expert);
  m.def("fp8_experts(Tensor x, Tensor rows, Tensor weights, Tensor offsets, Tensor gate_up, Tensor gate_up_scale, Tensor down, Tensor down_scale, ScalarType? out_dtype=None) -> Tensor", &fp8_experts);
  m.def("fp8_device_status(int device) -> int", &fp8_device_status);
}
