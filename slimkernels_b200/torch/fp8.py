"""FP8 products next to the 2-bit ones: for layers that 2-bit weights do not suit (the output head, say) and for
mixture-of-experts layers.  The reference has neither; its kernel prototype feeds e4m3 activations
(slimkernels/cute/gemm/wgmma_sm90_W2A8.cu:533-536).

A tensor is held as e4m3 codes and one scale per block of 128: activations [M, K] have scales [M, ceil(K / 128)], weights [N, K]
scales [ceil(N / 128), ceil(K / 128)].  Scales are float32 (any value, as checkpoints have them) or float8_e8m0fnu (powers of two,
what `quantize_fp8` and `prepare_weight_fp8` make either way); both operands of a product have the same type.  Everything runs
on the current CUDA stream, for inference: nothing is recorded for a backward pass.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import nn

from .ops import load_extension

_ops = {}


def _op(name):
    """The registered op (its only overload: looking that up on every call takes 2 us)."""
    op = _ops.get(name)
    if op is None:
        load_extension()
        op = _ops[name] = getattr(torch.ops.slimkernels, name).default
    return op


def quantize_fp8(x, scale_dtype=torch.float8_e8m0fnu):
    """x [..., K] (float16 / bfloat16 / float32) -> (codes [..., K], scales [..., ceil(K / 128)]).

    Per row and block of 128: a = max|x|, scale = 2^e with the smallest e such that a <= 448 * 2^e (1 for a block of zeros),
    code = x / scale rounded to nearest even.  A block with an infinity or a NaN becomes NaN.  The rows of the codes start on 16
    bytes, as the products want them.
    """
    return _op("quantize_fp8")(x, scale_dtype)


def prepare_weight_fp8(w, scale_dtype=torch.float8_e8m0fnu):
    """w [..., N, K] -> (codes [..., N, K], scales [..., ceil(N / 128), ceil(K / 128)]), by the same rule per 128 x 128 block."""
    return _op("prepare_weight_fp8")(w.detach(), scale_dtype)


def fp8_gemm(x_q, x_scale, w_q, w_scale, out_dtype=torch.bfloat16, out=None):
    """[M, N] = (x_q * x_scale) @ (w_q * w_scale).T, summed in fp32 (a sum over blocks that
    leaves its range is not finite) and rounded once.  `out` may be a column slice."""
    if out is None:
        return _op("fp8_gemm")(x_q, x_scale, w_q, w_scale, out_dtype)
    _op("fp8_gemm_out")(x_q, x_scale, w_q, w_scale, out)
    return out


def fp8_linear(x, w_q, w_scale, out_dtype=None):
    """x [..., K] -> [..., N]: `quantize_fp8` with the weight's type of scales, then `fp8_gemm`.  The result has x's type where that
    has 16 bits, else float16."""
    return _op("fp8_linear")(x, w_q, w_scale, out_dtype)


def fp8_grouped_gemm(x_q, x_scale, w_q, w_scale, offsets, out_dtype=torch.bfloat16, out=None):
    """Rows offsets[e] .. offsets[e + 1] - 1 of x times w[e].T, w [E, N, K], offsets int32 [E + 1] on the GPU, non-decreasing.

    Groups may be empty.  Rows that belong to no group are not written: in a given `out` they keep what they held, in a fresh
    result they hold anything.
    """
    if out is None:
        return _op("fp8_grouped_gemm")(x_q, x_scale, w_q, w_scale, offsets, out_dtype)
    _op("fp8_grouped_gemm_out")(x_q, x_scale, w_q, w_scale, offsets, out)
    return out


class Routing(NamedTuple):
    expert_ids: torch.Tensor     # int32 [T, k], or None where the experts were chosen elsewhere and are no longer needed
    weights: torch.Tensor        # float32 [T, k]
    rows: torch.Tensor           # int32 [T, k]: place of choice (t, j) among all, ordered by expert, then by t * k + j; -1: no expert here
    offsets: torch.Tensor        # int32 [E + 1]: the experts' first places


def route_tokens(logits, k, renormalize=True) -> Routing:
    """The k largest of each token's logits [T, E] (ties: the lower expert) with softmax weights, and the tokens' order by expert.

    renormalize: the weights are divided by the sum of the k chosen (else they are the softmax's over all experts).  A logit of
    -infinity masks an expert: it is chosen after all others and has weight zero; a token with nothing else gets weights of zero.
    NaN or +infinity gives the token NaN weights.  E <= 1024, k <= min(E, 32).
    """
    return Routing(*_op("route_tokens")(logits, k, renormalize))


def group_by_expert(expert_ids, experts: int):
    """(rows, offsets) of a `Routing` for experts [T, k] chosen elsewhere.  Ids outside [0, experts) are nobody's: their rows are -1."""
    return _op("group_by_expert")(expert_ids, experts)


def fp8_experts(x, routing: Routing, gate_up, gate_up_scale, down, down_scale, out_dtype=None):
    """sum_j weights[t, j] * ( down[e] q( SiLU(gate[e] q(x)) * up[e] q(x) ) ), e the expert of choice (t, j), q = `quantize_fp8`.

    x [..., hidden] with T tokens in all, gate_up codes [E, 2, inter, hidden] (gate first), down codes [E, hidden, inter].  Four
    kernels: quantise into the groups' rows, grouped product with SiLU * up and the re-quantisation in its epilogue, grouped
    product, weighted sum.  The experts' results and their sum are fp32, rounded once.
    """
    return _op("fp8_experts")(x, routing.rows, routing.weights, routing.offsets, gate_up, gate_up_scale, down, down_scale, out_dtype)


def fp8_device_status(device=None) -> int:
    """Reads and clears the device's note of a wait inside an FP8 kernel that ran into its limit (0: none).  Waits for all
    streams of the device."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    return _op("fp8_device_status")(torch.cuda.current_device() if index is None else index)


def _padded_codes(w, scale_dtype):
    """Codes whose rows are padded to a multiple of 16, as a whole tensor (what a module keeps: it survives .to() and a state dict)."""
    if w.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        w = w.to(torch.float32)
    codes, scale = prepare_weight_fp8(w, scale_dtype)
    full = codes.as_strided((*codes.shape[:-1], codes.stride(-2)), codes.stride()) if codes.stride(-2) != codes.shape[-1] else codes
    return full, scale


class _KeepsTypes(nn.Module):
    """Codes and scales are moved as they are: `.half()`, `.to(dtype)` and `.type(dtype)` are for what a model computes in, not for them, and
    a memory format is for its images."""

    _as_they_are = ()

    @staticmethod
    def _moved(fn, t):
        flat = t.reshape(-1).view(torch.uint8)          # (one row of bytes: casts of floats and memory formats pass it by)
        moved = fn(flat)
        if moved.dtype != flat.dtype:                   # (`.type(dtype)` casts whatever it meets)
            moved = flat.to(moved.device)
        return moved.view(t.dtype).view(t.shape)

    def _apply(self, fn, recurse=True):
        held = {name: t for name in self._as_they_are if (t := self._buffers.get(name)) is not None}
        for name in held:
            self._buffers[name] = None
        try:
            super()._apply(fn, recurse)
            moved = {name: self._moved(fn, t) for name, t in held.items()}
        except BaseException:
            self._buffers.update(held)
            raise
        self._buffers.update(moved)
        return self


class FP8Linear(_KeepsTypes):
    """y = x W^T (+ bias) with an 8-bit weight and activations quantised on the way.  w_q float8_e4m3fn [out_features, in_features
    padded to a multiple of 16], w_scale [ceil(out / 128), ceil(in / 128)].  The product is rounded to out_dtype, then the sum with the bias, as in
    the 2-bit layers."""

    _as_they_are = ("w_q", "w_scale")

    def __init__(self, w_q, w_scale, in_features, bias=None, out_dtype=torch.float16):
        super().__init__()
        self.register_buffer("w_q", w_q, persistent=True)
        self.register_buffer("w_scale", w_scale, persistent=True)
        self.register_buffer("bias", bias, persistent=True)
        self.in_features, self.out_features, self.out_dtype = int(in_features), w_q.shape[0], out_dtype

    @classmethod
    def from_float(cls, weight_out_in, bias=None, device="cuda", out_dtype=torch.float16, scale_dtype=torch.float8_e8m0fnu):
        w_q, w_scale = _padded_codes(weight_out_in.detach().to(device=device), scale_dtype)
        b = None if bias is None else bias.detach().to(device=device, dtype=out_dtype)
        return cls(w_q, w_scale, weight_out_in.shape[1], b, out_dtype)

    def forward(self, x):
        y = fp8_linear(x, self.w_q[:, :self.in_features], self.w_scale, self.out_dtype)
        return y if self.bias is None else y + self.bias.to(y.dtype)


class FP8Experts(_KeepsTypes):
    """The expert layers of a mixture-of-experts block with 8-bit weights: `fp8_experts` on tokens routed by the caller.

    gate_up [E, 2, inter, hidden padded to 16], down [E, hidden, inter padded to 16] and their scales.
    """

    _as_they_are = ("gate_up", "gate_up_scale", "down", "down_scale")

    def __init__(self, gate_up, gate_up_scale, down, down_scale, hidden, inter, out_dtype=torch.float16):
        super().__init__()
        for name, t in (("gate_up", gate_up), ("gate_up_scale", gate_up_scale), ("down", down), ("down_scale", down_scale)):
            self.register_buffer(name, t, persistent=True)
        self.hidden, self.inter, self.experts, self.out_dtype = int(hidden), int(inter), gate_up.shape[0], out_dtype

    @classmethod
    def from_float(cls, gate_up, down, device="cuda", out_dtype=torch.float16, scale_dtype=torch.float8_e8m0fnu):
        """gate_up [E, 2 * inter, hidden] (gate rows first), down [E, hidden, inter]."""
        E, hidden, inter = down.shape
        if tuple(gate_up.shape) != (E, 2 * inter, hidden):
            raise ValueError(f"gate_up {tuple(gate_up.shape)} and down {tuple(down.shape)} do not belong together")
        gu = _padded_codes(gate_up.detach().to(device=device).reshape(E, 2, inter, hidden), scale_dtype)
        dn = _padded_codes(down.detach().to(device=device), scale_dtype)
        return cls(*gu, *dn, hidden, inter, out_dtype)

    def forward_routed(self, x, routing: Routing):
        return fp8_experts(x, routing, self.gate_up[..., :self.hidden], self.gate_up_scale, self.down[..., :self.inter], self.down_scale, self.out_dtype)

    def forward(self, hidden_states, top_k_index, top_k_weights):
        """Experts and weights [T, k] chosen by the model's own router."""
        rows, offsets = group_by_expert(top_k_index, self.experts)
        return self.forward_routed(hidden_states, Routing(None, top_k_weights.to(torch.float32).contiguous(), rows, offsets))
