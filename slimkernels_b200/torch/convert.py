"""Swap the `nn.Linear` layers of a model for W2A8 layers.

The reference's torch directory wraps a Hugging Face causal LM for `generate` (slimkernels/torch/llama.py:4-47) and
stops there; this is the step it was heading towards: every linear projection of the loaded model is quantised with
the reference's own rule (quantize_to_uint2 + pack_matrix, run on the GPU) and replaced by a module that calls the
W2A8 GEMM.  Llama-style MLP blocks (gate_proj / up_proj / down_proj with SiLU) become one fused `W2A8LlamaMLP`
(gate and up share a GEMM; SiLU * up and the int8 re-quantisation are one kernel).  Layers that 2 bits do not suit, and the stacked
expert weights of mixture-of-experts blocks, can go to 8-bit floats instead.
"""
from __future__ import annotations

import torch
from torch import nn

from .fp8 import FP8Experts, FP8Linear
from .modules import W2A8Linear, W2A8LlamaMLP


class _W2A8LinearWithBias(nn.Module):
    def __init__(self, linear: W2A8Linear, bias: torch.Tensor):
        super().__init__()
        self.linear = linear
        self.register_buffer("bias", bias.detach().to(torch.float16))

    def forward(self, x):
        return self.linear(x) + self.bias


def _convertible(linear: nn.Linear, group_size: int) -> bool:
    return linear.in_features % group_size == 0 and linear.in_features % 32 == 0


_MLP_NAMES = ("gate_proj", "up_proj", "down_proj")


def _is_llama_mlp(module: nn.Module) -> bool:
    if not all(isinstance(getattr(module, n, None), nn.Linear) for n in _MLP_NAMES):
        return False
    if any(getattr(module, n).bias is not None for n in _MLP_NAMES):
        return False
    return _is_silu(getattr(module, "act_fn", None))


def _is_silu(act) -> bool:
    return isinstance(act, nn.SiLU) or type(act).__name__ in ("SiLU", "SiLUActivation")


def _is_experts(module: nn.Module) -> bool:
    """Stacked experts: parameters gate_up_proj [E, 2 * inter, hidden] (gate rows first) and down_proj [E, hidden, inter], SiLU, no biases;
    called with (hidden_states, top_k_index, top_k_weights)."""
    gate_up, down = getattr(module, "gate_up_proj", None), getattr(module, "down_proj", None)
    if not all(isinstance(w, nn.Parameter) and w.dim() == 3 for w in (gate_up, down)):
        return False
    E, hidden, inter = down.shape
    if tuple(gate_up.shape) != (E, 2 * inter, hidden) or E > 1024 or len(list(module.parameters(recurse=False))) != 2:
        return False
    return _is_silu(getattr(module, "act_fn", None))


def _out_dtype(weight):
    return weight.dtype if weight.dtype in (torch.float16, torch.bfloat16) else torch.float16


def quantize_linears(model: nn.Module, group_size: int = 128, skip=("lm_head",), fuse_mlp: bool = True,
                     device=None, fp8=(), experts: bool = False) -> dict:
    """Replace, in place, every `nn.Linear` whose in_features is a multiple of `group_size` (except names in `skip`).

    fp8: names of `nn.Linear` layers that become `FP8Linear` instead, whatever `skip` says (fp8=("lm_head",) for the output head).  An MLP
    block with a layer among them is not fused, and of a module that `skip` names they alone are converted (it counts as kept).  A name that
    fits no layer is an error.
    experts: stacked expert weights (see _is_experts) become `FP8Experts`.

    Returns {"linear": n, "mlp": n, "kept": [names left as they were]}, with `fp8` or `experts` also their numbers.  The model must be on
    a CUDA device (or `device` given): quantisation runs there.
    """
    fp8 = (fp8,) if isinstance(fp8, str) else tuple(fp8)
    linears = [full for full, m in model.named_modules(remove_duplicate=False) if isinstance(m, (nn.Linear, FP8Linear))]
    unknown = [n for n in fp8 if not any(n in (full, full.rpartition(".")[2]) for full in linears)]
    if unknown:
        raise ValueError(f"fp8 names layers that are no nn.Linear of this model: {unknown}")
    stats = {"linear": 0, "mlp": 0, "kept": []}
    if fp8:
        stats["fp8"] = 0
    if experts:
        stats["experts"] = 0

    def in_fp8(name, full):
        return name in fp8 or full in fp8

    def dev_of(linear):
        return device if device is not None else linear.weight.device

    def convert(linear: nn.Linear):
        q = W2A8Linear.from_float(linear.weight, group_size, device=dev_of(linear))
        return q if linear.bias is None else _W2A8LinearWithBias(q, linear.bias.to(dev_of(linear)))

    def walk(parent: nn.Module, prefix: str, skipped: bool = False):
        for name, child in list(parent.named_children()):
            full = f"{prefix}{name}"
            if isinstance(child, nn.Linear) and in_fp8(name, full):
                setattr(parent, name, FP8Linear.from_float(child.weight, child.bias, dev_of(child), _out_dtype(child.weight)))
                stats["fp8"] += 1
                continue
            if skipped or name in skip or full in skip:
                if not skipped:
                    stats["kept"].append(full)
                walk(child, full + ".", True)
                continue
            if fuse_mlp and _is_llama_mlp(child) and _convertible(child.gate_proj, group_size) \
                    and _convertible(child.down_proj, group_size) and not any(in_fp8(n, f"{full}.{n}") for n in _MLP_NAMES):
                gate_up = torch.cat([child.gate_proj.weight, child.up_proj.weight], dim=0)   # gate rows first
                fused = W2A8LlamaMLP(W2A8Linear.from_float(gate_up, group_size, device=dev_of(child.gate_proj)),
                                     W2A8Linear.from_float(child.down_proj.weight, group_size,
                                                           device=dev_of(child.down_proj)))
                setattr(parent, name, fused)
                stats["mlp"] += 1
            elif isinstance(child, nn.Linear):
                if _convertible(child, group_size):
                    setattr(parent, name, convert(child))
                    stats["linear"] += 1
                else:
                    stats["kept"].append(full)
            elif experts and _is_experts(child):
                setattr(parent, name, FP8Experts.from_float(child.gate_up_proj, child.down_proj,
                                                            device if device is not None else child.down_proj.device, _out_dtype(child.down_proj)))
                stats["experts"] += 1
            else:
                walk(child, full + ".")

    walk(model, "")
    return stats
