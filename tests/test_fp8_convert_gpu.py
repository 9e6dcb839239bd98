"""Models whose MLP blocks keep one projection in 8-bit floats."""
import copy

import pytest
import torch
from torch import nn

import slimkernels_b200.torch as sk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


class _MLP(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj = (nn.Linear(*s, bias=False) for s in ((128, 256), (128, 256), (256, 128)))
        self.act_fn = nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj"])
def test_one_projection_in_8_bits(name, dtype):
    torch.manual_seed(5)
    model = nn.ModuleDict({"mlp": _MLP(), "skipped": _MLP()}).cuda().to(dtype).eval()
    plain = copy.deepcopy(model)
    stats = sk.quantize_linears(model, skip=("skipped",), fp8=(name,))
    assert stats == {"linear": 2, "mlp": 0, "kept": ["skipped"], "fp8": 2}
    x = torch.randn(9, 128, device="cuda").to(dtype)

    def layer(mlp, n):
        weight = getattr(mlp, n).weight
        if n == name:
            w = sk.prepare_weight_fp8(weight)
            return lambda t: sk.fp8_linear(t, *w, dtype)
        return sk.W2A8Linear.from_float(weight) if mlp is plain["mlp"] else getattr(mlp, n)

    with torch.no_grad():
        for key in ("mlp", "skipped"):
            gate, up, down = (layer(plain[key], n) for n in ("gate_proj", "up_proj", "down_proj"))
            h = plain[key].act_fn(gate(x)) * up(x)
            want = down(h)
            got = model[key](x)
            assert torch.equal(got, want) and bool(torch.isfinite(got).all())
            assert isinstance(getattr(model[key], name), sk.FP8Linear)
    assert type(model["skipped"].down_proj) is (sk.FP8Linear if name == "down_proj" else nn.Linear)


class _Experts(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate_up_proj, self.down_proj, self.act_fn = nn.Parameter(torch.randn(3, 96, 64)), nn.Parameter(torch.randn(3, 64, 48)), nn.SiLU()


def test_weights_of_other_float_types_are_taken_as_by_the_2_bit_layers():
    torch.manual_seed(6)
    model = nn.ModuleDict({"experts": _Experts(), "head": nn.Linear(128, 40), "proj": nn.Linear(128, 40)}).cuda().double()
    plain = copy.deepcopy(model).float()
    assert sk.quantize_linears(model, fp8=("head",), experts=True) == {"linear": 1, "mlp": 0, "kept": [], "fp8": 1, "experts": 1}
    same = sk.FP8Linear.from_float(plain["head"].weight, plain["head"].bias)
    for n in ("w_q", "w_scale", "bias"):
        a, b = getattr(model["head"], n), getattr(same, n)
        assert a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    same = sk.FP8Experts.from_float(plain["experts"].gate_up_proj, plain["experts"].down_proj)
    assert all(torch.equal(getattr(model["experts"], n).view(torch.uint8), getattr(same, n).view(torch.uint8)) for n in same._as_they_are)
