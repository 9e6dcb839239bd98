"""Which layers `quantize_linears` sends to 8-bit floats; the conversions themselves, which need a GPU, are stand-ins."""
import pytest
import torch
from torch import nn

from slimkernels_b200.torch import convert


class _Made(nn.Module):
    def __init__(self, kind):
        super().__init__()
        self.kind = kind


@pytest.fixture(autouse=True)
def stand_ins(monkeypatch):
    for name, kind in (("FP8Linear", "8-bit"), ("W2A8Linear", "2-bit"), ("FP8Experts", "experts")):
        monkeypatch.setattr(getattr(convert, name), "from_float", classmethod(lambda cls, *a, kind=kind, **k: _Made(kind)))
    monkeypatch.setattr(convert, "W2A8LlamaMLP", lambda gate_up, down: _Made("mlp"))


class _MLP(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj = (nn.Linear(*s, bias=False) for s in ((128, 256), (128, 256), (256, 128)))
        self.act_fn = nn.SiLU()


class _Layer(nn.Module):
    def __init__(self):
        super().__init__()
        self.q_proj, self.mlp = nn.Linear(128, 128, bias=False), _MLP()


class _Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.layers, self.lm_head = nn.ModuleList(_Layer() for _ in range(2)), nn.Linear(128, 32)


def _kinds(model):
    return {n: m.kind for n, m in model.named_modules() if isinstance(m, _Made)}


def test_without_names_the_block_is_fused():
    m = _Model()
    assert convert.quantize_linears(m) == {"linear": 2, "mlp": 2, "kept": ["lm_head"]}
    assert _kinds(m) == {"layers.0.q_proj": "2-bit", "layers.0.mlp": "mlp", "layers.1.q_proj": "2-bit", "layers.1.mlp": "mlp"}


@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj"])
def test_a_named_projection_of_a_block_is_not_fused_away(name):
    m = _Model()
    stats = convert.quantize_linears(m, fp8=(name, "lm_head"))
    assert stats == {"linear": 6, "mlp": 0, "kept": [], "fp8": 3}
    kinds = _kinds(m)
    assert kinds["lm_head"] == "8-bit"
    for i in (0, 1):
        for n in ("gate_proj", "up_proj", "down_proj"):
            assert kinds[f"layers.{i}.mlp.{n}"] == ("8-bit" if n == name else "2-bit")


def test_a_full_name_opens_one_block_only():
    m = _Model()
    stats = convert.quantize_linears(m, fp8=("layers.1.mlp.down_proj",))
    assert stats == {"linear": 4, "mlp": 1, "kept": ["lm_head"], "fp8": 1}
    kinds = _kinds(m)
    assert kinds["layers.0.mlp"] == "mlp" and kinds["layers.1.mlp.down_proj"] == "8-bit" and kinds["layers.1.mlp.up_proj"] == "2-bit"


def test_names_below_a_skipped_module_are_converted():
    m = _Model()
    stats = convert.quantize_linears(m, skip=("mlp", "lm_head"), fp8=("down_proj",))
    assert stats == {"linear": 2, "mlp": 0, "kept": ["layers.0.mlp", "layers.1.mlp", "lm_head"], "fp8": 2}
    assert _kinds(m) == {f"layers.{i}.{n}": kind for i in (0, 1) for n, kind in (("q_proj", "2-bit"), ("mlp.down_proj", "8-bit"))}


def test_a_skipped_module_is_left_alone_otherwise():
    m = _Model()
    m.layers[0].mlp.gate_up_proj, m.layers[0].mlp.down = nn.Parameter(torch.zeros(2, 8, 4)), nn.Linear(128, 128)
    convert.quantize_linears(m, skip=("layers", "lm_head"), fp8=("layers.1.q_proj",), experts=True)
    assert _kinds(m) == {"layers.1.q_proj": "8-bit"}


@pytest.mark.parametrize("names", [("lm_haed",), ("lm_head", "layers.2.q_proj"), ("mlp",), ("embed",)])
def test_names_of_no_linear_layer_are_refused_before_anything_is_converted(names):
    m = _Model()
    with pytest.raises(ValueError, match=names[-1]):
        convert.quantize_linears(m, fp8=names)
    assert _kinds(m) == {}


def test_one_name_may_stand_alone():
    m = _Model()
    m.head = nn.Linear(100, 8)                              # (its name is a part of the other's)
    stats = convert.quantize_linears(m, fp8="lm_head")
    assert stats["fp8"] == 1 and _kinds(m)["lm_head"] == "8-bit" and stats["kept"] == ["head"]


def test_a_layer_that_is_converted_already_keeps_its_name():
    m = _Model()
    m.lm_head = convert.FP8Linear(torch.zeros(32, 128, dtype=torch.float8_e4m3fn), torch.ones(1, 1), 128)
    assert convert.quantize_linears(m, fp8=("lm_head",))["fp8"] == 0 and isinstance(m.lm_head, convert.FP8Linear)
