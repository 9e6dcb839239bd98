"""FP8Linear, FP8Experts and quantize_linears with them, on models that call them as theirs."""
import copy

import pytest
import torch
from torch import nn

import fp8_util as F
import slimkernels_b200.torch as sk

pytestmark = pytest.mark.gpu
E8M0, F32 = torch.float8_e8m0fnu, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


@pytest.mark.parametrize("scales", [E8M0, F32])
@pytest.mark.parametrize("N,K,bias", [(130, 256, True), (64, 100, False), (257, 1000, True)])
def test_linear_module(N, K, bias, scales):
    torch.manual_seed(N)
    lin = nn.Linear(K, N, bias=bias).cuda().to(torch.bfloat16)
    q = sk.FP8Linear.from_float(lin.weight, lin.bias, out_dtype=torch.bfloat16, scale_dtype=scales)
    x = F.random_rows(F.generator(1), 12, K, torch.bfloat16).view(3, 4, K)
    y = q(x)
    wv, _, _ = F.quantise(lin.weight.detach(), 128)
    codes, scale = sk.prepare_weight_fp8(lin.weight, scales)
    exact, tol = F.product_tolerance(F.quantised_values(x.view(12, K)), F.weight_values(codes, scale), torch.bfloat16)
    assert torch.equal(codes.double(), wv)
    if bias:                                                # the product is rounded, then the sum
        b = lin.bias.detach().double()
        exact = exact + b
        tol = tol + F.HALF_STEP[torch.bfloat16] * (exact.abs() + tol)
    F.assert_within(y.view(12, N), exact, tol)
    # buffers: a state dict and a move carry the layer
    again = sk.FP8Linear(torch.zeros_like(q.w_q), torch.ones_like(q.w_scale), K, None if q.bias is None else torch.zeros_like(q.bias), torch.bfloat16)
    again.load_state_dict(q.state_dict())
    assert torch.equal(again(x), y) and torch.equal(copy.deepcopy(q).cpu().cuda()(x), y)


class _Experts(nn.Module):
    """Stacked experts, called with the router's choices."""

    def __init__(self, E, hidden, inter):
        super().__init__()
        self.gate_up_proj = nn.Parameter(torch.randn(E, 2 * inter, hidden) * hidden ** -0.5)
        self.down_proj = nn.Parameter(torch.randn(E, hidden, inter) * inter ** -0.5)
        self.act_fn = nn.SiLU()

    def forward(self, hidden_states, top_k_index, top_k_weights):
        out = torch.zeros_like(hidden_states)
        for t in range(hidden_states.shape[0]):
            for e, w in zip(top_k_index[t].tolist(), top_k_weights[t]):
                gate, up = (self.gate_up_proj[e] @ hidden_states[t]).chunk(2)
                out[t] += w * (self.down_proj[e] @ (self.act_fn(gate) * up))
        return out


class _Block(nn.Module):
    def __init__(self, E, k, hidden, inter):
        super().__init__()
        self.gate, self.experts, self.k = nn.Linear(hidden, E, bias=False), _Experts(E, hidden, inter), k

    def forward(self, x):
        w, i = self.gate(x).float().softmax(-1).topk(self.k)
        return self.experts(x, i, (w / w.sum(-1, keepdim=True)).to(x.dtype))


class _Model(nn.Module):
    def __init__(self, hidden=144, inter=200):
        super().__init__()
        self.moe, self.lm_head = _Block(6, 2, hidden, inter), nn.Linear(hidden, 50, bias=False)

    def forward(self, x):
        return self.lm_head(x + self.moe(x))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_models_with_experts_and_an_8_bit_head(dtype):
    torch.manual_seed(3)
    model = _Model().cuda().to(dtype).eval()
    ref = copy.deepcopy(model).double()
    stats = sk.quantize_linears(model, skip=("lm_head", "gate"), fp8=("lm_head",), experts=True)
    assert stats == {"linear": 0, "mlp": 0, "kept": ["moe.gate"], "fp8": 1, "experts": 1}
    assert isinstance(model.moe.experts, sk.FP8Experts) and isinstance(model.lm_head, sk.FP8Linear)
    x = torch.randn(40, 144, device="cuda").to(dtype)
    with torch.no_grad():
        y, want = model(x), ref(x.double())
    # e4m3 codes are off by half a step of 2^-3 at most, a uniform error of 2^-4 / sqrt(3) = 3.6 % of a value at most; two operands per
    # product and three products on the longest way: sqrt(6) * 3.6 % = 9 %, if every code were as far off as it may be
    assert (y.double() - want).norm() <= 0.09 * want.norm()
    assert y.dtype == (dtype if dtype != torch.float32 else torch.float16)


def test_experts_module_is_the_operator():
    torch.manual_seed(4)
    e = _Experts(5, 100, 72).cuda().to(torch.bfloat16)
    for scales in (E8M0, F32):
        m = sk.FP8Experts.from_float(e.gate_up_proj, e.down_proj, out_dtype=torch.bfloat16, scale_dtype=scales)
        x = torch.randn(9, 100, device="cuda").to(torch.bfloat16)
        routing = sk.route_tokens(torch.randn(9, 5, device="cuda"), 3)
        y = m.forward_routed(x, routing)
        gu = sk.prepare_weight_fp8(e.gate_up_proj.reshape(5, 2, 72, 100), scales)
        dn = sk.prepare_weight_fp8(e.down_proj, scales)
        assert torch.equal(y, sk.fp8_experts(x, routing, *gu, *dn))
        assert torch.equal(y, m(x, routing.expert_ids.long(), routing.weights))
        again = copy.deepcopy(m).cpu()
        again.load_state_dict(m.state_dict())
        assert torch.equal(again.cuda().forward_routed(x, routing), y)
    with pytest.raises(ValueError):
        sk.FP8Experts.from_float(e.gate_up_proj[:, :100], e.down_proj)


def test_what_is_no_stack_of_experts_is_left_alone():
    model = _Model().cuda()
    model.moe.experts.act_fn = nn.GELU()
    assert sk.quantize_linears(model, skip=("lm_head", "gate"), experts=True) == {"linear": 0, "mlp": 0, "kept": ["moe.gate", "lm_head"], "experts": 0}
    assert isinstance(model.moe.experts, _Experts)



@pytest.mark.parametrize("scales", [E8M0, F32])
def test_casts_of_a_model_leave_codes_and_scales_alone(scales):
    torch.manual_seed(6)
    lin = sk.FP8Linear.from_float(torch.randn(130, 200), torch.randn(130), out_dtype=torch.bfloat16, scale_dtype=scales)
    experts = sk.FP8Experts.from_float(torch.randn(3, 96, 64), torch.randn(3, 64, 48), scale_dtype=scales)
    x, z = torch.randn(7, 200, device="cuda"), torch.randn(7, 64, device="cuda")
    ids, weights = torch.randint(0, 3, (7, 2), device="cuda"), torch.rand(7, 2, device="cuda")
    plain = sk.fp8_linear(x, lin.w_q[:, :200], lin.w_scale, torch.bfloat16)
    want = experts(z, ids, weights)
    for cast in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.cpu().to("cuda", torch.float16)):
        a, b = cast(copy.deepcopy(lin)), cast(copy.deepcopy(experts))
        for name in ("w_q", "w_scale"):
            t, u = getattr(a, name), getattr(lin, name)
            assert t.dtype == u.dtype and t.is_cuda and torch.equal(t.view(torch.uint8), u.view(torch.uint8))
        assert torch.equal(a(x), plain + a.bias.to(torch.bfloat16)) and a(x).dtype == torch.bfloat16
        assert torch.equal(b(z, ids, weights), want)
    assert list(lin.state_dict()) == ["w_q", "w_scale", "bias"] and list(experts.half().state_dict()) == ["gate_up", "gate_up_scale", "down", "down_scale"]
