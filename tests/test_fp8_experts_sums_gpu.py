"""The experts' results of an expert layer are summed in fp32 and rounded once."""
import pytest
import torch

import fp8_util as F
import slimkernels_b200.torch as sk
from slimkernels_b200 import capi
from test_fp8_experts_gpu import _interval_product, _layers, _quantised_interval

pytestmark = pytest.mark.gpu
E8M0, F32 = torch.float8_e8m0fnu, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


@pytest.fixture(params=[0, capi.FP8_FEW, capi.FP8_MANY, capi.FP8_PAIR])
def kernel(request):
    lib = capi.load()
    assert lib.sk_fp8_set_option(capi.SK_FP8_OPT_KERNEL, request.param) == 0
    yield request.param
    lib.sk_fp8_set_option(capi.SK_FP8_OPT_KERNEL, 0)
    assert sk.fp8_device_status() == 0


def _hidden_interval(xv, gu, e):
    """Values between which the codes' values of SiLU(gate) * up lie: gate and up are off by their accumulation, SiLU by 8 units."""
    g, dg = F.product_tolerance(xv, F.weight_values(gu[0][e, 0], gu[1][e, 0]), None)
    u, du = F.product_tolerance(xv, F.weight_values(gu[0][e, 1], gu[1][e, 1]), None)
    s = g * torch.sigmoid(g)
    h = s * u
    dh = 1.1 * dg * (u.abs() + du) + s.abs() * du + 8 * 2.0 ** -23 * h.abs() + 1e-30
    return _quantised_interval(h - dh, h + dh)


@pytest.mark.parametrize("scales", [E8M0, F32])
@pytest.mark.parametrize("hidden,inter", [(256, 128), (200, 144), (7, 300)])
def test_results_past_the_range_of_fp16_may_be_summed(hidden, inter, scales, kernel):
    """An expert's result reaches 10^6, the weighted sum stays within fp16."""
    T, E, k = 41, 3, 2
    g, gu, dn = _layers(E, hidden, inter, scales, hidden)
    dn = (dn[0], (F.scale_values(dn[1]).float() * 2.0 ** 18).to(dn[1].dtype))
    x = F.random_rows(g, T, hidden, torch.float16)
    ids = torch.stack([torch.randperm(E, generator=g, device="cuda")[:k] for _ in range(T)])
    weights = (torch.rand(T, k, generator=g, device="cuda") - 0.5) * 2.0 ** -8
    rows, offsets = sk.group_by_expert(ids, E)
    y = sk.fp8_experts(x, sk.Routing(None, weights, rows, offsets), *gu, *dn)
    assert y.dtype == torch.float16
    xv = F.quantised_values(x)
    out, tol, largest = torch.zeros(T, hidden, dtype=torch.float64, device="cuda"), 0.0, 0.0
    for j in range(k):
        mid, dy = torch.zeros_like(out), torch.zeros_like(out)
        for e in range(E):
            t = torch.nonzero(ids[:, j] == e).flatten()
            lo, hi = _hidden_interval(xv[t], gu, e)
            w = F.weight_values(dn[0][e], dn[1][e])
            mid[t], rad = _interval_product(lo, hi, w)
            dy[t] = rad + F.sum_roundings(inter) * 2.0 ** -23 * (torch.maximum(lo.abs(), hi.abs()) @ w.abs().T)
        largest = max(largest, float(mid.abs().max()))
        wt = weights[:, j, None].double()
        out += wt * mid
        tol = tol + wt.abs() * (dy + 33 * 2.0 ** -23 * (mid.abs() + dy))
    half = F.HALF_STEP[torch.float16]
    assert largest > 3 * 65504 and float(out.abs().max()) < 60000
    F.assert_within(y, out, tol + half * (out.abs() + tol) + 2.0 ** -25)


@pytest.mark.parametrize("scales", [E8M0, F32])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_small_difference_of_two_experts_survives(dtype, scales, kernel):
    """Two experts that differ in the sign of one column of their second matrix, with weights 1 and -1: what is left is that column's
    share twice.  h has the same codes in both, since the same operations on the same values make it; so beside the interval of the column's
    h only the two accumulations count, 138 * 2^-23 of sum |h w| each, a tenth of a step of the results."""
    T, hidden, inter, column = 50, 256, 128, 37
    g, gu, dn = _layers(1, hidden, inter, scales, 5)
    codes = dn[0].view(torch.uint8).expand(2, -1, -1).contiguous()
    codes[1, :, column] ^= 0x80
    two = lambda t: t.view(torch.uint8).expand(2, *t.shape[1:-1], -1).contiguous().view(t.dtype)      # noqa: E731
    gu, dn = (two(gu[0]), two(gu[1])), (codes.view(torch.float8_e4m3fn), two(dn[1]))
    x = F.random_rows(g, T, hidden, dtype)
    ids = torch.tensor([[0, 1]], device="cuda").expand(T, 2).contiguous()
    weights = torch.tensor([[1.0, -1.0]], device="cuda").expand(T, 2).contiguous()
    rows, offsets = sk.group_by_expert(ids, 2)
    y = sk.fp8_experts(x, sk.Routing(ids, weights, rows, offsets), *gu, *dn)
    lo, hi = _hidden_interval(F.quantised_values(x), gu, 0)
    w = F.weight_values(dn[0][0], dn[1][0])
    out, rad = _interval_product(lo[:, column:column + 1], hi[:, column:column + 1], 2 * w[:, column:column + 1])
    tol = rad + 2 * F.sum_roundings(inter) * 2.0 ** -23 * (torch.maximum(lo.abs(), hi.abs()) @ w.abs().T)
    tol = tol + 2 * 2.0 ** -23 * (out.abs() + tol)
    F.assert_within(y, out, tol + F.HALF_STEP[dtype] * (out.abs() + tol) + 2.0 ** -25)
