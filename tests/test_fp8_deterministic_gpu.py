"""torch's deterministic mode fills what nothing writes."""
import pytest
import torch

import fp8_util as F
import slimkernels_b200.torch as sk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


@pytest.mark.parametrize("scales", [torch.float8_e8m0fnu, torch.float32])
def test_rows_of_no_group_in_a_fresh_result_are_filled(scales):
    g = F.generator(1)
    x = sk.quantize_fp8(F.random_rows(g, 40, 256), scales)
    w = sk.prepare_weight_fp8(torch.randn(2, 100, 256, generator=g, device="cuda"), scales)
    offsets = torch.tensor([3, 10, 30], dtype=torch.int32, device="cuda")
    want = sk.fp8_grouped_gemm(*x, *w, offsets)[3:30].clone()
    assert torch.are_deterministic_algorithms_enabled() is False and torch.utils.deterministic.fill_uninitialized_memory
    torch.empty(40, 100, dtype=torch.bfloat16, device="cuda").zero_()       # (what the allocator hands out next)
    torch.use_deterministic_algorithms(True)
    try:
        y = sk.fp8_grouped_gemm(*x, *w, offsets)
    finally:
        torch.use_deterministic_algorithms(False)
    assert torch.equal(y[3:30], want)
    assert bool(torch.isnan(y[:3]).all()) and bool(torch.isnan(y[30:]).all())


@pytest.mark.parametrize("scales", [torch.float8_e8m0fnu, torch.float32])
def test_every_operator_in_deterministic_mode(scales):
    g = F.generator(2)
    x, weight = F.random_rows(g, 20, 200, torch.bfloat16), torch.randn(3, 2, 72, 200, generator=g, device="cuda")
    logits = torch.randn(20, 3, generator=g, device="cuda")

    def run():
        q, s = sk.quantize_fp8(x, scales)
        gu, dn = sk.prepare_weight_fp8(weight, scales), sk.prepare_weight_fp8(weight[:, 0].transpose(1, 2), scales)
        r = sk.route_tokens(logits, 2)
        rows, offsets = sk.group_by_expert(r.expert_ids, 3)
        one = gu[0][0, 0], gu[1][0, 0]
        bits = lambda t: t.contiguous().view(torch.uint8)      # noqa: E731
        return [bits(q), bits(s), *map(bits, gu), *map(bits, dn), *r, rows, offsets, sk.fp8_gemm(q, s, *one), sk.fp8_linear(x, *one),
                sk.fp8_experts(x, r, *gu, *dn)]

    want = run()
    torch.use_deterministic_algorithms(True)
    try:
        got = run()
    finally:
        torch.use_deterministic_algorithms(False)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
