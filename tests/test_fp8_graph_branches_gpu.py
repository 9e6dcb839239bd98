"""Captured graphs whose branches meet in front of the FP8 operators: what another branch writes is there, weights and offsets that are read early
among it."""
import pytest
import torch

import fp8_util as F
import slimkernels_b200.torch as sk

pytestmark = pytest.mark.gpu
E8M0, F32 = torch.float8_e8m0fnu, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


@pytest.mark.parametrize("scales", [E8M0, F32])
@pytest.mark.parametrize("M", [4, 300])
def test_weights_made_in_another_branch(M, scales):
    g = F.generator(M)
    N, K = 1024, 2048
    x, w = F.random_rows(g, M, K, torch.bfloat16), torch.randn(N, K, generator=g, device="cuda")
    other = sk.prepare_weight_fp8(torch.randn(N, K, generator=g, device="cuda"), scales)
    held = torch.empty_like(w)
    side = torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            held.copy_(w)                                   # a copy, a kernel of ours that waits for nobody, products of ours
            w_q, w_s = sk.prepare_weight_fp8(held, scales)
            first = sk.fp8_linear(x, w_q, w_s)
        busy = sk.fp8_linear(x, *other)
        main.wait_stream(side)
        y = sk.fp8_linear(x, w_q, w_s)
        z = sk.fp8_gemm(*sk.quantize_fp8(x, scales), w_q, w_s)
        return first, busy, y, z

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in range(12):
        w.copy_(torch.randn(N, K, generator=F.generator(seed), device="cuda"))
        graph.replay()
        want = sk.fp8_linear(x, *sk.prepare_weight_fp8(w, scales))
        assert torch.equal(got[0], want) and torch.equal(got[2], want) and torch.equal(got[3], want)
        assert torch.equal(got[1], sk.fp8_linear(x, *other))


def test_layers_routed_in_another_branch():
    T, E, k, hidden, inter = 40, 8, 2, 256, 128
    g = F.generator(3)
    gu = sk.prepare_weight_fp8(torch.randn(E, 2, inter, hidden, generator=g, device="cuda") * hidden ** -0.5)
    dn = sk.prepare_weight_fp8(torch.randn(E, hidden, inter, generator=g, device="cuda") * inter ** -0.5)
    x, logits = F.random_rows(g, T, hidden, torch.bfloat16), torch.randn(T, E, generator=g, device="cuda")
    side = torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            r = sk.route_tokens(logits, k)
        shared = sk.fp8_linear(x, gu[0][0, 0], gu[1][0, 0])      # (something on the main branch meanwhile)
        main.wait_stream(side)
        return sk.fp8_experts(x, r, *gu, *dn), shared

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = run()
    for seed in range(12):
        logits.copy_(torch.randn(T, E, generator=F.generator(seed), device="cuda"))
        graph.replay()
        assert torch.equal(y, sk.fp8_experts(x, sk.route_tokens(logits, k), *gu, *dn))
