"""The router, the order by expert and the expert layers against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import fp8_util as F
import slimkernels_b200.torch as sk
from slimkernels_b200 import capi

pytestmark = pytest.mark.gpu
E8M0, F32 = torch.float8_e8m0fnu, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


@pytest.fixture(autouse=True)
def _no_wait_expired():
    yield
    assert sk.fp8_device_status() == 0


# ------------------------------------------------------------------------------------------------------------ router
def _check_routing(logits, k, renormalize):
    got = sk.route_tokens(logits, k, renormalize)
    ids, weights, rows, offsets = F.route_reference(logits.double().cpu().numpy(), k, renormalize)
    np.testing.assert_array_equal(got.expert_ids.cpu().numpy(), ids)
    np.testing.assert_array_equal(got.rows.cpu().numpy(), rows)
    np.testing.assert_array_equal(got.offsets.cpu().numpy(), offsets)
    # exp of a difference d: two roundings of d and two units of expf, (|d| + 2) 2^-23 relatively; the sum of at most 1024 positive
    # terms 10 levels and 32 terms deep; the division half a unit
    T, E = logits.shape
    tol = weights * ((60 + 2 + 42 + 2) * 2.0 ** -23) + 1e-38
    w = got.weights.double().cpu().numpy()
    assert np.array_equal(np.isnan(w), np.isnan(weights))
    assert (np.abs(w - weights)[~np.isnan(weights)] <= tol[~np.isnan(weights)]).all()


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k,dtype", [(1, 1, 1, torch.float32), (1, 64, 8, torch.float32), (2, 2, 2, torch.float16), (63, 33, 3, torch.bfloat16),
                                         (64, 60, 4, torch.float32), (65, 128, 8, torch.bfloat16), (300, 8, 8, torch.float32),
                                         (1000, 257, 6, torch.float16), (129, 1000, 32, torch.float32), (5000, 16, 2, torch.bfloat16)])
def test_routing(T, E, k, dtype, renormalize):
    g = F.generator(T + E)
    logits = (torch.randn(T, E, generator=g, device="cuda") * 3).to(dtype)
    if T > 4:
        logits[1] = 0.5                                     # all equal: the lowest experts
        logits[2, ::2] = logits[2, :1].clone()              # many ties
        logits[3] = -logits[3].abs()
        logits[4, 0] = -0.0
    _check_routing(logits, k, renormalize)


@pytest.mark.parametrize("renormalize", [True, False])
def test_routing_of_masked_and_broken_logits(renormalize):
    inf = float("inf")
    logits = torch.randn(8, 40, generator=F.generator(1), device="cuda")
    logits[0, 3:] = -inf                                    # fewer experts than choices
    logits[1] = -inf                                        # none at all
    logits[2, 7] = float("nan")
    logits[3, 9] = inf
    logits[4, :] = -3.4e38
    logits[5, 0], logits[5, 1:] = 3e38, -3e38
    _check_routing(logits, 5, renormalize)
    w = sk.route_tokens(logits, 5, renormalize).weights
    assert bool((w[1] == 0).all()) and bool((w[0, 3:] == 0).all())


def test_routing_of_strided_logits_and_no_tokens():
    wide = torch.randn(70, 100, generator=F.generator(2), device="cuda")
    _check_routing(wide[:, 5:69], 4, True)
    _check_routing(wide[::3, :64], 4, True)
    _check_routing(wide.t()[:64, :70], 4, True)
    r = sk.route_tokens(wide[:0], 4)
    assert r.rows.shape == (0, 4) and r.offsets.tolist() == [0] * 101


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (7, 3, 5), (64, 8, 64), (65, 8, 64), (700, 2, 1024), (3000, 6, 17)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_group_by_expert(T, k, E, dtype):
    ids = torch.randint(-2, E + 2, (T, k), generator=F.generator(T), device="cuda").to(dtype)
    if dtype == torch.int64:
        ids[0, 0] = 2 ** 32                                 # (not expert 0)
    kept = ids.clone()
    rows, offsets = sk.group_by_expert(ids, E)
    want_rows, want_offsets = F.group_reference(ids.cpu().numpy(), E)
    np.testing.assert_array_equal(rows.cpu().numpy(), want_rows)
    np.testing.assert_array_equal(offsets.cpu().numpy(), want_offsets)
    assert torch.equal(ids, kept)


def test_router_refusals():
    logits = torch.zeros(4, 16, device="cuda")
    for call in (lambda: sk.route_tokens(logits, 0), lambda: sk.route_tokens(logits, 17), lambda: sk.route_tokens(logits[0], 2),
                 lambda: sk.route_tokens(logits.double(), 2), lambda: sk.route_tokens(torch.zeros(2, 1025, device="cuda"), 2),
                 lambda: sk.group_by_expert(logits, 16), lambda: sk.group_by_expert(torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 0)):
        with pytest.raises(RuntimeError):
            call()


# ----------------------------------------------------------------------------------------------------- expert layers
def _interval_product(lo, hi, w):
    """Bounds of h @ w.T for lo <= h <= hi."""
    mid, rad = (lo + hi) / 2, (hi - lo) / 2
    return mid @ w.T, rad @ w.abs().T


def _quantised_interval(lo, hi):
    """Values between which every quantisation of a row between lo and hi lies.

    Rounding is monotone for a given scale; the scale's exponent lies between those of the smallest and the largest maximum.
    """
    a_lo = torch.where((lo <= 0) & (hi >= 0), torch.zeros_like(lo), torch.minimum(lo.abs(), hi.abs()))
    a_hi = torch.maximum(lo.abs(), hi.abs())
    R, K = lo.shape
    kb = F.ceil_div(K, 128)
    pad = lambda t: torch.nn.functional.pad(t, (0, kb * 128 - K)).view(R, kb, 128)      # noqa: E731
    ends = [F.block_exponent(pad(a).amax(dim=2)) for a in (a_lo, a_hi)]
    ends[0] = torch.where(pad(a_lo).amax(dim=2) > 0, ends[0], ends[1])
    los, his = [], []
    for e in ends:
        s = F.pow2(e).repeat_interleave(128, dim=1)[:, :K]
        los.append(F.round_e4m3((lo / s).clamp(-448, 448)) * s)
        his.append(F.round_e4m3((hi / s).clamp(-448, 448)) * s)
    return torch.minimum(*los), torch.maximum(*his)


def _check_experts(x, rows, weights, offsets, gu, dn, y):
    """Every output within what the roundings on the way allow: gate and up are off by their accumulation, h by what SiLU makes of that
    and 8 units of its own evaluation, its codes lie between those of the ends of that interval, y is rounded to the output's type."""
    T, k = rows.shape
    xv = F.quantised_values(x.reshape(T, -1))
    rows, offsets, weights = rows.cpu(), offsets.tolist(), weights.double()
    half = F.HALF_STEP[y.dtype]
    out = torch.zeros(T, xv.shape[1], dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    token, choice = torch.nonzero(rows >= 0, as_tuple=True)
    place = rows[token, choice]
    for e in range(len(offsets) - 1):
        mine = (place >= offsets[e]) & (place < offsets[e + 1])
        if not bool(mine.any()):
            continue
        t, j = token[mine].cuda(), choice[mine].cuda()
        g, dg = F.product_tolerance(xv[t], F.weight_values(gu[0][e, 0], gu[1][e, 0]), None)
        u, du = F.product_tolerance(xv[t], F.weight_values(gu[0][e, 1], gu[1][e, 1]), None)
        s = g * torch.sigmoid(g)
        h = s * u
        dh = 1.1 * dg * (u.abs() + du) + s.abs() * du + 8 * 2.0 ** -23 * h.abs() + 1e-30
        lo, hi = _quantised_interval(h - dh, h + dh)
        w = F.weight_values(dn[0][e], dn[1][e])
        mid, rad = _interval_product(lo, hi, w)
        acc = F.sum_roundings(w.shape[1]) * 2.0 ** -23 * (torch.maximum(lo.abs(), hi.abs()) @ w.abs().T)
        dy = rad + acc
        dy = dy + half * (mid.abs() + dy) + 2.0 ** -25
        wt = weights[t, j][:, None]
        out.index_add_(0, t, wt * mid)
        tol.index_add_(0, t, wt.abs() * (dy + 33 * 2.0 ** -23 * (mid.abs() + dy)))
    F.assert_within(y.reshape(T, -1), out, tol + half * (out.abs() + tol) + 2.0 ** -25)


def _layers(E, hidden, inter, scales, seed):
    g = F.generator(seed)
    gu = sk.prepare_weight_fp8(torch.randn(E, 2, inter, hidden, generator=g, device="cuda") * hidden ** -0.5, scales)
    dn = sk.prepare_weight_fp8(torch.randn(E, hidden, inter, generator=g, device="cuda") * inter ** -0.5, scales)
    if scales == F32:
        gu, dn = (gu[0], F.arbitrary_scales(gu[1], g)), (dn[0], F.arbitrary_scales(dn[1], g))
    return g, gu, dn


@pytest.mark.parametrize("T,E,k,hidden,inter,dtype,scales", [
    (1, 1, 1, 16, 16, torch.bfloat16, E8M0), (1, 8, 2, 256, 128, torch.float16, E8M0), (16, 64, 8, 512, 256, torch.bfloat16, E8M0),
    (33, 5, 3, 200, 144, torch.bfloat16, F32), (100, 4, 2, 384, 300, torch.float16, F32), (257, 3, 2, 136, 1000, torch.float16, E8M0),
    (700, 8, 4, 512, 384, torch.bfloat16, E8M0), (40, 2, 2, 7, 130, torch.bfloat16, F32), (64, 200, 1, 128, 64, torch.float32, E8M0)])
def test_expert_layers(T, E, k, hidden, inter, dtype, scales):
    g, gu, dn = _layers(E, hidden, inter, scales, T + E)
    x = F.random_rows(g, T, hidden, dtype)
    routing = sk.route_tokens(torch.randn(T, E, generator=g, device="cuda"), k)
    y = sk.fp8_experts(x, routing, *gu, *dn)
    assert y.shape == (T, hidden) and y.dtype == (torch.bfloat16 if dtype == torch.bfloat16 else torch.float16)
    _check_experts(x, routing.rows, routing.weights, routing.offsets, gu, dn, y)
    assert torch.equal(y, sk.fp8_experts(x, routing, *gu, *dn))


@pytest.mark.parametrize("kernel,row_tile", [(capi.FP8_FEW, 0), (capi.FP8_MANY, 0), (capi.FP8_PAIR, 0)])
@pytest.mark.parametrize("hidden,inter,scales", [(384, 256, E8M0), (144, 300, F32), (272, 144, E8M0), (256, 1111, F32)])
def test_expert_layers_every_kernel(kernel, row_tile, hidden, inter, scales):
    T, E, k = 500, 5, 2
    g, gu, dn = _layers(E, hidden, inter, scales, 21)
    x = F.random_rows(g, T, hidden, torch.bfloat16)
    routing = sk.route_tokens(torch.randn(T, E, generator=g, device="cuda"), k)
    lib = capi.load()
    try:
        assert lib.sk_fp8_set_option(capi.SK_FP8_OPT_KERNEL, kernel) == 0 and lib.sk_fp8_set_option(capi.SK_FP8_OPT_ROW_TILE, row_tile) == 0
        y = sk.fp8_experts(x, routing, *gu, *dn)
    finally:
        lib.sk_fp8_set_option(capi.SK_FP8_OPT_KERNEL, 0)
        lib.sk_fp8_set_option(capi.SK_FP8_OPT_ROW_TILE, 0)
    _check_experts(x, routing.rows, routing.weights, routing.offsets, gu, dn, y)


def test_expert_layers_are_their_parts():
    """The run of operators written out: quantise, order, product, SiLU * up, quantise, product, weighted sum -- the intermediate of the
    fused layers is not rounded to 16 bits, so the parts agree with them within that."""
    T, E, k, hidden, inter = 50, 6, 2, 256, 256
    g, gu, dn = _layers(E, hidden, inter, E8M0, 3)
    x = F.random_rows(g, T, hidden, torch.float16)
    r = sk.route_tokens(torch.randn(T, E, generator=g, device="cuda"), k)
    order = torch.empty(T * k, dtype=torch.long, device="cuda")
    order[r.rows.flatten().long()] = torch.arange(T * k, device="cuda") // k
    x_q, x_s = sk.quantize_fp8(x[order])
    gate = sk.fp8_grouped_gemm(x_q, x_s, gu[0][:, 0].contiguous(), gu[1][:, 0].contiguous(), r.offsets, torch.float16).double()
    up = sk.fp8_grouped_gemm(x_q, x_s, gu[0][:, 1].contiguous(), gu[1][:, 1].contiguous(), r.offsets, torch.float16).double()
    h_q, h_s = sk.quantize_fp8((gate * torch.sigmoid(gate) * up).float())
    y = sk.fp8_grouped_gemm(h_q, h_s, *dn, r.offsets, torch.float16).double()
    want = (r.weights.double()[:, :, None] * y[r.rows.long()]).sum(1)
    got = sk.fp8_experts(x, r, *gu, *dn).double()
    # a code may move by a step of 2^-3 of its value where fp16 rounded gate or up (a few in a hundred do)
    assert (got - want).norm() <= 0.02 * want.norm()


def test_choices_of_experts_that_are_not_here():
    T, E, k, hidden, inter = 30, 4, 3, 128, 200
    g, gu, dn = _layers(E, hidden, inter, E8M0, 5)
    x = F.random_rows(g, T, hidden, torch.bfloat16)
    ids = torch.randint(-1, E + 3, (T, k), generator=g, device="cuda", dtype=torch.int32)
    ids[3] = -1                                             # a token with none
    weights = torch.rand(T, k, generator=g, device="cuda")
    rows, offsets = sk.group_by_expert(ids, E)
    y = sk.fp8_experts(x, sk.Routing(ids, weights, rows, offsets), *gu, *dn)
    _check_experts(x, rows, weights, offsets, gu, dn, y)
    assert bool((y[3] == 0).all())
    rows, offsets = sk.group_by_expert(ids * 0 - 1, E)
    assert bool((sk.fp8_experts(x, sk.Routing(ids, weights, rows, offsets), *gu, *dn) == 0).all())


def test_places_outside_the_rows_count_nothing():
    T, E, k, hidden, inter = 10, 3, 2, 128, 128
    g, gu, dn = _layers(E, hidden, inter, E8M0, 6)
    x = F.random_rows(g, T, hidden, torch.float16)
    r = sk.route_tokens(torch.randn(T, E, generator=g, device="cuda"), k)
    rows = r.rows.clone()
    rows[2, 0], rows[5, 1], rows[6, 0] = T * k, 2 ** 31 - 1, -(2 ** 31)
    y = sk.fp8_experts(x, r._replace(rows=rows), *gu, *dn)
    weights = r.weights.clone()
    weights[2, 0] = weights[5, 1] = weights[6, 0] = 0
    assert torch.equal(y, sk.fp8_experts(x, r._replace(weights=weights), *gu, *dn))


def test_a_broken_token_leaves_the_others_alone():
    T, E, k, hidden, inter = 20, 4, 2, 256, 128
    g, gu, dn = _layers(E, hidden, inter, E8M0, 7)
    x = F.random_rows(g, T, hidden, torch.bfloat16)
    logits = torch.randn(T, E, generator=g, device="cuda")
    routing = sk.route_tokens(logits, k)
    want = sk.fp8_experts(x, routing, *gu, *dn)
    x[4, 3] = float("nan")
    x[9] = float("inf")
    y = sk.fp8_experts(x, routing, *gu, *dn)
    assert bool(torch.isnan(y[4]).all()) and bool(torch.isnan(y[9]).all())
    keep = [t for t in range(T) if t not in (4, 9)]
    assert torch.equal(y[keep], want[keep])


def test_captured_layers_follow_their_inputs():
    T, E, k, hidden, inter = 12, 8, 2, 256, 256
    g, gu, dn = _layers(E, hidden, inter, E8M0, 9)
    x = F.random_rows(g, T, hidden, torch.bfloat16)
    logits = torch.randn(T, E, generator=g, device="cuda")
    run = lambda: sk.fp8_experts(x.view(3, 4, hidden), sk.route_tokens(logits, k), *gu, *dn)      # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    assert y.shape == (3, 4, hidden)
    for seed in (1, 2, 3):
        x.copy_(F.random_rows(F.generator(seed), T, hidden, torch.bfloat16))
        logits.copy_(torch.randn(T, E, generator=F.generator(seed + 10), device="cuda"))
        graph.replay()
        assert torch.equal(y, run())


def test_one_expert_twice_and_very_many_choices():
    T, E, hidden, inter = 9, 3, 128, 144
    g, gu, dn = _layers(E, hidden, inter, E8M0, 11)
    x = F.random_rows(g, T, hidden, torch.bfloat16)
    for k in (2, 40):                                       # (more choices than there are experts, and than a warp has lanes)
        ids = torch.randint(0, E, (T, k), generator=g, device="cuda")
        ids[:, 1] = ids[:, 0]
        weights = torch.rand(T, k, generator=g, device="cuda")
        rows, offsets = sk.group_by_expert(ids, E)
        y = sk.fp8_experts(x, sk.Routing(None, weights, rows, offsets), *gu, *dn)
        _check_experts(x, rows, weights, offsets, gu, dn, y)


def test_as_many_experts_as_there_may_be():
    T, E, hidden, inter = 70, 1024, 128, 128
    for scales in (E8M0, F32):
        g, gu, dn = _layers(E, hidden, inter, scales, 12)
        x = F.random_rows(g, T, hidden, torch.float16)
        routing = sk.route_tokens(torch.randn(T, E, generator=g, device="cuda"), 32)
        _check_experts(x, routing.rows, routing.weights, routing.offsets, gu, dn, sk.fp8_experts(x, routing, *gu, *dn))


def test_all_tokens_to_one_expert():
    T, E, hidden, inter = 600, 64, 256, 128
    for scales in (E8M0, F32):
        g, gu, dn = _layers(E, hidden, inter, scales, 13)
        x = F.random_rows(g, T, hidden, torch.bfloat16)
        logits = torch.full((T, E), float("-inf"), device="cuda")
        logits[:, 63] = torch.randn(T, generator=g, device="cuda")
        routing = sk.route_tokens(logits, 1)
        assert routing.offsets.tolist() == [0] * 64 + [T]
        _check_experts(x, routing.rows, routing.weights, routing.offsets, gu, dn, sk.fp8_experts(x, routing, *gu, *dn))


def test_layers_on_two_streams_at_once():
    T, E, k, hidden, inter = 40, 8, 2, 512, 256
    sets = []
    for seed in (1, 2):
        g, gu, dn = _layers(E, hidden, inter, E8M0, seed)
        sets.append((F.random_rows(g, T, hidden, torch.bfloat16), torch.randn(T, E, generator=g, device="cuda"), gu, dn))
    run = lambda x, logits, gu, dn: sk.fp8_experts(x, sk.route_tokens(logits, k), *gu, *dn)      # noqa: E731
    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in (0, 1) for y in got[i])


def test_two_graphs_that_share_their_memory():
    T, E, k, hidden, inter = 24, 8, 2, 256, 128
    g, gu, dn = _layers(E, hidden, inter, E8M0, 14)
    xs = [F.random_rows(g, n, hidden, torch.bfloat16) for n in (T, T + 70)]
    logits = [torch.randn(len(x), E, generator=g, device="cuda") for x in xs]
    run = lambda i: sk.fp8_experts(xs[i], sk.route_tokens(logits[i], k), *gu, *dn)      # noqa: E731
    want = [run(i).clone() for i in (0, 1)]
    pool, graphs, out = torch.cuda.graph_pool_handle(), [], []
    for i in (0, 1):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], pool=pool):
            out.append(run(i))
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
        assert torch.equal(out[i], want[i])


def test_places_past_32_bits():
    """More than 2^31 codes and results in the layers' workspace: the last tokens against the definition."""
    T, E, k, hidden, inter = 66000, 4, 8, 4096 + 16, 128
    g, gu, dn = _layers(E, hidden, inter, E8M0, 15)
    x = F.random_rows(g, T, hidden, torch.bfloat16)
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    weights = torch.rand(T, k, generator=g, device="cuda")
    rows, offsets = sk.group_by_expert(ids, E)
    assert T * k * hidden > 2 ** 31 and offsets.tolist() == [0, *torch.bincount(ids.flatten(), minlength=E).cumsum(0).tolist()]
    y = sk.fp8_experts(x, sk.Routing(ids, weights, rows, offsets), *gu, *dn)
    for part in (slice(0, 20), slice(T - 40, T)):
        r, o = sk.group_by_expert(ids[part].contiguous(), E)
        _check_experts(x[part], r, weights[part], o, gu, dn, y[part])


def test_expert_layer_refusals():
    g, gu, dn = _layers(4, 128, 256, E8M0, 1)
    x = torch.randn(6, 128, device="cuda")
    r = sk.route_tokens(torch.randn(6, 4, device="cuda"), 2)
    for call in (lambda: sk.fp8_experts(x[:, :64], r, *gu, *dn), lambda: sk.fp8_experts(x[:5], r, *gu, *dn),
                 lambda: sk.fp8_experts(x, r, gu[0].flatten(1, 2), gu[1].flatten(1, 2), *dn), lambda: sk.fp8_experts(x, r, *gu, dn[0][:3], dn[1][:3]),
                 lambda: sk.fp8_experts(x, r._replace(weights=r.weights.half()), *gu, *dn), lambda: sk.fp8_experts(x, r._replace(rows=r.rows.long()), *gu, *dn),
                 lambda: sk.fp8_experts(x, r._replace(offsets=r.offsets[:4]), *gu, *dn),
                 lambda: sk.fp8_experts(x, r, gu[0], F.scale_values(gu[1]).float(), *dn)):
        with pytest.raises(RuntimeError):
            call()
