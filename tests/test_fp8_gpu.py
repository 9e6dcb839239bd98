"""The FP8 quantisers and products on the GPU against their definition in 64 bits (tolerances: fp8_util)."""
import ctypes
import subprocess
import sys

import pytest
import torch

import fp8_util as F
import slimkernels_b200.torch as sk
from conftest import ROOT
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


def _options(row_tile=0, split=0, limit=0, skip=0, kernel=0):
    lib = capi.load()
    for key, value in ((capi.SK_FP8_OPT_ROW_TILE, row_tile), (capi.SK_FP8_OPT_SPLIT_K, split), (capi.SK_FP8_OPT_WAIT_LIMIT_CYCLES, limit),
                       (capi.SK_FP8_OPT_TEST_SKIP_COPY, skip), (capi.SK_FP8_OPT_KERNEL, kernel)):
        assert lib.sk_fp8_set_option(key, value) == 0


@pytest.fixture
def forced():
    yield _options
    _options()


# ------------------------------------------------------------------------------------------------------- quantisers
def _same_quantised(q, s, x, rows=1):
    rq, re, bad = F.quantise(x, rows)
    got = q.double()
    assert torch.equal(torch.isnan(got), torch.isnan(rq))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(rq))
    gs = F.scale_values(s)
    assert torch.equal(torch.isnan(gs), bad)
    assert torch.equal(gs[~bad], F.pow2(re)[~bad])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scales", [E8M0, F32])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 8), (2, 100), (5, 128), (17, 129), (4, 1000), (300, 4160), (1, 16384)])
def test_quantise_bit_exact(M, K, dtype, scales):
    g = F.generator(M * 31 + K)
    x = F.random_rows(g, M, K, dtype)
    if M > 2:
        x[0] = 0
        x[1, ::3] *= 2.0 ** -9
    x2 = x.clone()
    q, s = sk.quantize_fp8(x, scales)
    assert q.shape == (M, K) and s.shape == (M, F.ceil_div(K, 128)) and s.dtype == scales
    assert M == 1 or q.stride(0) % 16 == 0
    _same_quantised(q, s, x)
    assert torch.equal(x, x2)


@pytest.mark.parametrize("scales", [E8M0, F32])
def test_quantise_borders_ties_and_values_that_are_not_finite(scales):
    x = torch.zeros(12, 256, device="cuda")
    x[0, :6] = torch.tensor([448.0, 1.0625, 1.1875, -1.0625, 2.0 ** -10, 3 * 2.0 ** -10])     # ties; halves of the smallest code
    x[1, 0] = 448.0001                                                                        # the next exponent
    x[2, 0] = float("inf")
    x[2, 130] = 5.0
    x[3, 7] = float("nan")
    x[4, 0], x[4, 1] = 3e38, -1e-3
    x[5, 0] = 2.0 ** -130                                                                     # a subnormal: the smallest scale
    x[6, 128:] = -2.0
    x[7, 0] = float("-inf")
    x[8, 0], x[8, 1] = 1.75 * 2.0 ** 8, 1.7499999 * 2.0 ** 8
    x[9] = -0.0
    x[10, 255] = 65504.0
    q, s = sk.quantize_fp8(x, scales)
    _same_quantised(q, s, x)


def test_quantise_strided_and_leading_shapes():
    g = F.generator(5)
    wide = F.random_rows(g, 33, 700, torch.bfloat16)
    for x in (wide[:, 8:500], wide[:, 3:260], wide[::2, :256], wide.t()[:300]):
        q, s = sk.quantize_fp8(x)
        _same_quantised(q, s, x)
    x = F.random_rows(g, 24, 200).view(2, 3, 4, 200)
    q, s = sk.quantize_fp8(x)
    assert q.shape == x.shape and s.shape == (2, 3, 4, 2)
    _same_quantised(q.reshape(24, 200), s.reshape(24, 2), x.view(24, 200))
    q, s = sk.quantize_fp8(x[0, 0, 0])
    assert q.shape == (200,) and s.shape == (2,)
    q, s = sk.quantize_fp8(x[:0], F32)
    assert q.shape == (0, 3, 4, 200) and s.shape == (0, 3, 4, 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scales", [E8M0, F32])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 200), (3, 2, 129, 144), (2, 300, 77)])
def test_prepare_weight_bit_exact(shape, dtype, scales):
    g = F.generator(sum(shape))
    w = F.random_rows(g, 1, int(torch.tensor(shape).prod()), dtype).view(shape)
    w[..., 0, 0] *= 50
    q, s = sk.prepare_weight_fp8(w, scales)
    assert q.shape == w.shape and q.stride(-2) % 16 == 0
    N, K = shape[-2:]
    for qm, sm, wm in zip(q.reshape(-1, N, K), s.reshape(-1, F.ceil_div(N, 128), F.ceil_div(K, 128)), w.reshape(-1, N, K)):
        _same_quantised(qm, sm, wm, rows=128)


def test_prepare_weight_with_a_value_that_is_not_finite():
    w = torch.ones(200, 300, device="cuda")
    w[140, 10] = float("nan")
    w[3, 299] = float("inf")
    q, s = sk.prepare_weight_fp8(w)
    _same_quantised(q, s, w, rows=128)


# --------------------------------------------------------------------------------------------------------- products
def _operands(M, N, K, scales, seed, lead=()):
    g = F.generator(seed)
    x_q, x_s = sk.quantize_fp8(F.random_rows(g, M, K), scales)
    w_q, w_s = sk.prepare_weight_fp8(torch.randn(*lead, N, K, generator=g, device="cuda") * K ** -0.5, scales)
    if scales == F32:
        x_s, w_s = F.arbitrary_scales(x_s, g), F.arbitrary_scales(w_s, g)
    return x_q, x_s, w_q, w_s


def _check_product(x_q, x_s, w_q, w_s, out_dtype, **kw):
    exact, tol = F.product_tolerance(F.row_values(x_q, x_s), F.weight_values(w_q, w_s), out_dtype)
    y = sk.fp8_gemm(x_q, x_s, w_q, w_s, out_dtype, **kw)
    F.assert_within(y, exact, tol)
    return y


SIZES = [(1, 1, 1), (1, 128, 128), (2, 7, 16), (15, 129, 100), (16, 256, 512), (17, 300, 1000), (31, 1000, 144), (33, 128, 2048), (64, 640, 1024),
         (65, 384, 640), (127, 130, 272), (128, 512, 512), (129, 257, 1040), (300, 1024, 384), (513, 400, 2560), (1000, 777, 1111)]


@pytest.mark.parametrize("scales", [E8M0, F32])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K, scales, out_dtype):
    _check_product(*_operands(M, N, K, scales, M + N + K), out_dtype)


@pytest.mark.parametrize("scales", [E8M0, F32])
@pytest.mark.parametrize("M,N,K", [(5, 4096, 4096), (16, 12288, 1024), (96, 4096, 11008), (333, 5000, 4160), (2048, 4096, 1024), (4100, 2304, 512)])
def test_product_at_working_sizes(M, N, K, scales):
    _check_product(*_operands(M, N, K, scales, M + N + K), torch.bfloat16)


@pytest.mark.parametrize("row_tile", [16, 32])
@pytest.mark.parametrize("split", [1, 2, 4, 8])
@pytest.mark.parametrize("M,N,K", [(1, 128, 2048), (130, 200, 1100), (257, 1024, 1024)])
@pytest.mark.parametrize("scales", [E8M0, F32])
def test_few_rows_every_tile_and_split(M, N, K, scales, row_tile, split, forced):
    forced(row_tile, split, kernel=capi.FP8_FEW)
    x = _operands(M, N, K, scales, 3)
    y = _check_product(*x, torch.float16)
    assert torch.equal(y, sk.fp8_gemm(*x, torch.float16))


KERNELS = [(k, s) for k in (capi.FP8_FEW, capi.FP8_MANY, capi.FP8_PAIR) for s in (E8M0, F32) if (k, s) != (capi.FP8_PAIR, F32)]


@pytest.mark.parametrize("kernel,scales", KERNELS)
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 128, 2048), (130, 200, 1100), (128, 256, 128), (257, 1030, 1024), (300, 513, 400), (600, 8000, 640),
                                   (5000, 2560, 300)])
def test_every_kernel(M, N, K, kernel, scales, forced):
    forced(kernel=kernel)
    x = _operands(M, N, K, scales, 3)
    y = _check_product(*x, torch.float16)
    assert torch.equal(y, sk.fp8_gemm(*x, torch.float16))


@pytest.mark.parametrize("row_tile", [0, 16, 32])
@pytest.mark.parametrize("kernel", [capi.FP8_FEW, capi.FP8_MANY, capi.FP8_PAIR])
def test_every_scale_reaches_its_row_and_block(kernel, row_tile, forced):
    """Scales that differ from row to row and block to block by large factors, in any memory order: none may be taken for another's."""
    forced(row_tile, kernel=kernel)
    M, N, K = 300, 700, 1500
    x_q, x_s, w_q, w_s = _operands(M, N, K, E8M0, 4)
    g = F.generator(5)
    x_s.view(torch.uint8)[...] = torch.randint(100, 150, x_s.shape, generator=g, device="cuda").to(torch.uint8)
    w_s.view(torch.uint8)[...] = torch.randint(100, 150, w_s.shape, generator=g, device="cuda").to(torch.uint8)
    y = _check_product(x_q, x_s, w_q, w_s, torch.bfloat16)
    turned = x_s.view(torch.uint8).t().contiguous().t().view(E8M0)
    wide = torch.zeros(M, 13, dtype=torch.uint8, device="cuda")
    wide[:, 1:] = x_s.view(torch.uint8)
    assert turned.stride() == (1, M)
    for other in (turned, wide[:, 1:].view(E8M0)):
        assert torch.equal(y, sk.fp8_gemm(x_q, other, w_q, w_s))


def test_launches_are_what_the_rules_say(forced):
    lib = capi.load()
    sms = torch.cuda.get_device_properties(0).multi_processor_count

    def query(M, N, K, E=1, scales=E8M0):
        v = [ctypes.c_int() for _ in range(5)]
        assert lib.sk_fp8_query_launch(M, N, K, E, capi.SK_SCALE_E8M0 if scales == E8M0 else capi.SK_SCALE_F32, *map(ctypes.byref, v)) == 0
        return [i.value for i in v]

    assert query(1, 4096, 4096)[:4] == [capi.FP8_FEW, 16, 128, 4]
    assert query(17, 57344, 8192)[:4] == [capi.FP8_FEW, 32, 128, 1]
    assert query(256, 4096, 4096)[:3] == [capi.FP8_FEW, 32, 128] and query(4096, 4096, 4096)[:4] == [capi.FP8_PAIR, 256, 256, 1]
    assert query(64, 4096, 4096, scales=F32)[:3] == [capi.FP8_FEW, 16, 128] and query(512, 4096, 4096, scales=F32)[:3] == [capi.FP8_MANY, 128, 256]
    assert query(64, 2048, 2048, 64)[:3] == [capi.FP8_FEW, 16, 128] and query(64 * 20, 2048, 2048, 64)[:3] == [capi.FP8_FEW, 32, 128]
    assert query(64 * 100, 2048, 2048, 64)[:3] == [capi.FP8_MANY, 128, 256] and query(64 * 600, 2048, 2048, 64)[:3] == [capi.FP8_PAIR, 256, 256]
    assert query(64 * 20, 2048, 2048, 64, F32)[0] == capi.FP8_MANY
    kernel, tile, features, split, ctas = query(5, 1024, 8192)
    assert ctas == 8 * split and ctas <= sms and split == 8
    assert query(300, 512, 16384)[:4] == [capi.FP8_FEW, 32, 128, 4] and query(300, 512, 16384, scales=F32)[:4] == [capi.FP8_FEW, 16, 128, 2]
    assert query(256, 2048, 4096)[3] == 1 and query(16, 22016, 4096)[3] == 1 and query(100, 1000, 8192, scales=F32)[3] == 4
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 1, 2000)):
        assert lib.sk_fp8_query_launch(*bad, 0, None, None, None, None, None) == capi.SK_ERR_BAD_SHAPE
    forced(kernel=capi.FP8_PAIR)
    assert query(5, 1024, 8192)[0] == capi.FP8_PAIR and query(5, 1024, 8192, scales=F32)[0] == capi.FP8_MANY


def test_product_strides():
    """Padded rows, scales in either order or shared by broadcasting, a column slice of a wider result."""
    x_q, x_s, w_q, w_s = _operands(37, 200, 300, F32, 11)
    wide = torch.zeros(37, 512, device="cuda").to(torch.float8_e4m3fn)
    wide[:, :300] = x_q
    for xq in (x_q, wide[:, :300]):
        for xs in (x_s, x_s.contiguous(), x_s.t().contiguous().t(), x_s[:1].expand(37, -1)):
            exact, tol = F.product_tolerance(F.row_values(xq, xs), F.weight_values(w_q, w_s), torch.bfloat16)
            F.assert_within(sk.fp8_gemm(xq, xs, w_q, w_s), exact, tol)
    for lo in (8, 3):
        full = torch.full((37, 219), 9.0, dtype=torch.bfloat16, device="cuda")
        out = full[:, lo:lo + 200]
        assert sk.fp8_gemm(x_q, x_s, w_q, w_s, out=out) is out
        exact, tol = F.product_tolerance(F.row_values(x_q, x_s), F.weight_values(w_q, w_s), torch.bfloat16)
        F.assert_within(out, exact, tol)
        assert bool((full[:, :lo] == 9).all()) and bool((full[:, lo + 200:] == 9).all())
    assert sk.fp8_gemm(x_q[:0], x_s[:0], w_q, w_s).shape == (0, 200)


@pytest.mark.parametrize("kernel,scales", [(0, E8M0), (0, F32)] + KERNELS)
@pytest.mark.parametrize("M", [3, 40, 200])
def test_nan_stays_in_its_row_and_feature(M, kernel, scales, forced):
    forced(kernel=kernel)
    g = F.generator(M)
    x = F.random_rows(g, M, 600)
    w = torch.randn(300, 600, generator=g, device="cuda")
    x[1, 5] = float("nan")
    x[2, 599] = float("inf")
    w[290, 3] = float("nan")                    # its block: features 256 .. 299
    y = sk.fp8_gemm(*sk.quantize_fp8(x, scales), *sk.prepare_weight_fp8(w, scales))
    nan = torch.isnan(y)
    assert bool(nan[1:3].all()) and bool(nan[:, 256:].all())
    nan[1:3] = False
    nan[:, 256:] = False
    assert not bool(nan.any())


@pytest.mark.parametrize("kernel", [0, capi.FP8_FEW, capi.FP8_MANY, capi.FP8_PAIR])
def test_scales_at_the_ends_of_their_range(kernel, forced):
    """2^-127 (the smallest 8-bit scale, a subnormal float) times large ones; a NaN scale; sums that leave the range of fp32.

    The sum over the blocks is kept in fp32: where a block's share or the sum up to it is beyond 2^128, it is infinite from there on, or
    NaN once two infinities of either sign meet, whatever the whole sum would be.  There the result has to be not finite."""
    forced(kernel=kernel)
    x_q, x_s, w_q, w_s = _operands(4, 128, 256, E8M0, 2)
    bits = x_s.view(torch.uint8)
    bits[0], bits[1], bits[2, 0] = 0, 1, 255
    w_s.view(torch.uint8)[...] = 250
    xv, wv = F.row_values(x_q, x_s), F.weight_values(w_q, w_s)
    shares = torch.stack([xv[:, b:b + 128] @ wv[:, b:b + 128].T for b in (0, 128)])
    most = torch.maximum(shares, shares.cumsum(0)).abs().amax(0).maximum(shares.abs().amax(0))
    y = sk.fp8_gemm(x_q, x_s, w_q, w_s)
    gone, kept = most > 2.0 ** 128 * (1 + 2.0 ** -10), most < 2.0 ** 127
    assert bool(gone[3].any()) and not bool(torch.isfinite(y[gone]).any())
    exact, tol = F.product_tolerance(xv, wv, torch.bfloat16)
    kept |= torch.isnan(exact)
    F.assert_within(y[kept], exact[kept], tol[kept])


def test_linear_layers():
    g = F.generator(4)
    w = torch.randn(520, 392, generator=g, device="cuda") * 0.05
    for scales in (E8M0, F32):
        w_q, w_s = sk.prepare_weight_fp8(w, scales)
        wv = F.weight_values(w_q, w_s)
        for x in (F.random_rows(g, 5, 392, torch.bfloat16), F.random_rows(g, 70, 392, torch.float16), F.random_rows(g, 9, 392),
                  F.random_rows(g, 300, 400, torch.bfloat16)[:, 4:396], F.random_rows(g, 12, 392, torch.float16).view(3, 4, 392)):
            y = sk.fp8_linear(x, w_q, w_s)
            assert y.shape == (*x.shape[:-1], 520) and y.dtype == (torch.bfloat16 if x.dtype == torch.bfloat16 else torch.float16)
            exact, tol = F.product_tolerance(F.quantised_values(x.reshape(-1, 392)), wv, y.dtype)
            F.assert_within(y.reshape(-1, 520), exact, tol)
            # the same bits as its two halves
            q, s = sk.quantize_fp8(x.reshape(-1, 392), scales)
            assert torch.equal(y.reshape(-1, 520), sk.fp8_gemm(q, s, w_q, w_s, y.dtype))
        assert sk.fp8_linear(x[:0], w_q, w_s).shape == (0, 4, 520)
        assert sk.fp8_linear(x, w_q, w_s, torch.bfloat16).dtype == torch.bfloat16
    v = F.random_rows(g, 1, 392, torch.bfloat16)[0]
    assert sk.fp8_linear(v, w_q, w_s).shape == (520,)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("split", [0, 1, 8])
@pytest.mark.parametrize("M,N,K", [(1, 1, 8), (1, 4096, 4096), (7, 200, 136), (16, 384, 1000), (17, 130, 2056), (32, 1000, 128), (9, 12800, 520), (33, 256, 512)])
def test_linear_layers_of_few_rows_are_quantiser_and_product(M, N, K, split, dtype, forced):
    """The bits are those of the two calls, whatever reads the rows (aligned or not), values that are not finite and zeros included."""
    forced(split=split)
    g = F.generator(M + K)
    w_q, w_s = sk.prepare_weight_fp8(torch.randn(N, K, generator=g, device="cuda") * K ** -0.5)
    wide = F.random_rows(g, M, K + 16, dtype)
    wide[0, 8:70] = 0
    if M > 4:
        wide[1, 9], wide[2, K + 7], wide[3] = float("nan"), float("inf"), 0
    for lo in (0, 8, 3):
        x = wide[:, lo:lo + K]
        y = sk.fp8_linear(x, w_q, w_s)
        want = sk.fp8_gemm(*sk.quantize_fp8(x), w_q, w_s, dtype)
        assert torch.equal(torch.nan_to_num(y, 7.0), torch.nan_to_num(want, 7.0)) and torch.equal(torch.isnan(y), torch.isnan(want))


def test_refusals():
    x_q, x_s, w_q, w_s = _operands(8, 128, 256, F32, 1)
    e_s = torch.ones(1, 2, device="cuda").to(E8M0)
    bad = [lambda: sk.fp8_gemm(x_q, x_s, w_q, e_s),                                     # two types of scales
           lambda: sk.fp8_gemm(x_q, x_s[:, :1], w_q, w_s),                              # too few scales
           lambda: sk.fp8_gemm(x_q, x_s, w_q, w_s.t()),
           lambda: sk.fp8_gemm(x_q[:, :128], x_s[:, :1], w_q, w_s),                     # other features
           lambda: sk.fp8_gemm(x_q, x_s, w_q, w_s, torch.float32),
           lambda: sk.fp8_gemm(x_q[:, 1:], x_s, w_q[:, 1:], w_s),                       # rows that start anywhere
           lambda: sk.fp8_gemm(x_q.t().contiguous().t(), x_s, w_q, w_s),
           lambda: sk.fp8_gemm(x_q.float(), x_s, w_q, w_s),
           lambda: sk.fp8_gemm(x_q, x_s, w_q.cpu(), w_s),
           lambda: sk.fp8_gemm(x_q, x_s.cpu(), w_q, w_s),
           lambda: sk.fp8_gemm(x_q, x_s, w_q, w_s, out=torch.empty(8, 127, dtype=torch.bfloat16, device="cuda")),
           lambda: sk.fp8_gemm(x_q, x_s, w_q, w_s, out=torch.empty(8, 128, device="cuda")),
           lambda: sk.fp8_gemm(x_q, x_s, w_q, w_s, out=torch.empty(1, 128, dtype=torch.bfloat16, device="cuda").expand(8, 128)),
           lambda: sk.fp8_linear(torch.zeros(4, 255, device="cuda"), w_q, w_s),
           lambda: sk.fp8_linear(torch.zeros(4, 256, device="cuda", dtype=torch.float64), w_q, w_s),
           lambda: sk.quantize_fp8(torch.zeros(4, 0, device="cuda")),
           lambda: sk.quantize_fp8(torch.zeros(4, 8, device="cuda"), torch.float16),
           lambda: sk.fp8_grouped_gemm(x_q, x_s, w_q, w_s, torch.zeros(2, dtype=torch.int32, device="cuda")),
           lambda: sk.fp8_grouped_gemm(x_q, x_s, w_q[None], w_s[None], torch.zeros(3, dtype=torch.int32, device="cuda")),
           lambda: sk.fp8_grouped_gemm(x_q, x_s, w_q[None], w_s[None], torch.zeros(2, dtype=torch.int64, device="cuda"))]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()


# ------------------------------------------------------------------------------------------------ products by expert
def _check_grouped(offsets, rows, N, K, scales, out_dtype, seed=0):
    E = len(offsets) - 1
    x_q, x_s, w_q, w_s = _operands(rows, N, K, scales, seed, lead=(E,))
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    out = torch.full((rows, N), 77.0, dtype=out_dtype, device="cuda")
    assert sk.fp8_grouped_gemm(x_q, x_s, w_q, w_s, off, out=out) is out
    xv, covered = F.row_values(x_q, x_s), torch.zeros(rows, dtype=torch.bool)
    for e in range(E):
        lo, hi = offsets[e], offsets[e + 1]
        if hi > lo:
            exact, tol = F.product_tolerance(xv[lo:hi], F.weight_values(w_q[e], w_s[e]), out_dtype)
            F.assert_within(out[lo:hi], exact, tol, f"expert {e}")
            covered[lo:hi] = True
    assert bool((out[~covered.cuda()] == 77).all()), "rows of no group were written"
    return x_q, x_s, w_q, w_s, off, out


GROUPS = [[0, 5], [0, 0, 0, 1, 1], [0, 16, 16, 33, 50], [3, 20, 20, 21, 60, 60], [0, 1, 2, 3, 4, 5, 6, 7, 8], [0, 200, 201, 460], [7, 7, 7],
          [0] + [40] * 33 + [41] * 40]


@pytest.mark.parametrize("offsets", GROUPS)
@pytest.mark.parametrize("N,K,scales,out_dtype", [(130, 144, E8M0, torch.bfloat16), (256, 600, F32, torch.float16), (1, 16, F32, torch.bfloat16)])
def test_grouped_product(offsets, N, K, scales, out_dtype):
    _check_grouped(offsets, offsets[-1] + 9, N, K, scales, out_dtype)


@pytest.mark.parametrize("row_tile", [16, 32])
@pytest.mark.parametrize("scales", [E8M0, F32])
def test_grouped_product_of_few_rows_every_tile(scales, row_tile, forced):
    forced(row_tile, kernel=capi.FP8_FEW)
    _check_grouped([0, 130, 130, 131, 300, 420, 433], 440, 384, 400, scales, torch.float16)


@pytest.mark.parametrize("kernel,scales", KERNELS)
@pytest.mark.parametrize("N,K", [(384, 400), (130, 1040)])
def test_grouped_product_every_kernel(N, K, kernel, scales, forced):
    forced(kernel=kernel)
    _check_grouped([2, 130, 130, 131, 300, 700, 713], 720, N, K, scales, torch.float16)
    _check_grouped([0, 0, 0, 3], 3, N, K, scales, torch.bfloat16)


def test_grouped_product_many_experts_and_fresh_result():
    offsets = [0]
    for e in range(1024):
        offsets.append(offsets[-1] + (e * 7919) % 4)
    x_q, x_s, w_q, w_s, off, out = _check_grouped(offsets, offsets[-1], 136, 160, E8M0, torch.bfloat16)
    assert torch.equal(sk.fp8_grouped_gemm(x_q, x_s, w_q, w_s, off), out)
    assert sk.fp8_grouped_gemm(x_q[:0], x_s[:0], w_q, w_s, off * 0).shape == (0, 136)


def test_grouped_product_cuts_offsets_to_its_rows():
    """Offsets that run backwards or out of the rows are cut: nothing outside the result is touched, rows in order are right."""
    x_q, x_s, w_q, w_s = _operands(40, 128, 128, E8M0, 9, lead=(4,))
    out = torch.full((48, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    off = torch.tensor([-3, 10, 4, 30, 1000], dtype=torch.int32, device="cuda")        # cut to 0, 10, 10, 30, 40
    sk.fp8_grouped_gemm(x_q, x_s, w_q, w_s, off, out=out[:40])
    want = sk.fp8_grouped_gemm(x_q, x_s, w_q, w_s, torch.tensor([0, 10, 10, 30, 40], dtype=torch.int32, device="cuda"))
    assert torch.equal(out[:40], want) and bool((out[40:] == 5).all())


def test_nan_stays_in_its_group():
    g = F.generator(8)
    x = F.random_rows(g, 30, 256)
    x[10] = float("nan")
    w = torch.randn(3, 128, 256, generator=g, device="cuda")
    w[2] = float("nan")
    off = torch.tensor([0, 10, 20, 30], dtype=torch.int32, device="cuda")
    y = sk.fp8_grouped_gemm(*sk.quantize_fp8(x), *sk.prepare_weight_fp8(w), off)
    nan = torch.isnan(y)
    assert bool(nan[10].all()) and bool(nan[20:].all()) and not bool(nan[:10].any()) and not bool(nan[11:20].any())


# --------------------------------------------------------------------------------------------------- offsets past 32 bits
@pytest.mark.parametrize("M,N,K", [(264000, 128, 8192), (264000, 8200, 128)])
@pytest.mark.parametrize("scales", [E8M0, F32])
def test_linear_layers_past_32_bits(M, N, K, scales):
    """More than 2^31 activations, or results."""
    g = F.generator(N)
    w = sk.prepare_weight_fp8(torch.randn(N, K, generator=g, device="cuda"), scales)
    x = torch.randn(M, K, generator=g, device="cuda", dtype=torch.bfloat16)
    y = sk.fp8_linear(x, *w)
    for part in (slice(0, 20), slice(M - 70, M)):
        exact, tol = F.product_tolerance(F.quantised_values(x[part]), F.weight_values(*w), torch.bfloat16)
        F.assert_within(y[part], exact, tol)


@pytest.mark.parametrize("M,N,K,scales", [(594, 256, 10608, F32), (300, 512, 16384, E8M0), (100, 1000, 8192, F32), (16, 8192, 16384, E8M0)])
def test_split_products_of_two_ctas_to_an_sm(M, N, K, scales):
    x = _operands(M, N, K, scales, 5)
    y = sk.fp8_gemm(*x)
    exact, tol = F.product_tolerance(F.row_values(*x[:2]), F.weight_values(*x[2:]), torch.bfloat16)
    F.assert_within(y, exact, tol)
    assert torch.equal(y, sk.fp8_gemm(*x))


@pytest.mark.parametrize("kernel", [capi.FP8_MANY, capi.FP8_PAIR])
@pytest.mark.parametrize("scales", [E8M0, F32])
def test_odd_pitches_write_their_rows_and_columns_only(kernel, scales, forced):
    """Results whose rows start on 2 bytes, by groups that end inside a warp's rows, into a slice of a larger matrix."""
    g = F.generator(16)
    off = torch.tensor([0, 1, 34, 34, 200, 331], dtype=torch.int32, device="cuda")
    w = sk.prepare_weight_fp8(torch.randn(5, 413, 256, generator=g, device="cuda"), scales)
    x = sk.quantize_fp8(torch.randn(340, 256, generator=g, device="cuda"), scales)
    forced(kernel=kernel)
    want = torch.zeros(340, 416, dtype=torch.bfloat16, device="cuda")[:, :413]
    sk.fp8_grouped_gemm(*x, *w, off, out=want)
    whole = torch.full((345, 421), 7.0, dtype=torch.bfloat16, device="cuda")
    out = whole[3:343, 5:418]
    sk.fp8_grouped_gemm(*x, *w, off, out=out)
    assert torch.equal(out[:331], want[:331])
    out[:331] = 7.0
    assert bool((whole == 7.0).all())


@pytest.mark.parametrize("kernel", [capi.FP8_FEW, capi.FP8_MANY, capi.FP8_PAIR])
@pytest.mark.parametrize("scales", [E8M0, F32])
def test_weights_past_32_bits(kernel, scales, forced):
    E, N, K = 33, 8192, 8192
    g = F.generator(8)
    assert E * N * K > 2 ** 31
    w_q = (torch.randint(0, 256, (E, N, K), generator=g, device="cuda", dtype=torch.uint8) & 0xbe).view(torch.float8_e4m3fn)
    w_s = F.pow2(torch.randint(-4, 5, (E, N // 128, K // 128), generator=g, device="cuda")).float().to(scales)
    off = [0, 3] + [3] * (E - 3) + [5, 25]
    x = sk.quantize_fp8(F.random_rows(g, 25, K, torch.bfloat16), scales)
    forced(kernel=kernel)
    y = sk.fp8_grouped_gemm(*x, w_q, w_s, torch.tensor(off, dtype=torch.int32, device="cuda"))
    for e in (0, E - 2, E - 1):
        part = slice(off[e], off[e + 1])
        exact, tol = F.product_tolerance(F.row_values(x[0][part], x[1][part]), F.weight_values(w_q[e], w_s[e]), torch.bfloat16)
        F.assert_within(y[part], exact, tol)


def test_rows_far_apart():
    """A column slice of a matrix whose rows lie 2^29 bytes apart: pitches in 64 bits."""
    base = torch.zeros(6, 2 ** 29, dtype=torch.uint8, device="cuda")
    x_q, x_s = sk.quantize_fp8(torch.randn(6, 256, device="cuda", generator=F.generator(9)))
    far = base[:, 4096:4096 + 256].view(torch.float8_e4m3fn)
    far.view(torch.uint8).copy_(x_q.view(torch.uint8))
    w = sk.prepare_weight_fp8(torch.randn(160, 256, device="cuda", generator=F.generator(10)))
    out = base[:, 2 ** 28:2 ** 28 + 320].view(torch.bfloat16)
    want = sk.fp8_gemm(x_q, x_s, *w)
    sk.fp8_gemm(far, x_s, *w, out=out)
    assert torch.equal(out, want) and torch.equal(sk.quantize_fp8(out)[0].view(torch.uint8), sk.quantize_fp8(want)[0].view(torch.uint8))


# -------------------------------------------------------------------------------------------- streams, graphs, failure
def test_captured_products_follow_their_inputs():
    g = F.generator(6)
    w_q, w_s = sk.prepare_weight_fp8(torch.randn(640, 512, generator=g, device="cuda"))
    x = F.random_rows(g, 20, 512, torch.bfloat16)
    sk.fp8_linear(x, w_q, w_s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = sk.fp8_linear(x, w_q, w_s)
        z = sk.fp8_linear(y[:, :512], w_q, w_s)
    for seed in (1, 2):
        x.copy_(F.random_rows(F.generator(seed), 20, 512, torch.bfloat16))
        graph.replay()
        want = sk.fp8_linear(x, w_q, w_s)
        assert torch.equal(y, want) and torch.equal(z, sk.fp8_linear(want[:, :512], w_q, w_s))


_FIRST_CALL = """
import torch
import slimkernels_b200.torch as sk
w = torch.randn(256, 256, device="cuda")
x = torch.randn(3, 256, device="cuda")
off = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    w_q, w_s = sk.prepare_weight_fp8(w)
    y = sk.fp8_linear(x, w_q, w_s)
    r = sk.route_tokens(x, 2)
graph.replay()
torch.cuda.synchronize()
assert (y.float() - x @ w.t()).abs().max() < 8
print("captured")
"""


def test_first_call_of_a_process_may_be_captured():
    run = subprocess.run([sys.executable, "-c", _FIRST_CALL], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


def test_two_streams_at_once():
    ops = [_operands(24, 2048, 2048, E8M0, seed) for seed in (1, 2)]
    want = [sk.fp8_gemm(*o) for o in ops]
    streams = [torch.cuda.Stream() for _ in ops]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(sk.fp8_gemm(*ops[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in (0, 1) for y in got[i])


def test_weights_written_on_the_way_are_seen():
    """A layer whose weight the kernel in front of it writes, over and over: nothing is read early."""
    g = F.generator(12)
    x = F.random_rows(g, 8, 1024, torch.bfloat16)
    sets = [sk.prepare_weight_fp8(torch.randn(1024, 1024, generator=g, device="cuda")) for _ in range(2)]
    want = [sk.fp8_linear(x, *s) for s in sets]
    w_q, w_s = sets[0][0].clone(), sets[0][1].clone()
    got = []
    for i in range(40):
        w_q.copy_(sets[i % 2][0])
        w_s.copy_(sets[i % 2][1])
        got.append(sk.fp8_linear(x, w_q, w_s))
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))


@pytest.mark.parametrize("M,kernel,scales", [(4, 0, E8M0), (4, 0, F32), (200, capi.FP8_FEW, E8M0), (200, capi.FP8_FEW, F32), (200, capi.FP8_MANY, E8M0),
                                             (200, capi.FP8_MANY, F32), (500, capi.FP8_PAIR, E8M0)])
def test_a_copy_that_never_lands_ends_in_a_status(M, kernel, scales, forced):
    x = _operands(M, 256, 1024, scales, 3)
    forced(kernel=kernel)
    want = sk.fp8_gemm(*x)
    forced(limit=2_000_000, skip=3, kernel=kernel)
    sk.fp8_gemm(*x)
    torch.cuda.synchronize()
    assert sk.fp8_device_status() != 0
    assert sk.fp8_device_status() == 0
    forced(kernel=kernel)
    assert torch.equal(sk.fp8_gemm(*x), want)


def test_a_copy_that_never_lands_ends_in_a_status_in_a_linear_layer(forced):
    w = sk.prepare_weight_fp8(torch.randn(256, 1024, device="cuda"))
    x = torch.randn(5, 1024, device="cuda").half()
    want = sk.fp8_linear(x, *w)
    forced(limit=2_000_000, skip=3)
    sk.fp8_linear(x, *w)
    torch.cuda.synchronize()
    assert sk.fp8_device_status() != 0
    forced()
    assert torch.equal(sk.fp8_linear(x, *w), want)


@pytest.mark.skipif("not __import__('torch').cuda.is_available() or __import__('torch').cuda.device_count() < 2", reason="needs two GPUs")
def test_another_device_than_the_current_one():
    x = torch.randn(5, 256, device="cuda:1")
    w = sk.prepare_weight_fp8(torch.randn(128, 256, device="cuda:1"))
    y = sk.fp8_linear(x, *w)
    assert y.device == x.device
    exact, tol = F.product_tolerance(F.quantised_values(x), F.weight_values(*w), y.dtype)
    F.assert_within(y, exact, tol)
