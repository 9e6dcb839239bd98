"""How far a product's K range is split: as far as its clusters run at once, and no further than pays."""
import ctypes

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


def _split(M, tiles, K, scales):
    v = [ctypes.c_int() for _ in range(5)]
    assert capi.load().sk_fp8_query_launch(M, tiles * 128, K, 1, capi.SK_SCALE_E8M0 if scales == E8M0 else capi.SK_SCALE_F32, *map(ctypes.byref, v)) == 0
    assert v[0].value == capi.FP8_FEW
    return v[3].value


@pytest.mark.skipif("not __import__('torch').cuda.is_available() or __import__('torch').cuda.get_device_properties(0).multi_processor_count != 148",
                    reason="the rules' figures are those of 148 SMs")
def test_splits_are_what_the_figures_say():
    for scales in (E8M0, F32):
        assert _split(1, 56, 16384, scales) == 4
        beyond = [_split(1, t, 16384, scales) for t in range(56, 75)]       # (clusters of four that run at once: 71 here, but GPCs differ from chip to chip)
        assert set(beyond) <= {2, 4} and beyond == sorted(beyond, reverse=True)
        assert [_split(1, t, 4096, scales) for t in (16, 18, 36)] == [8, 8, 4]
    # 32-bit scales, one row tile: the more features, the longer K
    assert [_split(16, 80, K, F32) for K in (4096, 6144)] == [2, 2]
    assert [_split(16, 112, K, F32) for K in (4096, 6144)] == [1, 2]
    assert [_split(16, 148, K, F32) for K in (4096, 6144, 8192)] == [1, 1, 2]
    assert _split(128, 18, 4096, F32) == 2
    # 8-bit scales: only where several row tiles share the weights
    assert [_split(16, t, 8192, E8M0) for t in (80, 96, 148)] == [1, 1, 1]
    assert [_split(64, t, 8192, E8M0) for t in (40, 72)] == [2, 1] and _split(256, 18, 8192, E8M0) == 2


@pytest.mark.parametrize("scales", [E8M0, F32])
@pytest.mark.parametrize("tiles", [15, 16, 18, 33, 34, 37])
def test_products_whose_clusters_share_sms(tiles, scales):
    g = F.generator(tiles)
    K = 4096
    x = F.random_rows(g, 9, K)
    w_q, w_s = sk.prepare_weight_fp8(torch.randn(tiles * 128 - 5, K, generator=g, device="cuda") * K ** -0.5, scales)
    x_q, x_s = sk.quantize_fp8(x, scales)
    exact, tol = F.product_tolerance(F.row_values(x_q, x_s), F.weight_values(w_q, w_s), torch.bfloat16)
    y = sk.fp8_gemm(x_q, x_s, w_q, w_s)
    F.assert_within(y, exact, tol)
    assert torch.equal(y, sk.fp8_gemm(x_q, x_s, w_q, w_s))
