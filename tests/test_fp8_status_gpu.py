"""The note of a wait that ran into its limit, read while the kernel is still running."""
import pytest
import torch

import slimkernels_b200.torch as sk
from slimkernels_b200 import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


def test_the_status_waits_for_a_stream_of_its_own():
    """A stream that does not synchronise with the legacy one; the kernel gives up after 10 million cycles, 5 ms or so."""
    w = sk.prepare_weight_fp8(torch.randn(256, 1024, device="cuda"))
    x = torch.randn(5, 1024, device="cuda").half()
    want = sk.fp8_linear(x, *w)
    assert sk.fp8_device_status() == 0
    lib, stream = capi.load(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    try:
        assert lib.sk_fp8_set_option(capi.SK_FP8_OPT_WAIT_LIMIT_CYCLES, 10_000_000) == 0 and lib.sk_fp8_set_option(capi.SK_FP8_OPT_TEST_SKIP_COPY, 3) == 0
        with torch.cuda.stream(stream):
            sk.fp8_linear(x, *w)
        status = sk.fp8_device_status()
    finally:
        lib.sk_fp8_set_option(capi.SK_FP8_OPT_WAIT_LIMIT_CYCLES, 0)
        lib.sk_fp8_set_option(capi.SK_FP8_OPT_TEST_SKIP_COPY, 0)
        torch.cuda.synchronize()
        left = sk.fp8_device_status()
    assert status != 0 and left == 0
    assert torch.equal(sk.fp8_linear(x, *w), want)
