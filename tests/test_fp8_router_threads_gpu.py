"""Calls of the router from several host threads at once."""
import threading

import pytest
import torch

import fp8_util as F
import slimkernels_b200.torch as sk
from slimkernels_b200 import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


def _at_once(calls):
    """Runs the calls in threads that start together; the errors they raised."""
    start, errors = threading.Barrier(len(calls)), []

    def run(call):
        try:
            start.wait()
            call()
        except Exception as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return errors


@pytest.mark.parametrize("sizes", [((25, 512), (40, 512)), ((64, 400), (33, 500))])
def test_threads_whose_tables_differ(sizes):
    """One kernel, tables of 52.5 and 67.6 (52.8 and 68) kB: what one thread asks for must not lower what the other is about to launch with.  Called
    through the C ABI, which holds no lock."""
    lib = capi.load()

    def caller(T, E, k=8, repeats=20000):
        logits = torch.randn(T, E, generator=F.generator(E), device="cuda")
        ids, weights = torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(T, k, device="cuda")
        rows, offsets = torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        want = sk.route_tokens(logits, k)

        def call():
            for _ in range(repeats):
                rc = lib.sk_route_tokens(logits.data_ptr(), capi.SK_FLOAT_F32, E, T, E, k, 1, ids.data_ptr(), weights.data_ptr(), rows.data_ptr(),
                                         offsets.data_ptr(), None, 0, stream.cuda_stream)
                if rc != 0:
                    raise RuntimeError(f"{T} tokens, {E} experts: status {rc}")

        def check():
            for got, expected in zip((ids, weights, rows, offsets), want):
                assert torch.equal(got, expected)

        return call, check

    callers = [caller(*s) for s in sizes]
    torch.cuda.synchronize()
    assert not _at_once([call for call, _ in callers])
    torch.cuda.synchronize()
    for _, check in callers:
        check()
