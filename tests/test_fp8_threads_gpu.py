"""Every FP8 operator from several host threads at once, each on a stream of its own; the first calls of a process, too."""
import subprocess
import sys
import threading

import pytest
import torch

import fp8_util as F
import slimkernels_b200.torch as sk
from conftest import ROOT

pytestmark = pytest.mark.gpu
E8M0, F32 = torch.float8_e8m0fnu, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


def at_once(calls):
    """Runs the calls in threads that start together; raises what one of them raised."""
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
    if errors:
        raise errors[0]


def run_operators(seed, T, E, scales):
    """One pass through all of them; sizes, types and launches differ with the arguments."""
    g = F.generator(seed)
    hidden, inter, k = 256 + 16 * (seed % 3), 128 + 72 * (seed % 2), min(E, 4)
    x = F.random_rows(g, T, hidden, torch.bfloat16)
    weight = torch.randn(E, 2, inter, hidden, generator=g, device="cuda") * hidden ** -0.5
    gu = sk.prepare_weight_fp8(weight, scales)
    dn = sk.prepare_weight_fp8(weight[:, 0].transpose(1, 2), scales)
    r = sk.route_tokens(torch.randn(T, E, generator=g, device="cuda"), k)
    rows, offsets = sk.group_by_expert(r.expert_ids.long(), E)
    q, s = sk.quantize_fp8(x, scales)
    order = torch.empty(T * k, dtype=torch.long, device="cuda")
    order[r.rows.flatten().long()] = torch.arange(T * k, device="cuda") // k
    xq, xs = sk.quantize_fp8(x[order], scales)
    one = gu[0][0, 0], gu[1][0, 0]
    return [q.contiguous().view(torch.uint8), s.contiguous().view(torch.uint8), *r, rows, offsets, sk.fp8_gemm(q, s, *one), sk.fp8_linear(x, *one),
            sk.fp8_grouped_gemm(xq, xs, gu[0][:, 1].contiguous(), gu[1][:, 1].contiguous(), r.offsets), sk.fp8_experts(x, r, *gu, *dn)]


SETS = [(1, 5, 4, E8M0), (2, 64, 400, E8M0), (3, 300, 8, F32), (4, 33, 500, F32), (5, 700, 3, E8M0), (6, 1, 64, F32)]


def test_operators_from_threads():
    want = [run_operators(*s) for s in SETS]
    torch.cuda.synchronize()
    got = [[] for _ in SETS]

    def caller(i):
        def call():
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(15):
                    got[i].append(run_operators(*SETS[i]))
            stream.synchronize()
        return call

    at_once([caller(i) for i in range(len(SETS))])
    for i, w in enumerate(want):
        assert len(got[i]) == 15
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, w))
    assert sk.fp8_device_status() == 0


_FIRST = """
import sys
sys.path.insert(0, "tests")
import torch
from test_fp8_threads_gpu import SETS, at_once, run_operators
torch.zeros(1, device="cuda")
got = {}
def caller(i):
    def call():
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = run_operators(*SETS[i])
            torch.cuda.current_stream().synchronize()
    return call
at_once([caller(i) for i in range(len(SETS))])
for i, s in enumerate(SETS):
    assert all(torch.equal(a, b) for a, b in zip(got[i], run_operators(*s)))
print("equal")
"""


def test_first_calls_of_a_process_from_threads():
    run = subprocess.run([sys.executable, "-c", _FIRST], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert run.returncode == 0 and "equal" in run.stdout, run.stderr[-2000:]
