"""Launches of the router whose tables fill the shared memory that a kernel has without asking for more."""
import subprocess
import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(built_libs):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests selected but no CUDA device is visible")


# Experts and warps whose tables, (warps + 1) * E + 1 integers, come to 49024 .. 49152 bytes: with the kernel's own 128 bytes more than the 48 KiB that a
# launch may have without asking for it.
_BORDER = """
import sys
import torch
import fp8_util as F
import slimkernels_b200.torch as sk
for E, warps in [(372, 32), (383, 31), (396, 30), (511, 23), (1022, 11), (1023, 11)]:
    for T in {warps, 64} if warps == 32 else {warps}:
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            logits = torch.randn(T, E, generator=F.generator(E + T), device="cuda").to(dtype)
            r = sk.route_tokens(logits, 3)
            ids, weights, rows, offsets = F.route_reference(logits.double().cpu().numpy(), 3, True)
            assert r.expert_ids.tolist() == ids.tolist() and r.rows.tolist() == rows.tolist() and r.offsets.tolist() == offsets.tolist()
    for T, k in ((warps, 32), (2, 16 * warps)):            # (a warp for every 32 choices)
        chosen = torch.randint(-1, E + 1, (T, k), generator=F.generator(T), device="cuda")
        rows, offsets = sk.group_by_expert(chosen, E)
        want_rows, want_offsets = F.group_reference(chosen.cpu().numpy(), E)
        assert rows.tolist() == want_rows.tolist() and offsets.tolist() == want_offsets.tolist()
print("routed")
"""


def test_tables_at_the_border_of_the_default_shared_memory():
    """In a process of its own: a larger call before would have raised the kernel's limit."""
    run = subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, 'tests')\n" + _BORDER], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert run.returncode == 0 and "routed" in run.stdout, run.stderr[-2000:]
