"""Products that read weights and offsets before their wait count on the quantiser in front of them: it lets them start behind its own wait.
No run shows that reliably, so the source is checked."""
from test_dependent_launch_sources import _code, _kernels


def test_the_quantiser_lets_its_followers_start_behind_its_wait():
    body = {kernel: body for kernel, _, body in _kernels(_code("fp8_rows.cuh"))}["fp8_quantize_kernel"]
    assert body.count("grid_dep_wait();") == body.count("grid_dep_launch_dependents();") == 1
    assert body.index("grid_dep_wait();") < body.index("grid_dep_launch_dependents();")
