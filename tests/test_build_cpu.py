"""What the build does when there is nothing to do."""
import os

import pytest

from slimkernels_b200 import _build


@pytest.fixture
def lib_dir(tmp_path, monkeypatch):
    monkeypatch.setattr(_build, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(_build, "CUDA_LIB", str(tmp_path / "libsk_w2a8.so"))
    runs = []
    monkeypatch.setattr(_build, "_run", lambda cmd, verbose: runs.append(cmd))
    return tmp_path, runs


def test_a_library_newer_than_its_sources_is_enough(lib_dir):
    """As it is shipped: without the objects it was linked from."""
    path, runs = lib_dir
    (path / "libsk_w2a8.so").write_bytes(b"")
    assert _build.build_cuda_lib() == str(path / "libsk_w2a8.so") and runs == []


def test_an_older_library_is_built_again(lib_dir):
    path, runs = lib_dir
    lib = path / "libsk_w2a8.so"
    lib.write_bytes(b"")
    os.utime(lib, (0, 0))
    _build.build_cuda_lib()
    assert sorted(os.path.basename(cmd[-1]) for cmd in runs[:-1]) == ["sk_fp8.cu", "sk_w2a8.cu"] and runs[-1][-2:] == [str(path / f"{n}.o") for n in ("sk_w2a8", "sk_fp8")]


def test_a_build_by_force_builds(lib_dir):
    path, runs = lib_dir
    (path / "libsk_w2a8.so").write_bytes(b"")
    _build.build_cuda_lib(force=True)
    assert len(runs) == 3
