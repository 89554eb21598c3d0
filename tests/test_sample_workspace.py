"""How much memory a call of the sampling operator takes besides its results (CPU only)."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.join(ROOT, "mlx-tree-spec_amd", "mlx_tree_spec_amd")


def test_workspace_is_bounded(tmp_path):
    """At most 1 GiB of lists (and their heads), whatever the rows and the vocabulary."""
    cxx = shutil.which("g++")
    if cxx is None or not os.path.exists(os.path.join(LIBDIR, "libqmm4.so")):
        pytest.skip("needs g++ and the built library")
    exe = tmp_path / "sample_workspace"
    cmd = [cxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(ROOT, "mlx-tree-spec_amd", "csrc"), os.path.join(ROOT, "tests", "sample_workspace.cpp"),
           "-L", LIBDIR, "-lqmm4", f"-Wl,-rpath,{LIBDIR}", "-o", str(exe)]
    build = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stderr[-4000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and int(run.stdout) <= (1 << 30) + (1 << 20), run.stdout
