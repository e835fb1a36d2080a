"""Sizes that the tiled feed-forward kernels take, and that others find the direct ones: the rule is built from the library's own source and run
without a GPU."""
import os
import subprocess

import pytest

from test_ffn_cpu import ROOT, _nvcc


@pytest.mark.skipif(_nvcc() is None, reason="needs nvcc's headers")
def test_sizes_of_the_tiled_kernels(tmp_path):
    exe = str(tmp_path / "ffn_reach_cases")
    src = os.path.join(ROOT, "tests", "native", "ffn_reach_cases.cu")
    build = subprocess.run([_nvcc(), "-O1", "-std=c++17", "-Wno-deprecated-gpu-targets", "-o", exe, src], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


def test_no_size_is_refused_behind_the_rule():
    """A product that passes the argument rules has a kernel: the tiled ones' launch refuses none for its number of tiles."""
    text = open(os.path.join(ROOT, "reference_model_b200", "csrc", "ffn_pair.cu")).read()
    assert "too large" not in text
