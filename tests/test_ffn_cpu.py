"""Argument rules of the feed-forward operators, built from the library's own source and run without a GPU, and the binding's table
of activations against the header's."""
import os
import re
import shutil
import subprocess

import pytest

from reference_model_b200 import binding

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _nvcc():
    for cand in ("/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    return None


@pytest.mark.skipif(_nvcc() is None, reason="needs nvcc's headers")
def test_argument_rules(tmp_path):
    exe = str(tmp_path / "ffn_check_cases")
    src = os.path.join(ROOT, "tests", "native", "ffn_check_cases.cu")
    build = subprocess.run([_nvcc(), "-O1", "-std=c++17", "-Wno-deprecated-gpu-targets", "-o", exe, src], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


def test_activations_are_the_headers():
    text = open(os.path.join(ROOT, "include", "tb200.h")).read()
    assert {k: int(v) for k, v in re.findall(r"TB200_ACT_(\w+)\s*=\s*(\d+)", text)} == binding.ACTIVATION
