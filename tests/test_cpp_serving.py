"""The C++ mirror's methods for shared prefixes, eviction and log probabilities
(include/kraken/hip_context.hpp) through tests/cpp/serving_check.cpp: refusals without a
GPU, closed forms on one."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "kraken-infer_amd", "build", "serving_check")


def _run(mode):
    if not os.path.exists(BIN):
        subprocess.run(["make", "-C", os.path.join(ROOT, "kraken-infer_amd")], check=True,
                       capture_output=True)
    proc = subprocess.run([BIN, mode], capture_output=True, text=True, timeout=120)
    print(proc.stdout)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    assert "all checks passed" in proc.stdout


def test_cpp_serving_refusals():
    _run("cpu")


@pytest.mark.gpu
def test_cpp_serving_step():
    _run("gpu")
