"""The host code that the standalone operators' entry points share, compiled here against fakes of the CUDA calls
(tests/ops_common_check.cpp): what takes a second device or a failing CUDA call needs no GPU this way."""

import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("ops") / "ops_common_check")
    cuda = os.environ.get("CUDA", "/usr/local/cuda")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I" + os.path.join(cuda, "include"),
                           "-I" + os.path.join(os.path.dirname(HERE), "katago-rs_b200", "csrc"), "-o", exe,
                           os.path.join(HERE, "ops_common_check.cpp")])
    return exe


@pytest.mark.parametrize("check", ["managed_memory", "failed_call"])
def test_shared_host_code(program, check):
    r = subprocess.run([program, check], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
