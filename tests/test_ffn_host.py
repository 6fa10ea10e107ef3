"""The feed-forward operators' bookkeeping (tt_lazy_b200/csrc/ffn.cuh) compiled for
the host (tests/native/ffn_host_check.cpp): what happens when a wait runs out or
a set-up call fails is shown here, without a GPU."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path_factory.mktemp("ffn") / "check")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-I" + os.path.join(ROOT, "include"),
                           "-I" + os.path.join(ROOT, "tt_lazy_b200", "csrc"), "-I" + os.path.join(CUDA_HOME, "include"),
                           os.path.join(HERE, "native", "ffn_host_check.cpp"), "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout.split()


def test_a_copy_whose_wait_ran_out_is_waited_for_again(lines):
    assert "copies_in_flight=ok" in lines


def test_a_set_up_that_failed_is_tried_again(lines):
    assert "set_up_once=ok" in lines
