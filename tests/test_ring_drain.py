"""What the attention kernels over the 4-bit cache wait for when they give up (csrc/ring_order.h), on the CPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = os.path.join(str(tmp_path_factory.mktemp("drain")), "ring_drain_check")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "ml-drift_b200", "csrc"), "-o", exe,
                           os.path.join(ROOT, "tests", "ring_drain_check.cc")])
    return exe


@pytest.mark.parametrize("stages", [1, 2, 3, 4])
def test_every_copy_in_flight_is_waited_for(check, stages):
    out = subprocess.run([check, str(stages)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout
