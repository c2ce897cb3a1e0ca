"""The ring of the experts' products for few rows (csrc/few_ring.h): a model of its roles on the CPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = os.path.join(str(tmp_path_factory.mktemp("few")), "few_ring_check")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "ml-drift_b200", "csrc"), "-o", exe,
                           os.path.join(ROOT, "tests", "few_ring_check.cc")])
    return exe


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("boxes", [1, 2, 3, 4, 7, 8, 9, 16, 256])
def test_what_is_kept_of_an_item_stays_until_all_have_read_it(check, bits, boxes):
    out = subprocess.run([check, str(bits), str(boxes)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout
