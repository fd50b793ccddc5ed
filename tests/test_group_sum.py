"""The sums between the waves of a wide row (symmetrix-xl_amd/csrc/group_sum.hpp), compiled for the CPU with a thread a
lane and one wave late after every barrier: no wave writes what another has still to read."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_wave_overwrites_what_a_late_one_reads(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not available")
    program = str(tmp_path / "group_sum")
    out = subprocess.run([gxx, "-std=c++20", "-O1", "-pthread", "-Wall", "-Wno-unknown-pragmas",
                          "-I", os.path.join(ROOT, "symmetrix-xl_amd", "csrc"),
                          os.path.join(ROOT, "tests", "group_sum_host.cpp"), "-o", program],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-4000:]
    out = subprocess.run([program], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert out.stdout == "128 lanes: 0 wrong\n256 lanes: 0 wrong\n"
