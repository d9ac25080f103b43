"""The position check of the attention calls (csrc/work_cut.h, rows_fit), compiled with g++ and run on the CPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_positions_at_the_ends_of_the_cache_and_of_32_bits(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "position_test")
    # (an overflow of signed integers ends the program)
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-ftrapv",
                        os.path.join(ROOT, "tests", "host", "position_test.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr
