"""The division that finds the page of a run of tokens, by a native driver (tests/native/exact_division.cc): exact for every
numerator of 31 bits, whatever the number of runs in a page."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_exact_division(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("needs g++")
    exe = str(tmp_path / "exact_division")
    built = subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                            os.path.join(ROOT, "tests", "native", "exact_division.cc"), "-o", exe], capture_output=True, text=True, timeout=300)
    assert built.returncode == 0, built.stderr[-4000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, (run.stdout + run.stderr)[-4000:]
    assert "all checks passed" in run.stdout
