"""The merge of a split prefill launch reads no more shares than there are where that costs time (host code only)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM_INCLUDE = "/opt/rocm/include"


def test_shares_at_once(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None or not os.path.isdir(ROCM_INCLUDE):
        pytest.skip("needs g++ and the HIP headers")
    exe = str(tmp_path / "merge_rule")
    built = subprocess.run([gxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I" + ROCM_INCLUDE,
                            os.path.join(ROOT, "tests", "native", "merge_rule.cc"), "-o", exe], capture_output=True, text=True, timeout=600)
    assert built.returncode == 0, built.stderr[-4000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "all checks passed" in run.stdout, run.stdout
