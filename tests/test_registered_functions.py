"""The registration source, compiled against a few lines that stand for tvm-ffi: what its functions take."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def call(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("needs g++")
    exe = str(tmp_path_factory.mktemp("registered") / "registered_functions")
    built = subprocess.run([gxx, "-std=c++17", "-I" + os.path.join(ROOT, "tests", "native", "ffi_stub"),
                            os.path.join(ROOT, "tests", "native", "registered_functions.cc"),
                            os.path.join(ROOT, "tvm_amd", "csrc", "tvm_ffi_adapter.cc"),
                            "-Wl,--unresolved-symbols=ignore-all", "-o", exe], capture_output=True, text=True, timeout=600)
    assert built.returncode == 0, built.stderr[-4000:]

    def run(*args):
        done = subprocess.run([exe, *args], capture_output=True, text=True, timeout=60)
        return done.returncode, done.stdout.strip()

    return run


def test_the_move_with_and_without_sums(call):
    assert call("tvmkv.move_kept_tokens", "1", "2", "3", "4", "5", "6") == (0, "1 2 3 4 5 6")
    assert call("tvmkv.move_kept_tokens", "1", "-", "3", "4", "-", "6") == (0, "1 -1 3 4 -1 6")


def test_what_is_no_tensor_is_refused(call):
    assert call("tvmkv.move_kept_tokens", "-", "2", "3", "4", "5", "6")[0] == 1
    assert call("tvmkv.move_kept_tokens", "1", "2", "3", "4", "5")[0] == 1
