"""The move of kept tokens on a CPU, wave by wave: whichever wave of a workgroup is ahead, rows go where the list says."""
import ctypes
import itertools
import os
import shutil
import subprocess

import numpy as np
import pytest

from oracle import eviction

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
IN_ORDER, FIRST, SECOND = range(3)


@pytest.fixture(scope="module")
def waves(tmp_path_factory):
    clang = shutil.which("clang++") or "/opt/rocm/llvm/bin/clang++"
    if not os.path.exists(clang):
        pytest.skip("needs clang++")
    folder = tmp_path_factory.mktemp("waves")
    source = open(os.path.join(ROOT, "tvm_amd", "csrc", "kernels_evict.hip")).read()
    begin, end = source.index("struct MoveParams {"), source.index("// Launches\n")
    (folder / "move_kept_kernel.inc").write_text(source[begin:source.rindex("// ---", begin, end)])
    library = str(folder / "move_kept_waves.so")
    built = subprocess.run([clang, "-std=c++17", "-O1", "-shared", "-fPIC", "-Wno-unknown-attributes", "-I" + str(folder),
                            os.path.join(ROOT, "tests", "native", "move_kept_waves.cc"), "-o", library], capture_output=True, text=True, timeout=600)
    assert built.returncode == 0, built.stderr[-4000:]
    return ctypes.CDLL(library)


def pool(rng, stored, h_kv, page, d):
    counts = [-(-n // page) for n in stored]
    total = sum(counts) + 2
    ids, weight_ids = (rng.permutation(total)[:sum(counts)].astype(np.int32) for _ in range(2))
    return (rng.standard_normal((total, 2, h_kv, page, d)).astype(np.float16), rng.random((total, h_kv, page)).astype(np.float32),
            np.concatenate(([0], np.cumsum(counts))).astype(np.int32), ids, weight_ids)


def move(waves, launches, tables, kept, order, parts, slices):
    pages, sums, indptr, ids, weight_ids = tables
    pages, sums, kept = pages.copy(), sums.copy(), np.ascontiguousarray(kept, np.int32)
    _, _, h_kv, page, d = pages.shape
    p = lambda x: x.ctypes.data_as(ctypes.c_void_p)
    for launch in launches:
        rc = waves.move_kept(launch, p(pages), p(sums), p(indptr), p(ids), p(weight_ids), p(kept), len(indptr) - 1, h_kv, kept.shape[2],
                             page.bit_length() - 1, 2 * d * 2 // 16, slices, parts, p(np.array(order, np.int32)))
        assert rc == 0, "threads of a workgroup wait at different barriers"
    return pages, sums


LISTS = {
    "choice": lambda n: [np.concatenate((np.arange(n // 3), np.arange(n - n // 4, n)))],
    "recent": lambda n: [np.arange(7, n)],                # every token by fewer places than they are: in order
    "few": lambda n: [np.concatenate(([n - 3], np.arange(1, 200), [n - 2, n - 1]))],
    "same": lambda n: [np.maximum(np.sort(np.random.default_rng(n).integers(0, n, n - n // 4)), np.arange(n - n // 4))],  # tokens several times
    "odd": lambda n: [np.array([n - 1, 1, 1 << 30, 9, -5] + [-1] * 300)],
}


@pytest.mark.parametrize("kind", LISTS)
@pytest.mark.parametrize("launches, parts, slices", [((IN_ORDER,), 2, 2), ((FIRST, SECOND), 3, 2), ((FIRST, SECOND), 1, 1)])
def test_any_wave_may_be_ahead(waves, launches, parts, slices, kind):
    rng = np.random.default_rng(parts)
    tables = pool(rng, [700], 1, 16, 64)
    kept = np.array(LISTS[kind](700), np.int32)[:, None]
    want, want_sums = eviction.move(tables[0], tables[1], tables[2], tables[3], tables[4], kept)
    for order in itertools.permutations(range(4)):
        pages, sums = move(waves, launches, tables, kept, order, parts, slices)
        assert np.array_equal(pages.view(np.uint16), want.view(np.uint16)), f"waves in the order {order}"
        assert np.array_equal(sums, want_sums), f"waves in the order {order}"
