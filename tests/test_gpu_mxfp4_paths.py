"""The kernels of the 4-bit cache on the paths that small launches do not take by themselves, against the definition in 64 bits
(oracle/mxfp4.py) within the bounds that tests/test_gpu_mxfp4.py derives."""
import numpy as np
import pytest
import torch

from oracle import mxfp4
from tests.gpu_util import DEV, dev, host, i32
from tests.test_gpu_mxfp4 import Pool, compare, rows_like
from tvm_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [1048592, 606832, 66848])
def test_pages_of_many_runs(page):
    """65 537, 37 927 and 4178 runs of 16 tokens: the keys that a window leaves lie on both sides of a page's end."""
    rng = np.random.default_rng(page)
    d, seen_in_first, stored = 64, 100, 2 * page + 40
    ids = np.array([2, 0, 1], np.int32)
    pool = kernels.mxfp4_pages(3, 1, page, d)
    keys = np.arange(2 * page - seen_in_first, stored)
    k, v = rows_like(rng, len(keys), 1, d), rows_like(rng, len(keys), 1, d)
    kernels.mxfp4_append(pool, dev(k), dev(v), i32(ids[keys // page] * page + keys % page))
    small = Pool(rng, [len(keys)], 1, 16, d)
    small.pages = mxfp4.append(mxfp4.empty_pages(len(small.pages), 1, 16, d), k, v, [small.slot(0, t) for t in range(len(keys))])
    info = i32([[40], [2 * page - seen_in_first], [0]])
    q = rng.standard_normal((3, 4, d)).astype(np.float16)
    out, lse = torch.empty((3, 4, d), dtype=torch.float16, device=DEV), torch.empty((3, 4), device=DEV)
    kernels.mxfp4_batch_prefill_paged_kv(dev(q), i32([0, 3]), pool, i32([0, 3]), i32(ids), info, out, lse, 1, 0.125)
    compare(q, [3], small, True, host(out), host(lse), 0.125)
    kernels.mxfp4_batch_decode_paged_kv(dev(q[:1]), pool, i32([0, 3]), i32(ids), info, out[:1], lse[:1], 0.125)
    compare(q[:1], [1], small, False, host(out[:1]), host(lse[:1]), 0.125)
