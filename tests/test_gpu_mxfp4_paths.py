"""The kernels of the 4-bit cache on the paths that small launches do not take by themselves, against the definition in 64 bits
(oracle/mxfp4.py) within the bounds that tests/test_gpu_mxfp4.py derives."""
import numpy as np
import pytest
import torch

import tvm_amd
from oracle import mxfp4
from tests.gpu_util import DEV, dev, host, i32
from tests.test_gpu_mxfp4 import Pool, compare, rows_like
from tvm_amd import kernels
from tvm_amd._lib import check

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


@pytest.mark.parametrize("arrivals", [1, 2, 5])
def test_launches_after_an_abandoned_one_join_all_their_states(arrivals):
    """Counters that an earlier launch left half way, at every buffer of the stream, of the fp16 decode kernel as well."""
    rng = np.random.default_rng(arrivals)
    pool = Pool(rng, [3000, 40, 1700], 2, 16, 128)
    pages, indptr, ids, info = pool.device()
    q = rng.standard_normal((3, 8, 128)).astype(np.float16)
    rows = np.repeat(q, 2, 0)
    d_q, d_rows = dev(q), dev(rows)
    others = -d_q, -d_rows
    fp16_pages = torch.randn((len(pool.pages), 2, 2, 16, 128), device=DEV).half()
    zeros = torch.zeros(3, dtype=torch.int32, device=DEV)

    def run(d_q=d_q, d_rows=d_rows):
        o, s = ([torch.full((n, 8, *rest), 7.0, dtype=t, device=DEV) for n in (3, 3, 6)] for rest, t in (((128,), torch.float16), ((), torch.float32)))
        kernels.batch_decode_paged_kv(d_q, fp16_pages, indptr, ids, info, zeros, zeros, o[0], s[0], 0, 1.0, 1e4, 0.1)
        kernels.mxfp4_batch_decode_paged_kv(d_q, pages, indptr, ids, info, o[1], s[1], 0.1)
        kernels.mxfp4_batch_prefill_paged_kv(d_rows, i32([0, 2, 4, 6]), pages, indptr, ids, info, o[2], s[2], 0, 0.1)
        return [host(t) for t in o + s]

    previous = [tvm_amd.set_option(name, value) for name, value in (("decode_chunk_pages", 8), ("prefill_kv_splits", 7))]
    try:
        run()
        check(tvm_amd.lib().tvmkv_debug_abandon_scratch_launches(0))  # whole, whatever the tests before left
        want = run()
        for _ in range(3):
            run(*others)  # what is joined too early is these rows' states
            torch.cuda.synchronize()
            check(tvm_amd.lib().tvmkv_debug_abandon_scratch_launches(arrivals))
            assert all(np.array_equal(a, b) for a, b in zip(run(), want))
        compare(q, [1] * 3, pool, False, want[1], want[4], 0.1)
        compare(rows, [2] * 3, pool, False, want[2], want[5], 0.1)
    finally:
        for name, value in zip(("decode_chunk_pages", "prefill_kv_splits"), previous):
            tvm_amd.set_option(name, value)


@pytest.mark.parametrize("begin, batch", [(90, 40), (90, 400), (90, 560)])
def test_some_sequences_of_a_larger_table(begin, batch):
    """page_indptr and q_indptr that do not begin at 0: the rest of the tables stays where it is."""
    rng = np.random.default_rng(batch)
    stored, q_lens = rng.integers(1, 50, 660).tolist(), rng.integers(0, 4, 660).tolist()
    pool = Pool(rng, stored, 1, 16, 64)
    pages, indptr, ids, info = pool.device()
    some = slice(begin, begin + batch)
    q = rng.standard_normal((660, 2, 64)).astype(np.float16)
    out, lse = torch.zeros((batch, 2, 64), dtype=torch.float16, device=DEV), torch.zeros((batch, 2), device=DEV)
    kernels.mxfp4_batch_decode_paged_kv(dev(q[some]), pages, indptr[begin:begin + batch + 1], ids, info[some], out, lse, 0.125)
    whole = Pool.__new__(Pool)
    whole.__dict__.update(pool.__dict__, indptr=pool.indptr[begin:begin + batch + 1], info=pool.info[some])
    compare(q[some], [1] * batch, whole, False, host(out), host(lse), 0.125)
    q_indptr = np.concatenate(([0], np.cumsum(q_lens)))
    q = rng.standard_normal((q_indptr[-1], 2, 64)).astype(np.float16)
    out, lse = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV), torch.full(q.shape[:2], 7.0, device=DEV)
    kernels.mxfp4_batch_prefill_paged_kv(dev(q), i32(q_indptr[begin:begin + batch + 1]), pages, indptr[begin:begin + batch + 1], ids, info[some],
                                         out, lse, 1, 0.125)
    rows = slice(q_indptr[begin], q_indptr[begin + batch])
    compare(q[rows], q_lens[some], whole, True, host(out)[rows], host(lse)[rows], 0.125)
    others = np.ones(len(q), bool)
    others[rows] = False
    assert (host(out)[others] == 7).all() and (host(lse)[others] == 7).all()
