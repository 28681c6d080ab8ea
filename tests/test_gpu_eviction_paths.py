"""Paths of the eviction calls that options and sizes choose (bounds: tests/test_gpu_eviction.py)."""
import contextlib

import numpy as np
import pytest
import torch

import tvm_amd
from oracle import eviction
from tests.gpu_util import DEV, dev, host, i32
from tests.test_gpu_eviction import Pool, check_attention, prefill, queries
from tvm_amd import kernels

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def options(**chosen):
    previous = {name: tvm_amd.set_option(name, value) for name, value in chosen.items()}
    try:
        yield
    finally:
        for name, value in previous.items():
            tvm_amd.set_option(name, value)


@pytest.mark.parametrize("d", [64, 80, 96, 112, 128, 256])
@pytest.mark.parametrize("shares", [2, 3, 5, 6, 7, 8, 9, 33, 64])
def test_shares_of_prefill(shares, d):
    """Merge and weights in one launch and apart, shares without keys, rows behind the last sequence."""
    rng = np.random.default_rng(shares + d)
    for h_q, h_kv, q_lens, stored in ((8, 2, [5, 2, 0], [700, 40, 9]), (16, 2, [60, 1, 33], [150, 700, 30])):
        pool = Pool(rng, stored, h_kv, 16, d)
        n = sum(q_lens)
        q = queries(rng, n + 3, h_q, d)
        with options(prefill_kv_splits=shares):
            out, lse, sums = prefill(q, q_lens, pool, 1)
        assert (out[n:] == 7.0).all() and (lse[n:] == 7.0).all()
        check_attention(q[:n], q_lens, pool, True, 0, (out[:n], lse[:n], sums), f"{q_lens}")


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shares", [2, 3, 4, 5, 7, 8, 9, 64])
def test_shares_in_fp16(shares, d):
    """The plain call's shares are rounded to fp16 before they are merged: 2^-11 of sum w |v| more, also into a state that is there."""
    rng = np.random.default_rng(shares + d)
    for q_lens, stored in (([3, 2], [300, 140]), ([150, 90, 200], [160, 700, 300])):
        pool = Pool(rng, stored, 4, 16, d)
        q, n = queries(rng, sum(q_lens) + 2, 16, d), sum(q_lens)
        indptr, ids, info, _ = pool.table()
        zeros = i32([0] * len(q)), i32([0] * len(stored))
        out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV)
        lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device=DEV)
        with options(prefill_kv_splits=shares):
            kernels.batch_prefill_paged_kv(dev(q), i32(np.concatenate(([0], np.cumsum(q_lens)))), dev(pool.pages), indptr, ids, info, zeros[1],
                                           zeros[0], out, lse, 1, 0, 1.0, 1e4, d ** -0.5)
        out, lse = host(out), host(lse)
        assert (out[n:] == 7.0).all() and (lse[n:] == 7.0).all()
        want, want_lse, _, _, size = eviction.attention(q[:n], q_lens, pool.pages, pool.indptr, pool.ids, pool.info, True, d ** -0.5, pool.sums,
                                                        pool.weight_ids)
        largest = np.nanmax(np.abs(pool.pages[:, 1].astype(np.float64)))
        bound = 1.25 * (3 * 2.0 ** -11 * size + max(stored) * 2.0 ** -24 * largest) + 2.0 ** -24
        assert (np.abs(out[:n] - want) <= bound).all()
        reach = np.abs(q[:n].astype(np.float64)).sum(-1) * np.nanmax(np.abs(pool.pages[:, 0].astype(np.float64))) * d ** -0.5 * 1.4427
        assert (np.abs(lse[:n] - want_lse) <= ((d + 2) * reach + np.abs(want_lse) + 8) * 2.0 ** -23).all()
