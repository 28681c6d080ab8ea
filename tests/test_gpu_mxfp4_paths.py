"""The kernels of the 4-bit cache on the paths that small launches do not take by themselves, against the definition in 64 bits
(oracle/mxfp4.py) within the bounds that tests/test_gpu_mxfp4.py derives."""
import contextlib

import numpy as np
import pytest
import torch

import tvm_amd
from oracle import mxfp4
from tests.gpu_util import DEV, dev, host, i32
from tests.test_gpu_mxfp4 import Pool, bound, compare, decode, prefill, rows_like
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


# ---- every number of rows that a work item takes ------------------------------------------------------------------------

EVERY_ITEM = [(d, blocks) for d in (64, 96, 128, 256) for blocks in (1, 2, 3) if d < 256 or blocks < 3]


@contextlib.contextmanager
def options(**values):
    previous = {name: tvm_amd.set_option(name, value) for name, value in values.items()}
    try:
        yield
    finally:
        for name, value in previous.items():
            tvm_amd.set_option(name, value)


def compare_where_finite(q, q_lens, pool, causal, out, lse, sm_scale):
    """NaN exactly where the definition has NaN, and elsewhere within the bound."""
    rows = mxfp4.rows_of(pool.pages, pool.d)
    want, want_lse = mxfp4.attention(q, q_lens, rows, pool.indptr, pool.ids, pool.info, causal, sm_scale)
    assert np.array_equal(np.isnan(out), np.isnan(want)) and np.array_equal(np.isnan(lse), np.isnan(want_lse))
    off = np.abs(out.astype(np.float64) - want) - bound(q, q_lens, pool, causal, sm_scale)
    assert np.nanmax(off, initial=-1.0) <= 0
    assert np.nanmax(np.abs(lse - want_lse), initial=0.0) <= 5e-5


@pytest.mark.parametrize("d, blocks", EVERY_ITEM)
@pytest.mark.parametrize("chunk", [0, 8])
def test_decode_of_every_item(d, blocks, chunk):
    """Groups of 40 and 17 heads: whole and partly filled blocks of rows; sequences whole and in chunks of 128 tokens."""
    rng = np.random.default_rng(d + blocks)
    for group, stored in ((40, [0, 1, 33, 129, 700, 1500]), (17, [16, 300, 2]), (3, [500, 31])):
        pool = Pool(rng, stored, 2, 16, d)
        q = (1.5 * rng.standard_normal((len(stored), 2 * group, d))).astype(np.float16)
        with options(mxfp4_row_blocks=blocks, decode_chunk_pages=chunk):
            out, lse = decode(q, pool, d ** -0.5)
        compare(q, [1] * len(stored), pool, False, out, lse, d ** -0.5)


@pytest.mark.parametrize("d, blocks", EVERY_ITEM)
@pytest.mark.parametrize("causal, shares", [(1, 1), (0, 1), (1, 3)])
def test_prefill_of_every_item(d, blocks, causal, shares):
    """Prompts that end in every part of an item of 16, 32 or 48 rows, with and without keys in front of them."""
    rng = np.random.default_rng(d + blocks + shares)
    stored, q_lens = [130, 5, 40, 0, 470, 70, 33, 16, 3], [130, 5, 17, 2, 11, 0, 33, 16, 6]
    for group in (1, 5):
        pool = Pool(rng, stored, 2, 32, d)
        q = (1.5 * rng.standard_normal((sum(q_lens), 2 * group, d))).astype(np.float16)
        with options(mxfp4_row_blocks=blocks, prefill_kv_splits=shares):
            out, lse = prefill(q, q_lens, pool, causal, d ** -0.5)
        compare(q, q_lens, pool, causal, out, lse, d ** -0.5)


@pytest.mark.parametrize("d, blocks", EVERY_ITEM)
def test_windows_with_sinks_of_every_item(d, blocks):
    rng = np.random.default_rng(7 * d + blocks)
    stored, q_lens = [120, 7, 45, 400, 60, 3], [40, 7, 30, 1, 44, 3]
    for sinks, evicted, shares, chunk in ((4, 13, 1, 0), (20, 50, 2, 8)):
        pool = Pool(rng, stored, 1, 16, d, sinks, evicted)
        for causal in (1, 0):
            q = (1.5 * rng.standard_normal((sum(q_lens), 6, d))).astype(np.float16)
            with options(mxfp4_row_blocks=blocks, prefill_kv_splits=shares):
                out, lse = prefill(q, q_lens, pool, causal, d ** -0.5)
            compare(q, q_lens, pool, causal, out, lse, d ** -0.5)
        q = (1.5 * rng.standard_normal((len(stored), 20, d))).astype(np.float16)
        with options(mxfp4_row_blocks=blocks, decode_chunk_pages=chunk):
            out, lse = decode(q, pool, d ** -0.5)
        compare(q, [1] * len(stored), pool, False, out, lse, d ** -0.5)


@pytest.mark.parametrize("d, blocks", EVERY_ITEM)
@pytest.mark.parametrize("split", [False, True])
def test_what_is_not_finite_stays_with_its_rows_in_every_item(d, blocks, split):
    """NaN keys and values behind the end, among evicted tokens and behind some of an item's queries reach the rows that see
    them and no others; so do NaN and infinite queries."""
    rng = np.random.default_rng(3 * d + blocks)
    stored, q_lens = [330, 100, 75], [60, 9, 40]
    pool = Pool(rng, stored, 1, 16, d, 4, 20)
    nan = np.full((1, 1, d), np.nan, np.float16)
    for b, t in ((0, 330), (1, 100), (1, 5), (1, 23), (2, 79)):  # seen by nobody
        pool.pages = mxfp4.append(pool.pages, nan, nan, [pool.slot(b, t)])
    for b, t, what in ((0, 300, "v"), (0, 317, "k"), (2, 50, "v"), (2, 72, "kv")):  # by the later queries
        k, v = rows_like(rng, 1, 1, d), rows_like(rng, 1, 1, d)
        if "k" in what:
            k[0, 0, 3] = np.inf
        if "v" in what:
            v[0, 0, d - 20] = np.nan
        pool.pages = mxfp4.append(pool.pages, k, v, [pool.slot(b, t)])
    q = rng.standard_normal((sum(q_lens), 5, d)).astype(np.float16)
    q[62, 1, 9] = np.nan
    with options(mxfp4_row_blocks=blocks, prefill_kv_splits=3 if split else 1, decode_chunk_pages=8 if split else 0):
        for causal in (1, 0):
            out, lse = prefill(q, q_lens, pool, causal, 0.1)
            compare_where_finite(q, q_lens, pool, causal, out, lse, 0.1)
        q = rng.standard_normal((3, 20, d)).astype(np.float16)
        q[1, 18] = np.nan
        out, lse = decode(q, pool, 0.1)
        compare_where_finite(q, [1] * 3, pool, False, out, lse, 0.1)


@pytest.mark.parametrize("d, blocks", EVERY_ITEM)
def test_items_of_more_than_512_runs(d, blocks):
    """A wave's page ids are those of 64 steps of eight runs: it reads more of them on the way."""
    rng = np.random.default_rng(d * blocks)
    stored = [8193, 17000, 5]
    pool = Pool(rng, stored, 1, 16, d)
    q = (1.5 * rng.standard_normal((3, 18, d))).astype(np.float16)
    with options(mxfp4_row_blocks=blocks, decode_chunk_pages=2048, prefill_kv_splits=1):
        out, lse = decode(q, pool, d ** -0.5)
        compare(q, [1] * 3, pool, False, out, lse, d ** -0.5)
        q = (1.5 * rng.standard_normal((7, 6, d))).astype(np.float16)
        out, lse = prefill(q, [3, 3, 1], pool, 1, d ** -0.5)
        compare(q, [3, 3, 1], pool, True, out, lse, d ** -0.5)


@pytest.mark.parametrize("d, blocks", EVERY_ITEM)
def test_rows_of_more_than_64_states(d, blocks):
    """Joined 64 at a time: of 80, 129 and 64 chunks of 128 tokens."""
    rng = np.random.default_rng(d * blocks + 1)
    stored = [80 * 128, 128 * 128 + 1, 100, 64 * 128]
    pool = Pool(rng, stored, 1, 16, d)
    q = (1.5 * rng.standard_normal((4, 19, d))).astype(np.float16)
    with options(mxfp4_row_blocks=blocks, decode_chunk_pages=8):
        out, lse = decode(q, pool, d ** -0.5)
    compare(q, [1] * 4, pool, False, out, lse, d ** -0.5)


@pytest.mark.parametrize("batch", [64, 65, 130, 512, 513, 700])
@pytest.mark.parametrize("blocks", [1, 3])
def test_batches_whose_sequences_have_several_items(batch, blocks):
    """Long sequences and prompts of several blocks at both ends of a batch and among the others, on every search path."""
    rng = np.random.default_rng(batch + blocks)
    stored = (rng.integers(0, 40, batch) * (rng.random(batch) < 0.8)).tolist()
    for b in (0, 1, 7, 8, 9, batch // 2, batch - 2, batch - 1):
        stored[b] = int(rng.integers(200, 1500))
    pool = Pool(rng, stored, 1, 16, 64)
    q = rng.standard_normal((batch, 20, 64)).astype(np.float16)
    with options(mxfp4_row_blocks=blocks, decode_chunk_pages=8):
        out, lse = decode(q, pool, 0.125)
    compare(q, [1] * batch, pool, False, out, lse, 0.125)
    q_lens = rng.integers(0, 3, batch).tolist()
    for b in (0, 3, 4, batch // 2, batch - 1):
        q_lens[b] = int(rng.integers(20, 70))
    q = rng.standard_normal((sum(q_lens), 3, 64)).astype(np.float16)
    for shares in (1, 2):
        with options(mxfp4_row_blocks=blocks, prefill_kv_splits=shares):
            out, lse = prefill(q, q_lens, pool, 1, 0.125)
        compare(q, q_lens, pool, True, out, lse, 0.125)


def test_more_row_blocks_than_there_are():
    """More blocks than there are kernels for give the largest there is."""
    rng = np.random.default_rng(2)
    for d in (128, 256):
        pool = Pool(rng, [100, 30], 1, 16, d)
        q = rng.standard_normal((2, 50, d)).astype(np.float16)
        with options(mxfp4_row_blocks=100):
            compare(q, [1, 1], pool, False, *decode(q, pool, 0.1), 0.1)
            compare(q, [1, 1], pool, True, *prefill(q, [1, 1], pool, 1, 0.1), 0.1)


def test_more_shares_than_there_are():
    """More shares than the option has give the most there are, as in the fp16 launches."""
    rng = np.random.default_rng(4)
    pool = Pool(rng, [9000, 30], 1, 16, 128)
    q = rng.standard_normal((4, 2, 128)).astype(np.float16)
    with options(prefill_kv_splits=64):
        want = prefill(q, [2, 2], pool, 1, 0.1)
    with options(prefill_kv_splits=100000):
        out = prefill(q, [2, 2], pool, 1, 0.1)
    assert all(np.array_equal(a, b) for a, b in zip(out, want))
    compare(q, [2, 2], pool, True, *out, 0.1)


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("k_scale, q_scale, v_scale", [(-18, 12, -21), (-22, 14, -22), (12, -11, 12), (11, 3, 11)])
def test_rows_of_every_magnitude(d, k_scale, q_scale, v_scale):
    """Values among fp16's subnormal numbers and near its largest, in keys and in values; scores that leave one key."""
    rng = np.random.default_rng(d + k_scale)
    stored, q_lens = [300, 17, 64], [20, 17, 3]
    pool = Pool(rng, stored, 2, 16, d)
    n = len(pool.pages) * 16
    k = (rng.uniform(-2, 2, (n, 2, d)) * 2.0 ** k_scale).astype(np.float16)
    v = (rng.uniform(-2, 2, (n, 2, d)) * 2.0 ** v_scale).astype(np.float16)
    pool.pages = mxfp4.append(pool.pages, k, v, np.arange(n))
    q = (rng.uniform(-2, 2, (sum(q_lens), 6, d)) * 2.0 ** q_scale).astype(np.float16)
    sm_scale = 2.0 ** min(0, -k_scale - q_scale) if k_scale < 0 else 1.0
    rows = mxfp4.rows_of(pool.pages, d)
    for q_here, lens, causal, (out, lse) in ((q, q_lens, 1, prefill(q, q_lens, pool, 1, sm_scale)), (q[:3], [1] * 3, 0, decode(q[:3], pool, sm_scale))):
        want, want_lse = mxfp4.attention(q_here, lens, rows, pool.indptr, pool.ids, pool.info, causal, sm_scale)
        # a score's float32 sum is off by up to D 2^-24 of the sum of its products' magnitudes, a weight by twice that part of itself
        # (the keys' scores against the row's largest), and a row by twice that part of A, which bound() has 1.25 * 2^-10 of
        most = d * np.abs(q_here.astype(np.float64)).max() * np.abs(rows[:, 0]).max() * sm_scale / np.log(2.0)
        shaky = 2 * d * 2.0 ** -24 * most
        limit = bound(q_here, lens, pool, causal, sm_scale) * (1 + 2 * shaky * 2.0 ** 10 / 1.25)
        assert (np.abs(out.astype(np.float64) - want) <= np.minimum(limit, 2 * np.abs(rows[:, 1]).max())).all()
        assert (np.abs(lse - want_lse) <= 5e-5 + shaky + 2.0 ** -22 * np.abs(want_lse)).all()
