"""Paths of the eviction calls that options and sizes choose (bounds: tests/test_gpu_eviction.py)."""
import contextlib

import numpy as np
import pytest
import torch

import tvm_amd
from oracle import eviction
from tests.gpu_util import DEV, dev, host, i32
from tests.test_gpu_eviction import Pool, check_attention, decode, prefill, queries, table_of, values
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


@pytest.mark.parametrize("stored", [[500], [1, 300, 17, 0], [900, 100, 100]])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_decode_with_chunks_and_separate_merges(d, stored):
    """Launches that add their own sums: several chunks a sequence; a merge of its own, which leaves the sums to another launch."""
    rng = np.random.default_rng(d + len(stored))
    pool = Pool(rng, stored, 2, 16, d)
    q = queries(rng, len(stored), 8, d)
    for chosen in (dict(decode_chunk_pages=8), dict(decode_separate_merge=1), dict(decode_separate_merge=1, decode_chunk_pages=8)):
        with options(**chosen):
            check_attention(q, [1] * len(stored), pool, False, 0, decode(q, pool), f"{chosen}")


def test_decode_whose_scores_are_not_kept():
    """More than 512 MiB of scores: K is read again.  A sequence of 2.1 million tokens on pages that repeat, with sums of their own."""
    rng = np.random.default_rng(70)
    h_q, h_kv, d, page, distinct, table = 64, 4, 64, 128, 40, 16700
    stored = [(table - 4) * page + 77, 300]
    assert table * page * h_q * 4 > 1 << 29
    pages = rng.standard_normal((distinct, 2, h_kv, page, d)).astype(np.float16)
    ids = rng.integers(0, distinct, table).astype(np.int32)
    weight_ids = rng.permutation(table).astype(np.int32)
    indptr, info = np.array([0, table - 3, table], np.int32), np.array([77, 300 - 2 * page], np.int32)
    before = rng.random((table, h_kv, page)).astype(np.float32)
    q = queries(rng, 2, h_q, d)
    sums, out = dev(before), torch.empty(q.shape, dtype=torch.float16, device=DEV)
    lse = torch.empty(q.shape[:2], device=DEV)
    kernels.batch_decode_paged_kv_weights(dev(q), dev(pages), i32(indptr), i32(ids), i32(info), out, lse, sums, i32(weight_ids), d ** -0.5)
    out, lse, sums = host(out), host(lse), host(sums)
    want_sums, slack = before.astype(np.float64), np.zeros(before.shape)
    for b, n in enumerate(stored):
        mine, weights = ids[indptr[b]:indptr[b + 1]], weight_ids[indptr[b]:indptr[b + 1]]
        times = np.zeros((distinct, page))  # how often a row is a token
        np.add.at(times, mine[:-1], 1.0)
        times[mine[-1], :info[b]] += 1.0
        for h in range(h_q):
            k, v = pages[:, 0, h // 16].astype(np.float64), pages[:, 1, h // 16].astype(np.float64)
            x = q[b, h].astype(np.float64)
            s, reach = k @ x * d ** -0.5 / np.log(2.0), np.abs(k) @ np.abs(x) * d ** -0.5 / np.log(2.0)
            top = s[times > 0].max()
            total = (times * np.exp2(s - top)).sum()
            want_lse = top + np.log2(total)
            w = np.exp2(s - want_lse)
            worst = reach[times > 0].max()
            want = np.einsum("pt,ptd->d", times * w, v)
            size = np.einsum("pt,ptd->d", times * w, np.abs(v))
            assert (np.abs(out[b, h] - want) <= 1.25 * (2.0 ** -10 * size + n * 2.0 ** -24 * np.abs(v).max()) + 2.0 ** -25).all()
            assert abs(lse[b, h] - want_lse) <= ((d + 2) * worst + abs(want_lse) + 8) * 2.0 ** -23
            rel = np.log(2.0) * ((d + 2) * (reach + worst) + 2 * abs(want_lse) + 8) * 2.0 ** -23 + (1 + 16 + 4) * 2.0 ** -23
            want_sums[weights[:-1], h // 16] += w[mine[:-1]]
            slack[weights[:-1], h // 16] += (rel * w)[mine[:-1]]
            want_sums[weights[-1], h // 16, :info[b]] += w[mine[-1], :info[b]]
            slack[weights[-1], h // 16, :info[b]] += (rel * w)[mine[-1], :info[b]]
    assert (np.abs(sums - want_sums) <= slack + want_sums * 2.0 ** -23).all()


def test_what_an_earlier_choice_left_in_scratch_memory_does_not_count():
    """Choices of other shapes on the same stream, in an order in which the words of one lie where the next has its histograms and counts of
    arrivals; the first needs the most memory, so that the buffer stays."""
    rng = np.random.default_rng(71)
    shapes = [([300000, 310000], [60000, 70000], 2, "sums"), ([33000, 34000], [4000, 7000], 1, "ties"), ([300000, 310000], [300, 290000], 2, "any"),
              ([40000], [30000], 1, "equal"), ([70000] + [1] * 20, [20000] * 21, 1, "ties"), ([33000, 36000], [4000, 35000], 2, "close"),
              ([36000, 33000, 40000], [4000, 7000, 100], 1, "sums")]
    stream = torch.cuda.Stream()
    for _ in range(2):
        for stored, keep, heads, kind in shapes:
            total, (indptr, info, weight_ids) = table_of(rng, stored, 64)
            sums = values(rng, kind, (total, heads, 64))
            kept = torch.full((len(stored), heads, max(keep)), 77, dtype=torch.int32, device=DEV)
            args = dev(sums), i32(indptr), i32(weight_ids), i32(info), i32(keep)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                kernels.select_kept_tokens(*args, kept, 4, 30)
            torch.cuda.synchronize()
            assert np.array_equal(host(kept), eviction.select(sums, indptr, weight_ids, info, keep, max(keep), 4, 30)), (stored, kind)


@pytest.mark.parametrize("begin, batch", [(30, 40), (30, 400), (210, 70), (1, 1)])
def test_some_sequences_of_a_larger_table(begin, batch):
    """page_indptr and q_indptr that do not begin at 0: rows, sums and pages of the other sequences stay as they are."""
    rng = np.random.default_rng(begin + batch)
    total = begin + batch + 25
    pool = Pool(rng, [int(n) for n in rng.integers(1, 60, total - 1)] + [500], 2, 16, 64)
    q_lens = [int(min(n, x)) for n, x in zip(rng.integers(0, 4, total), pool.stored)]
    some, pages, ids, weight_ids = slice(begin, begin + batch), dev(pool.pages), i32(pool.ids), i32(pool.weight_ids)
    whole = Pool.__new__(Pool)
    whole.__dict__.update(pool.__dict__, indptr=pool.indptr[begin:begin + batch + 1], info=pool.info[some], stored=pool.stored[some])
    indptr, info = i32(pool.indptr)[begin:begin + batch + 1], i32(pool.info)[some]
    q_indptr = np.concatenate(([0], np.cumsum(q_lens)))
    rows = slice(q_indptr[begin], q_indptr[begin + batch])
    others = np.ones(q_indptr[-1], bool)
    others[rows] = False

    def outputs(n):
        return (torch.full((n, 8, 64), 7.0, dtype=torch.float16, device=DEV), torch.full((n, 8), 7.0, device=DEV), dev(pool.sums))

    for chosen in (dict(), dict(decode_chunk_pages=8, prefill_kv_splits=3), dict(decode_separate_merge=1, prefill_kv_splits=7)):
        with options(**chosen):
            q = queries(rng, batch, 8, 64)
            out, lse, sums = outputs(batch)
            kernels.batch_decode_paged_kv_weights(dev(q), pages, indptr, ids, info, out, lse, sums, weight_ids, 0.125)
            check_attention(q, [1] * batch, whole, False, 0, (host(out), host(lse), host(sums)), f"decode {chosen}")
            plain = outputs(batch)
            zero = i32([0] * batch)
            kernels.batch_decode_paged_kv(dev(q), pages, indptr, ids, info, zero, zero, plain[0], plain[1], 0, 1.0, 1e4, 0.125)
            check_attention(q, [1] * batch, whole, False, 0, (host(plain[0]), host(plain[1]), host(sums)), f"plain decode {chosen}")
            q = queries(rng, q_indptr[-1], 8, 64)
            out, lse, sums = outputs(len(q))
            kernels.batch_prefill_paged_kv_weights(dev(q), i32(q_indptr)[begin:begin + batch + 1], pages, indptr, ids, info, out, lse, sums,
                                                   weight_ids, 1, 2, 0.125)
            out, lse = host(out), host(lse)
            check_attention(q[rows], q_lens[some], whole, True, 2, (out[rows], lse[rows], host(sums)), f"prefill {chosen}")
            assert (out[others] == 7.0).all() and (lse[others] == 7.0).all()
    kept = torch.full((batch, 2, 20), 77, dtype=torch.int32, device=DEV)
    kernels.select_kept_tokens(dev(pool.sums), indptr, weight_ids, info, i32([20] * batch), kept, 2, 5)
    want = eviction.select(pool.sums, whole.indptr, pool.weight_ids, whole.info, [20] * batch, 20, 2, 5)
    assert np.array_equal(host(kept), want)
    sums = dev(pool.sums)
    kernels.move_kept_tokens(pages, sums, indptr, ids, weight_ids, kept)
    want_pages, want_sums = eviction.move(pool.pages, pool.sums, whole.indptr, pool.ids, pool.weight_ids, want)
    assert np.array_equal(host(pages).view(np.uint16), want_pages.view(np.uint16)) and np.array_equal(host(sums), want_sums)


@pytest.mark.parametrize("stored, entries", [([600, 90], 400), ([5000, 2600], 4100), ([5000, 40], 2600)])
def test_move_of_lists_that_name_a_token_several_times(stored, entries):
    rng = np.random.default_rng(entries)
    pool = Pool(rng, stored, 2, 16, 64)
    kept = np.full((2, 2, entries), -1, np.int32)
    for b, n in enumerate(stored):
        for h in range(2):
            m = min(entries, n - n // 5)
            kept[b, h, :m] = np.maximum(np.sort(rng.integers(0, n, m)), np.arange(m))
    assert len(set(kept[0, 0].tolist())) < entries - 10
    indptr, ids, _, weight_ids = pool.table()
    pages, sums = dev(pool.pages), dev(pool.sums)
    kernels.move_kept_tokens(pages, sums, indptr, ids, weight_ids, i32(kept))
    want, want_sums = eviction.move(pool.pages, pool.sums, pool.indptr, pool.ids, pool.weight_ids, kept)
    assert np.array_equal(host(pages).view(np.uint16), want.view(np.uint16)) and np.array_equal(host(sums), want_sums)
