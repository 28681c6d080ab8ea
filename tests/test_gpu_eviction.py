"""Eviction by attention weight against its definition in 64 bits (oracle/eviction.py).

Bounds.  Outputs: attention rounds the weights of a row to 11 bits and the output once more, an element is off by at most
2^-11 (A + |out|) <= 2^-10 A, A = sum w |v| / sum w; weights under fp16's normal range by up to 2^-25 of the largest one each: keys x
2^-24 max|v| (the reference point of a row may lie 2^8 under its maximum).  A quarter more for the float32 sums and exp2, 2^-25 for
outputs that are subnormal themselves.  Log-sum-exps and sums: a score is a float32 sum of d products, off by at most (d + 2) 2^-24
of the sum of their magnitudes, doubled, as the matrix instructions need not round to nearest; a weight is off by ln 2 times what
its score and its row's log-sum-exp are; the oracle adds this up over what a sum holds.  The choice and the move are exact."""
import numpy as np
import pytest
import torch

from oracle import eviction
from tests.gpu_util import DEV, dev, host, i32
from tvm_amd import kernels

pytestmark = pytest.mark.gpu


class Pool:
    """Sequences of given lengths on permuted pages of a pool whose other slots hold NaN, with sums on pages of their own."""

    def __init__(self, rng, stored, h_kv, page, d, dtype=np.float16):
        self.d, self.page, self.stored = d, page, list(stored)
        counts = [-(-n // page) for n in stored]
        total = sum(counts) + 3
        self.ids, self.weight_ids = (rng.permutation(total)[:sum(counts)].astype(np.int32) for _ in range(2))
        self.indptr = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
        self.info = np.array([n - (c - 1) * page if c else 0 for n, c in zip(stored, counts)], np.int32)
        self.pages = np.full((total, 2, h_kv, page, d), np.nan, dtype)
        self.sums = (rng.standard_normal((total, h_kv, page)) ** 2).astype(np.float32)
        channel = np.exp(0.6 * rng.standard_normal(d))
        for b, n in enumerate(stored):
            for t in range(n):
                at = (self.ids[self.indptr[b] + t // page], t % page)
                self.pages[at[0], :, :, at[1]] = rng.standard_normal((2, h_kv, d)) * channel
        # the slots behind a sequence's last token hold finite rows of sequences that are gone, as in a pool in use
        dead = np.isnan(self.pages[self.ids]) if len(self.ids) else None
        if dead is not None:
            rows = self.pages[self.ids]
            rows[dead] = rng.standard_normal(int(dead.sum())).astype(dtype)
            self.pages[self.ids] = rows

    def table(self):
        return i32(self.indptr), i32(self.ids), i32(self.info), i32(self.weight_ids)


def check_attention(q, q_lens, pool, causal, observed, got, what="", sm_scale=None):
    sm_scale = pool.d ** -0.5 if sm_scale is None else sm_scale
    out, lse, sums = got
    want, want_lse, want_sums, slack, size = eviction.attention(q, q_lens, pool.pages, pool.indptr, pool.ids, pool.info, causal, sm_scale,
                                                                pool.sums, pool.weight_ids, observed)
    keys = max(pool.stored, default=0)
    largest = np.nanmax(np.abs(pool.pages[:, 1].astype(np.float64)), initial=0.0)
    bound = 1.25 * (2.0 ** -10 * size + keys * 2.0 ** -24 * largest) + 2.0 ** -25
    off = np.abs(out.astype(np.float64) - want) - bound
    assert off.max(initial=-1.0) <= 0, f"{what}: output {off.max()} over the bound at {np.unravel_index(off.argmax(), off.shape)}"
    reach = np.abs(q.astype(np.float64)).sum(-1) * np.nanmax(np.abs(pool.pages[:, 0].astype(np.float64)), initial=0.0) * abs(sm_scale) * 1.4427
    off = np.abs(lse - want_lse) - ((pool.d + 2) * reach + np.abs(want_lse) + 8) * 2.0 ** -23
    assert off.max(initial=-1.0) <= 0, f"{what}: lse {off.max()} over the bound"
    off = np.abs(sums.astype(np.float64) - want_sums) - slack
    assert off.max(initial=-1.0) <= 0, f"{what}: sums {off.max()} over the bound at {np.unravel_index(off.argmax(), off.shape)}"
    untouched = np.ones(sums.shape, bool)
    for b, n in enumerate(pool.stored):
        t = np.arange(n)
        untouched[pool.weight_ids[pool.indptr[b] + t // pool.page], :, t % pool.page] = False
    assert np.array_equal(sums[untouched], pool.sums[untouched]), f"{what}: a slot without a token was written"


def decode(q, pool, sm_scale=None):
    indptr, ids, info, weight_ids = pool.table()
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device=DEV)
    sums = dev(pool.sums)
    kernels.batch_decode_paged_kv_weights(dev(q), dev(pool.pages), indptr, ids, info, out, lse, sums, weight_ids,
                                          pool.d ** -0.5 if sm_scale is None else sm_scale)
    return host(out), host(lse), host(sums)


def prefill(q, q_lens, pool, causal, observed=0):
    indptr, ids, info, weight_ids = pool.table()
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device=DEV)
    sums = dev(pool.sums)
    q_indptr = i32(np.concatenate(([0], np.cumsum(q_lens))))
    kernels.batch_prefill_paged_kv_weights(dev(q), q_indptr, dev(pool.pages), indptr, ids, info, out, lse, sums, weight_ids, causal,
                                           observed, pool.d ** -0.5)
    return host(out), host(lse), host(sums)


def queries(rng, n, h_q, d):
    return (1.5 * rng.standard_normal((n, h_q, d))).astype(np.float16)


HEADS = [(1, 1), (8, 2), (7, 1), (12, 4), (16, 1), (34, 2), (40, 1)]


# ---- attention that adds up weights ------------------------------------------------------------------------------


@pytest.mark.parametrize("d", [64, 80, 96, 112, 128, 256])
@pytest.mark.parametrize("h_q, h_kv", HEADS)
def test_decode(d, h_q, h_kv):
    rng = np.random.default_rng(d + h_q)
    page = (16, 32, 64, 128)[(d // 16 + h_q) % 4]
    stored = [1, 0, page, page + 1, 33, 2 * page - 1, 400, 0]
    pool = Pool(rng, stored, h_kv, page, d)
    q = queries(rng, len(stored), h_q, d)
    check_attention(q, [1] * len(stored), pool, False, 0, decode(q, pool))


@pytest.mark.parametrize("stored", [[2000], [5000, 1, 17], [130] * 70, [1, 40] * 300])
def test_decode_of_long_and_of_many_sequences(stored):
    rng = np.random.default_rng(len(stored))
    pool = Pool(rng, stored, 2, 16, 64)
    q = queries(rng, len(stored), 8, 64)
    check_attention(q, [1] * len(stored), pool, False, 0, decode(q, pool))


@pytest.mark.parametrize("d", [64, 80, 96, 112, 128, 256])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("observed", [0, 1, 5])
def test_prefill(d, causal, observed):
    rng = np.random.default_rng(d + causal)
    h_q, h_kv = HEADS[(d // 16 + observed) % len(HEADS)]
    page = (16, 32, 64, 128)[(d // 16 + causal) % 4]
    stored = [1, 0, page + 1, 33, 300, 145, 60]
    q_lens = [1, 0, 7, 33, 41, 1, 0]
    pool = Pool(rng, stored, h_kv, page, d)
    q = queries(rng, sum(q_lens), h_q, d)
    check_attention(q, q_lens, pool, causal, observed, prefill(q, q_lens, pool, causal, observed))


@pytest.mark.parametrize("observed", [0, 1, 3, 64, 1000])
def test_queries_in_front_of_every_key_and_sequences_without_keys_add_nothing(observed):
    rng = np.random.default_rng(observed)
    stored, q_lens = [5, 0, 40], [9, 4, 40]  # the first four queries of the first sequence see nothing
    pool = Pool(rng, stored, 2, 16, 128)
    q = queries(rng, sum(q_lens), 6, 128)
    out, lse, sums = prefill(q, q_lens, pool, 1, observed)
    check_attention(q, q_lens, pool, True, observed, (out, lse, sums))
    assert (out[:4] == 0).all() and (lse[:4] == -5e4).all() and (out[9:13] == 0).all() and (lse[9:13] == -5e4).all()


@pytest.mark.parametrize("q_len, stored", [(200, 700), (700, 700), (5, 3000), (130, 1)])
@pytest.mark.parametrize("observed", [0, 32])
def test_prefill_of_one_long_sequence(q_len, stored, observed):
    rng = np.random.default_rng(q_len)
    pool = Pool(rng, [stored], 2, 32, 128)
    q = queries(rng, q_len, 8, 128)
    check_attention(q, [q_len], pool, 1, observed, prefill(q, [q_len], pool, 1, observed))


def test_prefill_of_many_sequences():
    rng = np.random.default_rng(3)
    stored = [int(x) for x in rng.integers(0, 90, 150)]
    q_lens = [int(min(x, s)) for x, s in zip(rng.integers(0, 20, 150), stored)]
    pool = Pool(rng, stored, 3, 16, 64)
    q = queries(rng, sum(q_lens), 9, 64)
    check_attention(q, q_lens, pool, 1, 4, prefill(q, q_lens, pool, 1, 4))


@pytest.mark.parametrize("q_lens, stored", [([5, 3], [700, 2000]), ([40, 300], [900, 300])])
def test_rows_and_sums_behind_the_last_sequence_stay_as_they_are(q_lens, stored):
    """A padded batch: q, out and lse have rows that no sequence has, the page table entries that none has."""
    rng = np.random.default_rng(q_lens[0])
    pool = Pool(rng, stored, 2, 16, 128)
    q = queries(rng, sum(q_lens) + 7, 8, 128)
    pool.ids, pool.weight_ids = (np.concatenate((x, x[:1], x[:1])) for x in (pool.ids, pool.weight_ids))
    out, lse, sums = prefill(q, q_lens, pool, 1)
    n = sum(q_lens)
    assert (out[n:] == 7.0).all() and (lse[n:] == 7.0).all()
    check_attention(q[:n], q_lens, pool, True, 0, (out[:n], lse[:n], sums))


@pytest.mark.parametrize("d", [64, 80, 96, 112, 128, 256])
@pytest.mark.parametrize("causal, observed", [(1, 0), (0, 2), (1, 3)])
@pytest.mark.parametrize("q_lens, stored", [([5], [700]), ([70, 9], [2500, 700]), ([2, 1, 0, 3], [3000, 900, 40, 0]), ([4], [9000]), ([30] + [0] * 7, [1000] + [200] * 7),
                                            ([9, 1], [4, 600])])
def test_few_rows_on_long_sequences(q_lens, stored, d, causal, observed):
    """Launches in shares: of few and of many, a sequence with most of the rows, queries without keys."""
    rng = np.random.default_rng(sum(q_lens) + d)
    pool = Pool(rng, stored, 2, 64, d)
    q = queries(rng, sum(q_lens) + 2, 8, d)  # two rows are no sequence's
    out, lse, sums = prefill(q, q_lens, pool, causal, observed)
    n = sum(q_lens)
    assert (out[n:] == 7.0).all() and (lse[n:] == 7.0).all()
    check_attention(q[:n], q_lens, pool, causal, observed, (out[:n], lse[:n], sums))


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("causal, observed", [(1, 0), (0, 0), (1, 300)])
@pytest.mark.parametrize("h_q, h_kv, q_lens, stored", [(40, 1, [150, 0, 43], [261, 100, 229]), (12, 2, [700], [901]), (16, 1, [3, 190, 0, 90, 1], [500, 190, 33, 60, 0]),
                                                       (8, 1, [40] * 70, [40, 90] * 35)])
def test_many_rows_on_few_keys(h_q, h_kv, q_lens, stored, d, causal, observed):
    """Rows that workgroups share: unlike sequences, some without queries, queries without keys, batches of more than 64."""
    rng = np.random.default_rng(sum(q_lens) + d)
    pool = Pool(rng, stored, h_kv, 16, d)
    q = queries(rng, sum(q_lens) + 2, h_q, d)
    out, lse, sums = prefill(q, q_lens, pool, causal, observed)
    n = sum(q_lens)
    assert (out[n:] == 7.0).all() and (lse[n:] == 7.0).all()
    check_attention(q[:n], q_lens, pool, causal, observed, (out[:n], lse[:n], sums))


@pytest.mark.parametrize("h_q, h_kv", [(64, 1), (100, 1), (128, 1), (71, 1), (130, 2)])
def test_many_query_heads_on_one(h_q, h_kv):
    rng = np.random.default_rng(h_q)
    pool = Pool(rng, [300, 40, 1], h_kv, 16, 64)
    q = queries(rng, 3, h_q, 64)
    check_attention(q, [1] * 3, pool, False, 0, decode(q, pool))
    for q_lens in ([2, 1, 0], [50, 40, 1]):
        q = queries(rng, sum(q_lens), h_q, 64)
        check_attention(q, q_lens, pool, True, 0, prefill(q, q_lens, pool, 1))


def test_more_queries_observed_than_there_are():
    rng = np.random.default_rng(8)
    pool = Pool(rng, [300, 20], 2, 16, 64)
    q = queries(rng, 12, 8, 64)
    check_attention(q, [10, 2], pool, True, 0, prefill(q, [10, 2], pool, 1, (1 << 63) - 1))


def test_pools_of_more_than_4_gib():
    """Offsets of rows and of sums that 32 bits do not hold."""
    rng = np.random.default_rng(12)
    pool = Pool(rng, [200, 90], 8, 128, 128)
    high_pages, high_sums = 9000, 1 << 20  # 512 KiB a page, 4 KiB a page of sums
    big = torch.zeros((high_pages + len(pool.pages), 2, 8, 128, 128), dtype=torch.float16, device=DEV)
    big_sums = torch.zeros((high_sums + len(pool.sums), 8, 128), dtype=torch.float32, device=DEV)
    big[high_pages:] = dev(pool.pages)
    big_sums[high_sums:] = dev(pool.sums)
    indptr, ids, info, weight_ids = pool.table()
    ids, weight_ids = ids + high_pages, weight_ids + high_sums
    for q_lens in ([1, 1], [40, 3]):
        pool.sums = host(big_sums[high_sums:])
        q = queries(rng, sum(q_lens), 16, 128)
        out = torch.empty(q.shape, dtype=torch.float16, device=DEV)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=DEV)
        if q_lens == [1, 1]:
            kernels.batch_decode_paged_kv_weights(dev(q), big, indptr, ids, info, out, lse, big_sums, weight_ids, 128 ** -0.5)
        else:
            kernels.batch_prefill_paged_kv_weights(dev(q), i32([0, 40, 43]), big, indptr, ids, info, out, lse, big_sums, weight_ids, 1, 0,
                                                   128 ** -0.5)
        check_attention(q, q_lens, pool, True, 0, (host(out), host(lse), host(big_sums[high_sums:])))
    sums = host(big_sums[high_sums:])
    kept = torch.empty((2, 8, 80), dtype=torch.int32, device=DEV)
    kernels.select_kept_tokens(big_sums, indptr, weight_ids, info, i32([80, 60]), kept, 2, 20)
    want = eviction.select(sums, pool.indptr, pool.weight_ids, pool.info, [80, 60], 80, 2, 20)
    assert np.array_equal(host(kept), want)
    kernels.move_kept_tokens(big, big_sums, indptr, ids, weight_ids, kept)
    want_pages, want_sums = eviction.move(pool.pages, sums, pool.indptr, pool.ids, pool.weight_ids, want)
    assert np.array_equal(host(big[high_pages:]).view(np.uint16), want_pages.view(np.uint16))
    assert np.array_equal(host(big_sums[high_sums:]), want_sums)
    assert not big[:high_pages].any() and not big_sums[:high_sums].any()


def test_weights_of_a_query_add_up_to_one():
    rng = np.random.default_rng(4)
    pool = Pool(rng, [777], 1, 16, 128)
    pool.sums[:] = 0
    q = queries(rng, 1, 1, 128)
    assert abs(decode(q, pool)[2].astype(np.float64).sum() - 1) <= 1e-5


@pytest.mark.parametrize("scale", [0.0, -0.11, 4.0])
def test_scales(scale):
    rng = np.random.default_rng(5)
    pool = Pool(rng, [90, 300], 2, 16, 64)
    q = queries(rng, 2, 8, 64)
    check_attention(q, [1, 1], pool, False, 0, decode(q, pool, scale), sm_scale=scale)


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 65504.0])
def test_what_does_not_count_does_not_reach_the_sums(value):
    """Queries that are not observed, and the slots behind the last token."""
    rng = np.random.default_rng(6)
    pool = Pool(rng, [21, 40], 1, 32, 64)
    pool.pages[pool.ids[0], 0, :, 21:] = value
    q_lens = [5, 3]
    q = queries(rng, sum(q_lens), 4, 64)
    _, _, want, slack, _ = eviction.attention(q, q_lens, pool.pages, pool.indptr, pool.ids, pool.info, True, 64 ** -0.5, pool.sums,
                                              pool.weight_ids, observed=2)
    q[:3] = q[5] = value
    sums = prefill(q, q_lens, pool, 1, 2)[2]
    assert (np.abs(sums - want) <= slack).all()


def test_values_that_are_not_finite_stay_in_their_sequence():
    rng = np.random.default_rng(9)
    pool = Pool(rng, [50, 300, 20], 2, 16, 128)
    pool.pages[pool.ids[5], 0, 1, 3] = np.nan
    q = queries(rng, 3, 4, 128)
    sums = decode(q, pool)[2]
    clean = pool.pages.copy()
    clean[pool.ids[5], 0, 1, 3] = 0.0
    _, _, want, slack, _ = eviction.attention(q, [1] * 3, clean, pool.indptr, pool.ids, pool.info, False, 128 ** -0.5, pool.sums, pool.weight_ids)
    poisoned = np.zeros(sums.shape, bool)
    t = np.arange(300)
    poisoned[pool.weight_ids[pool.indptr[1] + t // 16], 1, t % 16] = True
    assert np.isnan(sums[poisoned]).all()
    assert (np.abs(sums - want) <= slack)[~poisoned].all()


def test_shared_pages_with_sums_of_their_own():
    """Two sequences on the same K/V pages: each has its own sums."""
    rng = np.random.default_rng(7)
    pool = Pool(rng, [70, 70], 2, 16, 128)
    pool.ids[5:9] = pool.ids[0:4]
    q = queries(rng, 2, 8, 128)
    check_attention(q, [1, 1], pool, False, 0, decode(q, pool))


def test_the_same_bits_again():
    rng = np.random.default_rng(8)
    pool = Pool(rng, [3000, 900, 20], 2, 16, 128)
    q = queries(rng, 3, 16, 128)
    first = decode(q, pool)
    for _ in range(3):
        assert all(np.array_equal(x, y) for x, y in zip(first, decode(q, pool)))


# ---- the choice --------------------------------------------------------------------------------------------------


def select(sums, pool_table, keep, max_keep, sinks, recent):
    indptr, info, weight_ids = pool_table
    kept = torch.full((len(keep), sums.shape[1], max_keep), 77, dtype=torch.int32, device=DEV)
    kernels.select_kept_tokens(dev(sums), i32(indptr), i32(weight_ids), i32(info), i32(keep), kept, sinks, recent)
    return host(kept)


def table_of(rng, stored, page):
    counts = [-(-n // page) for n in stored]
    total = sum(counts) + 2
    indptr = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    info = np.array([n - (c - 1) * page if c else 0 for n, c in zip(stored, counts)], np.int32)
    return total, (indptr, info, rng.permutation(total)[:sum(counts)].astype(np.int32))


def values(rng, kind, shape):
    if kind == "sums":
        return np.exp(2.0 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        return rng.integers(0, 4, shape).astype(np.float32)
    if kind == "equal":
        return np.zeros(shape, np.float32)
    if kind == "close":  # differ in the last bits alone
        return (1.0 + rng.integers(0, 300, shape) * 2.0 ** -23).astype(np.float32)
    x = rng.standard_normal(shape).astype(np.float32)  # "any"
    special = np.array([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38], np.float32)
    return np.where(rng.random(shape) < 0.5, special[rng.integers(0, len(special), shape)], x)


@pytest.mark.parametrize("kind", ["sums", "ties", "equal", "close", "any"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("sinks, recent", [(0, 0), (4, 16), (1, 0), (0, 63), (100, 200), (1 << 40, 1 << 40)])
def test_select(kind, page, sinks, recent):
    rng = np.random.default_rng(page + sinks % 97)
    stored = [1, 0, 63, 64, 65, 200, 500, 1500, 2, 130, 128, 300]
    keep = [1, 5, 64, 63, 64, 20, 128, 333, 1, 0, 127, -3]
    total, table = table_of(rng, stored, page)
    sums = values(rng, kind, (total, 3, page))
    for max_keep in (333, 90):
        want = eviction.select(sums, table[0], table[2], table[1], keep, max_keep, sinks, recent)
        assert np.array_equal(select(sums, table, keep, max_keep, sinks, recent), want)


@pytest.mark.parametrize("stored, keep, heads", [([70000], [5000], 2), ([300000], [60000], 1), ([5, 270000, 3000], [9, 269000, 500], 1)])
@pytest.mark.parametrize("kind", ["sums", "ties"])
def test_select_of_long_sequences(stored, keep, heads, kind):
    """In chunks, by several launches."""
    rng = np.random.default_rng(len(stored))
    total, table = table_of(rng, stored, 128)
    sums = values(rng, kind, (total, heads, 128))
    want = eviction.select(sums, table[0], table[2], table[1], keep, max(keep), 4, 700)
    assert np.array_equal(select(sums, table, keep, max(keep), 4, 700), want)


@pytest.mark.parametrize("stored, keep", [([70000] + [1] * 20, 20000), ([40000] + [10] * 5, 30000), ([300000] + [1] * 30, 100000),
                                          ([1000] * 9 + [0, 33000], 700)])
@pytest.mark.parametrize("kind", ["sums", "ties", "any"])
def test_select_of_a_long_sequence_among_short_ones(stored, keep, kind):
    """A workgroup a list, whose tokens are more than its registers hold, their bits more than its shared memory does."""
    rng = np.random.default_rng(len(stored))
    total, table = table_of(rng, stored, 32)
    sums = values(rng, kind, (total, 1, 32))
    want = eviction.select(sums, table[0], table[2], table[1], [keep] * len(stored), keep, 4, 100)
    assert np.array_equal(select(sums, table, [keep] * len(stored), keep, 4, 100), want)


@pytest.mark.parametrize("kind", ["ties", "equal", "close", "any"])
@pytest.mark.parametrize("stored, keep, sinks, recent", [([20000, 33000], [4096, 8192], 0, 0), ([50000], [49999], 4097, 4095), ([17000], [1], 0, 0),
                                                         ([17000], [0], 0, 0), ([40000], [30000], 0, 0), ([4096 * 9 + 1], [4097], 3, 1),
                                                         ([66000, 40000], [4096, 8192], 0, 0), ([40000], [1], 0, 0), ([40000], [0], 0, 0)])
def test_select_in_chunks(stored, keep, sinks, recent, kind):
    rng = np.random.default_rng(sinks + recent)
    total, table = table_of(rng, stored, 64)
    sums = values(rng, kind, (total, 2, 64))
    want = eviction.select(sums, table[0], table[2], table[1], keep, max(keep) + 5, sinks, recent)
    assert np.array_equal(select(sums, table, keep, max(keep) + 5, sinks, recent), want)


def test_select_of_many_sequences():
    rng = np.random.default_rng(11)
    stored = [int(x) for x in rng.integers(0, 300, 700)]
    keep = [int(x) for x in rng.integers(0, 200, 700)]
    total, table = table_of(rng, stored, 16)
    sums = values(rng, "sums", (total, 1, 16))
    assert np.array_equal(select(sums, table, keep, 180, 2, 10), eviction.select(sums, table[0], table[2], table[1], keep, 180, 2, 10))


# ---- the move ----------------------------------------------------------------------------------------------------


def move(pool, kept, with_sums=True):
    indptr, ids, _, weight_ids = pool.table()
    pages, sums = dev(pool.pages), dev(pool.sums) if with_sums else None
    kernels.move_kept_tokens(pages, sums, indptr, ids, weight_ids if with_sums else None, i32(kept))
    return host(pages), host(sums) if with_sums else None


def check_move(pool, kept, with_sums=True):
    pages, sums = move(pool, kept, with_sums)
    want, want_sums = eviction.move(pool.pages, pool.sums if with_sums else None, pool.indptr, pool.ids, pool.weight_ids, kept)
    bits = np.uint16 if pool.pages.dtype == np.float16 else np.uint32
    assert np.array_equal(pages.view(bits), want.view(bits))
    assert not with_sums or np.array_equal(sums, want_sums)


@pytest.mark.parametrize("d", [64, 80, 96, 112, 128, 256])
@pytest.mark.parametrize("recent", [0, 40, 300])
def test_move_of_what_select_chose(d, recent):
    rng = np.random.default_rng(d + recent)
    page = (16, 32, 64, 128)[d // 16 % 4]
    stored, keep = [700, 1, 0, 333, 64, 400], [400, 1, 5, 32, 64, 390]
    pool = Pool(rng, stored, 2, page, d)
    kept = eviction.select(pool.sums, pool.indptr, pool.weight_ids, pool.info, keep, 400, 4, recent)
    check_move(pool, kept)
    check_move(pool, kept, with_sums=False)


@pytest.mark.parametrize("d", [4, 60, 128, 256])
def test_move_of_float32_rows(d):
    rng = np.random.default_rng(d)
    pool = Pool(rng, [300, 90], 3, 16, d, np.float32)
    check_move(pool, eviction.select(pool.sums, pool.indptr, pool.weight_ids, pool.info, [100, 60], 100, 1, 20))


@pytest.mark.parametrize("heads", [1, 3])
def test_move_of_ascending_and_of_odd_lists(heads):
    """Ascending lists, as a caller's own choice gives; entries that name no token behind their place move nothing."""
    rng = np.random.default_rng(heads)
    pool = Pool(rng, [2000, 600, 40], heads, 16, 64)
    kept = np.full((3, heads, 1100), -1, np.int32)
    for h in range(heads):
        kept[0, h] = np.sort(rng.permutation(2000)[:1100])
        kept[1, h, :600 - 1 - h] = np.arange(1 + h, 600)  # every token by a few places
        kept[2, h, :8] = [0, 1, 1 << 30, 2, -5, 39, 6, 48]  # 48: behind the last page
    check_move(pool, kept)


@pytest.mark.parametrize("d, dtype", [(64, np.float16), (80, np.float16), (256, np.float16), (128, np.float32)])
@pytest.mark.parametrize("keep, recent", [([2600, 500, 9], 100), ([4800, 590, 30], 2500), ([2500, 600, 40], 2499), ([4999, 599, 39], 0)])
def test_move_of_long_lists(keep, recent, d, dtype):
    """By ranges of places; recent tokens that move by fewer places than they are."""
    rng = np.random.default_rng(d + recent)
    pool = Pool(rng, [5000, 600, 40], 1, 32, d, dtype)
    kept = eviction.select(pool.sums, pool.indptr, pool.weight_ids, pool.info, keep, keep[0], 4, recent)
    check_move(pool, kept)
    check_move(pool, kept, with_sums=False)


@pytest.mark.parametrize("heads", [1, 2])
def test_move_of_long_ascending_and_odd_lists(heads):
    rng = np.random.default_rng(heads)
    pool = Pool(rng, [5000, 2600, 40], heads, 16, 64)
    kept = np.full((3, heads, 2700), -1, np.int32)
    for h in range(heads):
        kept[0, h] = np.sort(rng.permutation(5000)[:2700])
        kept[1, h, :2600 - 1 - h] = np.arange(1 + h, 2600)
        kept[2, h, :8] = [0, 1, 1 << 30, 2, -5, 39, 6, 48]
        kept[2, h, 2650] = 2699  # behind the last page
    check_move(pool, kept)


# ---- together, streams, graphs -----------------------------------------------------------------------------------


def test_a_conversation_under_a_budget():
    """A prompt, answers token by token, evictions at a budget: outputs, sums and pages against the same steps in 64 bits."""
    rng = np.random.default_rng(20)
    h_q, h_kv, d, page, budget, slack_tokens = 8, 2, 128, 16, 96, 24
    pages_each = -(-(budget + slack_tokens) // page) + 6
    prompts = [150, 40]
    pages = np.zeros((2 * pages_each + 1, 2, h_kv, page, d), np.float16)
    sums = np.zeros((2 * pages_each, h_kv, page), np.float32)
    ids = [rng.permutation(2 * pages_each + 1)[:2 * pages_each].astype(np.int32)[b * pages_each:(b + 1) * pages_each] for b in range(2)]
    ids[1] = np.setdiff1d(np.arange(2 * pages_each + 1), ids[0])[:pages_each].astype(np.int32)
    weight_ids = [np.arange(b * pages_each, (b + 1) * pages_each, dtype=np.int32) for b in range(2)]
    d_pages, d_sums = dev(pages), dev(sums)
    length = [0, 0]
    pool = Pool(rng, [16], h_kv, page, d)
    for step in range(60):
        new = prompts if step == 0 else [1, 1]
        rows = rng.standard_normal((2, sum(new), h_kv, d)).astype(np.float16)
        slots, begin = [], 0
        for b in range(2):
            for t in range(length[b], length[b] + new[b]):
                slots.append(ids[b][t // page] * page + t % page)
                pages[ids[b][t // page], :, :, t % page] = rows[:, begin]
                sums[weight_ids[b][t // page], :, t % page] = 0  # a place that an evicted token had
                begin += 1
            length[b] += new[b]
        kernels.tir_kv_cache_transpose_append(d_pages, dev(rows[0]), dev(rows[1]), i32(slots))
        d_sums.view(-1)[:] = dev(sums).view(-1) if step == 0 else d_sums.view(-1)
        for b in range(2):  # the new tokens' sums begin at 0
            t = np.arange(length[b] - new[b], length[b])
            d_sums[torch.from_numpy(weight_ids[b][t // page].astype(np.int64)).to(DEV), :, torch.from_numpy(t % page).to(DEV)] = 0
        counts = [-(-n // page) for n in length]
        pool.stored, pool.pages, pool.sums = list(length), pages, sums
        pool.ids = np.concatenate([ids[b][:counts[b]] for b in range(2)])
        pool.weight_ids = np.concatenate([weight_ids[b][:counts[b]] for b in range(2)])
        pool.indptr = np.array([0, counts[0], counts[0] + counts[1]], np.int32)
        pool.info = np.array([n - (c - 1) * page for n, c in zip(length, counts)], np.int32)
        indptr, page_ids, info, w_ids = pool.table()
        q = queries(rng, sum(new), h_q, d)
        out = torch.empty(q.shape, dtype=torch.float16, device=DEV)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=DEV)
        if step == 0:
            kernels.batch_prefill_paged_kv_weights(dev(q), i32([0, new[0], sum(new)]), d_pages, indptr, page_ids, info, out, lse, d_sums, w_ids,
                                                   1, 32, d ** -0.5)
        else:
            kernels.batch_decode_paged_kv_weights(dev(q), d_pages, indptr, page_ids, info, out, lse, d_sums, w_ids, d ** -0.5)
        check_attention(q, new, pool, 1, 32, (host(out), host(lse), host(d_sums)), f"step {step}")
        sums = host(d_sums).copy()  # the kernel's own from here on, so that close sums do not choose differently
        if max(length) >= budget + slack_tokens:
            kept = torch.empty((2, h_kv, budget), dtype=torch.int32, device=DEV)
            kernels.select_kept_tokens(d_sums, indptr, w_ids, info, i32([budget, budget]), kept, 4, 16)
            kernels.move_kept_tokens(d_pages, d_sums, indptr, page_ids, w_ids, kept)
            want = eviction.select(sums, pool.indptr, pool.weight_ids, pool.info, [budget] * 2, budget, 4, 16)
            assert np.array_equal(host(kept), want)
            pages, sums = eviction.move(pages, sums, pool.indptr, pool.ids, pool.weight_ids, want)
            length = [min(n, budget) for n in length]
    assert np.array_equal(host(d_pages).view(np.uint16), pages.view(np.uint16)) and np.array_equal(host(d_sums), sums)


def step(pool, state, q, out, lse):
    """Decode, choice and move on what `state` has on the device."""
    kernels.batch_decode_paged_kv_weights(q, state["pages"], *state["table"][:3], out, lse, state["sums"], state["table"][3], pool.d ** -0.5)
    kernels.select_kept_tokens(state["sums"], state["table"][0], state["table"][3], state["table"][2], state["keep"], state["kept"], 2, 20)
    kernels.move_kept_tokens(state["pages"], state["sums"], state["table"][0], state["table"][1], state["table"][3], state["kept"])


def state_of(pool, keep, h_kv):
    return {"pages": dev(pool.pages), "sums": dev(pool.sums), "table": pool.table(), "keep": i32([keep] * len(pool.stored)),
            "kept": torch.zeros((len(pool.stored), h_kv, keep), dtype=torch.int32, device=DEV)}


def test_a_captured_step_replays():
    rng = np.random.default_rng(30)
    pool = Pool(rng, [900, 2500, 40], 2, 16, 128)
    q = dev(queries(rng, 3, 8, 128))
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        state = state_of(pool, 600, 2)
        step(pool, state, q, out, lse)  # what the kernels allocate is there
        state = state_of(pool, 600, 2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(pool, state, q, out, lse)
    for seed in (31, 32, 33):
        fresh = np.random.default_rng(seed)
        rows = [dev((fresh.standard_normal(pool.pages.shape)).astype(np.float16)), dev(fresh.random(pool.sums.shape).astype(np.float32))]
        new_q = dev(queries(fresh, 3, 8, 128))
        eager = state_of(pool, 600, 2)
        eager["pages"].copy_(rows[0])
        eager["sums"].copy_(rows[1])
        eager_out, eager_lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV)
        step(pool, eager, new_q, eager_out, eager_lse)
        torch.cuda.synchronize()
        state["pages"].copy_(rows[0])
        state["sums"].copy_(rows[1])
        q.copy_(new_q)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager_out) and torch.equal(lse, eager_lse) and torch.equal(state["kept"], eager["kept"])
        assert torch.equal(state["sums"], eager["sums"]) and torch.equal(state["pages"].view(torch.int16), eager["pages"].view(torch.int16))


@pytest.mark.parametrize("stored", [[30000, 20000, 9], [60000, 50000, 9]])
def test_a_captured_choice_of_long_lists_replays(stored):
    rng = np.random.default_rng(35)
    keep = [5000, 300, 50]
    total, (indptr, info, weight_ids) = table_of(rng, stored, 64)
    sums, kept = torch.zeros((total, 2, 64), device=DEV), torch.zeros((3, 2, 5000), dtype=torch.int32, device=DEV)
    args = (i32(indptr), i32(weight_ids), i32(info), i32(keep))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        kernels.select_kept_tokens(sums, *args, kept, 4, 30)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            kernels.select_kept_tokens(sums, *args, kept, 4, 30)
    for kind in ("sums", "ties", "any", "equal"):
        fresh = values(rng, kind, (total, 2, 64))
        torch.cuda.synchronize()
        sums.copy_(dev(fresh))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(kept), eviction.select(fresh, indptr, weight_ids, info, keep, 5000, 4, 30))
        eager = torch.empty_like(kept)
        kernels.select_kept_tokens(sums, *args, eager, 4, 30)
        assert torch.equal(kept, eager)


@pytest.mark.parametrize("h_q, h_kv, q_lens, stored", [(8, 2, [5], [700]), (8, 2, [5, 2, 0], [2000, 9000, 30]), (40, 1, [150, 43], [261, 229]),
                                                       (8, 2, [300], [900])])
def test_captured_prefill_replays(h_q, h_kv, q_lens, stored):
    """Shares of keys and of rows, their joins: each replay as the eager call, bit for bit."""
    rng = np.random.default_rng(sum(q_lens))
    pool = Pool(rng, stored, h_kv, 16, 128)
    indptr, ids, info, weight_ids = pool.table()
    pages, q_indptr = dev(pool.pages), i32(np.concatenate(([0], np.cumsum(q_lens))))
    q = torch.zeros((sum(q_lens), h_q, 128), dtype=torch.float16, device=DEV)

    def outputs():
        return torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV), dev(pool.sums)

    def call(out, lse, sums):
        kernels.batch_prefill_paged_kv_weights(q, q_indptr, pages, indptr, ids, info, out, lse, sums, weight_ids, 1, 0, 128 ** -0.5)

    got, stream = outputs(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call(*got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(*got)
    for _ in range(4):
        fresh, eager = queries(rng, len(q), h_q, 128), outputs()
        torch.cuda.synchronize()
        q.copy_(dev(fresh))
        got[2].copy_(dev(pool.sums))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        call(*eager)
        for x, y in zip(got, eager):
            assert torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0))
        check_attention(fresh, q_lens, pool, True, 0, tuple(host(x) for x in eager))


def test_prefill_on_two_streams_at_once():
    rng = np.random.default_rng(41)
    shapes = [([150, 43], [261, 229], 40, 1), ([5], [3000], 8, 2)]
    pools = [Pool(rng, stored, h_kv, 16, 128) for _, stored, _, h_kv in shapes]
    qs = [queries(rng, sum(q_lens), h_q, 128) for q_lens, _, h_q, _ in shapes]
    streams, calls = [torch.cuda.Stream() for _ in shapes], []
    for (q_lens, *_), pool, q, stream in list(zip(shapes, pools, qs, streams)) * 3:
        indptr, ids, info, weight_ids = pool.table()
        inputs = dev(q), i32(np.concatenate(([0], np.cumsum(q_lens)))), dev(pool.pages), indptr, ids, info
        outs = torch.zeros_like(inputs[0]), torch.zeros(q.shape[:2], device=DEV), dev(pool.sums)
        calls.append((inputs, outs, weight_ids, stream, q, q_lens, pool))
    torch.cuda.synchronize()
    for inputs, outs, weight_ids, stream, *_ in calls:
        with torch.cuda.stream(stream):
            kernels.batch_prefill_paged_kv_weights(*inputs, *outs, weight_ids, 1, 0, 128 ** -0.5)
    torch.cuda.synchronize()
    for _, outs, _, _, q, q_lens, pool in calls:
        check_attention(q, q_lens, pool, True, 0, tuple(host(x) for x in outs))


def test_scratch_counters_of_an_older_launch_do_not_count():
    import ctypes

    from tvm_amd._lib import check, lib
    rng = np.random.default_rng(36)
    total, table = table_of(rng, [30000, 40000], 64)
    sums = values(rng, "sums", (total, 1, 64))
    want = eviction.select(sums, table[0], table[2], table[1], [4000, 7000], 7000, 4, 30)
    for arrivals in (1, 3, 7):
        assert np.array_equal(select(sums, table, [4000, 7000], 7000, 4, 30), want)
        check(lib().tvmkv_debug_abandon_scratch_launches(ctypes.c_uint32(arrivals)))
    assert np.array_equal(select(sums, table, [4000, 7000], 7000, 4, 30), want)


def test_two_streams_at_once():
    rng = np.random.default_rng(40)
    pools = [Pool(rng, [3000, 700], 2, 16, 128), Pool(rng, [1500, 2600], 2, 16, 128)]
    q = [dev(queries(rng, 2, 8, 128)) for _ in pools]
    alone = []
    for pool, x in zip(pools, q):
        state, out, lse = state_of(pool, 500, 2), torch.zeros_like(x), torch.zeros(x.shape[:2], device=DEV)
        step(pool, state, x, out, lse)
        torch.cuda.synchronize()
        alone.append((out, lse, state["kept"], state["sums"], state["pages"].view(torch.int16)))
    streams = [torch.cuda.Stream() for _ in pools]
    states = [state_of(pool, 500, 2) for pool in pools]
    outs = [(torch.zeros_like(x), torch.zeros(x.shape[:2], device=DEV)) for x in q]
    torch.cuda.synchronize()
    for pool, x, stream, state, (out, lse) in zip(pools, q, streams, states, outs):
        with torch.cuda.stream(stream):
            step(pool, state, x, out, lse)
    torch.cuda.synchronize()
    for want, state, (out, lse) in zip(alone, states, outs):
        for x, y in zip(want, (out, lse, state["kept"], state["sums"], state["pages"].view(torch.int16))):
            assert torch.equal(x, y)


def test_tensor_level_entry_points():
    from tvm_amd import dlpack as dl
    rng = np.random.default_rng(50)
    pool = Pool(rng, [200, 90], 2, 16, 64)
    indptr, ids, info, weight_ids = pool.table()
    q = dev(queries(rng, 2, 8, 64))
    want = decode(host(q), pool)
    out, lse, sums, pages = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV), dev(pool.sums), dev(pool.pages)
    t = dl.tensor
    dl.call("batch_decode_paged_kv_weights", t(q), t(pages), t(indptr), t(ids), t(info), t(out), t(lse), t(sums), t(weight_ids), 0.125)
    assert np.array_equal(host(out), want[0]) and np.array_equal(host(lse), want[1]) and np.array_equal(host(sums), want[2])
    q_lens = [3, 2]
    q = dev(queries(rng, 5, 8, 64))
    want = prefill(host(q), q_lens, pool, 1, 2)
    out, lse, sums = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV), dev(pool.sums)
    dl.call("batch_prefill_paged_kv_weights", t(q), t(i32([0, 3, 5])), t(pages), t(indptr), t(ids), t(info), t(out), t(lse), t(sums),
            t(weight_ids), 1, 2, 0.125)
    assert np.array_equal(host(out), want[0]) and np.array_equal(host(lse), want[1]) and np.array_equal(host(sums), want[2])
    kept = torch.zeros((2, 2, 60), dtype=torch.int32, device=DEV)
    dl.call("select_kept_tokens", t(sums), t(indptr), t(weight_ids), t(info), t(i32([60, 50])), t(kept), 4, 8)
    want_kept = eviction.select(want[2], pool.indptr, pool.weight_ids, pool.info, [60, 50], 60, 4, 8)
    assert np.array_equal(host(kept), want_kept)
    dl.call("move_kept_tokens", t(pages), t(sums), t(indptr), t(ids), t(weight_ids), t(kept))
    want_pages, want_sums = eviction.move(pool.pages, want[2], pool.indptr, pool.ids, pool.weight_ids, want_kept)
    assert np.array_equal(host(pages).view(np.uint16), want_pages.view(np.uint16)) and np.array_equal(host(sums), want_sums)
    dl.call("move_kept_tokens", t(pages), None, t(indptr), t(ids), None, t(kept))
