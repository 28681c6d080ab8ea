"""The kernels of the 4-bit cache against its definition in 64 bits (oracle/mxfp4.py).

Bounds.  Writing and reading back are exact.  Attention rounds the weights of a row to 11 bits and the output once
more: an element is off by at most 2^-11 (A + |out|) <= 2^-10 A, A = sum w |v| / sum w.  Weights under fp16's normal range are
off by up to 2^-25 of the largest one each: keys x 2^-25 max|v|.  A quarter more for the float32 sums and exp2; outputs
themselves may be subnormal (2^-25).  The log-sum-exp's scores come from float32 sums of D products: 5e-5 at |score| <= 100."""
import numpy as np
import pytest
import torch

from oracle import mxfp4
from tests.gpu_util import DEV, dev, host, i32
from tvm_amd import kernels

pytestmark = pytest.mark.gpu


def rows_like(rng, *shape):
    """K or V rows with channels of unlike sizes."""
    return (rng.standard_normal(shape) * np.exp(0.6 * rng.standard_normal(shape[-1]))).astype(np.float16)


class Pool:
    """Sequences of given stored lengths on permuted pages of a pool whose other slots hold other rows."""

    def __init__(self, rng, stored, h_kv, page, d, sinks=0, evicted=None):
        self.d, self.page = d, page
        counts = [-(-n // page) for n in stored]
        total = sum(counts) + 3
        self.ids = rng.permutation(total)[:sum(counts)].astype(np.int32)
        self.indptr = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
        k, v = rows_like(rng, total * page, h_kv, d), rows_like(rng, total * page, h_kv, d)
        self.pages = mxfp4.append(mxfp4.empty_pages(total, h_kv, page, d), k, v, np.arange(total * page))
        last = np.array([n - (c - 1) * page if c else 0 for n, c in zip(stored, counts)], np.int32)
        self.info = last
        if evicted is not None:
            sink = np.minimum(sinks, stored)
            self.info = np.stack((last, np.minimum(sink + evicted, stored), sink)).astype(np.int32)

    def slot(self, b, t):
        return self.ids[self.indptr[b] + t // self.page] * self.page + t % self.page

    def device(self):
        return dev(self.pages), i32(self.indptr), i32(self.ids), i32(self.info)


def bound(q, q_lens, pool, causal, sm_scale):
    """A of the module's comment: attention with the same weights over |v|, and keys x max|v|."""
    rows = mxfp4.rows_of(pool.pages, pool.d)
    sizes = rows.copy()
    sizes[:, 1] = np.abs(sizes[:, 1])
    a, _ = mxfp4.attention(q, q_lens, sizes, pool.indptr, pool.ids, pool.info, causal, sm_scale)
    keys = np.diff(pool.indptr).max(initial=0) * pool.page
    return 1.25 * (2.0 ** -10 * a + keys * 2.0 ** -25 * np.nanmax(sizes[:, 1], initial=0.0)) + 2.0 ** -25


def compare(q, q_lens, pool, causal, out, lse, sm_scale, what=""):
    rows = mxfp4.rows_of(pool.pages, pool.d)
    want, want_lse = mxfp4.attention(q, q_lens, rows, pool.indptr, pool.ids, pool.info, causal, sm_scale)
    off = np.abs(out.astype(np.float64) - want) - bound(q, q_lens, pool, causal, sm_scale)
    assert off.max(initial=-1.0) <= 0, f"{what}: {off.max()} over the bound at {np.unravel_index(off.argmax(), off.shape)}"
    assert np.abs(lse - want_lse).max(initial=0.0) <= 5e-5, what


def decode(q, pool, sm_scale):
    pages, indptr, ids, info = pool.device()
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device=DEV)
    kernels.mxfp4_batch_decode_paged_kv(dev(q), pages, indptr, ids, info, out, lse, sm_scale)
    return host(out), host(lse)


def prefill(q, q_lens, pool, causal, sm_scale):
    pages, indptr, ids, info = pool.device()
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device=DEV)
    q_indptr = i32(np.concatenate(([0], np.cumsum(q_lens))))
    kernels.mxfp4_batch_prefill_paged_kv(dev(q), q_indptr, pages, indptr, ids, info, out, lse, causal, sm_scale)
    return host(out), host(lse)


# ---- writing and reading back -------------------------------------------------------------------------------------


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("h_kv, page", [(1, 16), (3, 48), (8, 128)])
def test_append_and_read_are_exact(d, h_kv, page):
    rng = np.random.default_rng(d + page)
    total = 4 * page
    n = 77 if total > 80 else 41
    slots = rng.permutation(total)[:n].astype(np.int32)
    slots[5] = slots[17] = -1
    k, v = rows_like(rng, n, h_kv, d), rows_like(rng, n, h_kv, d)
    bits = rng.integers(0, 1 << 16, (4, h_kv, d)).astype(np.uint16)  # any pattern, infinities and NaN among them
    k[:4] = bits.view(np.float16)
    k[4], v[0], v[1, 0, :32] = 0.0, -0.0, np.float16(65504)
    v[2] = (rng.standard_normal((h_kv, d)) * 1e-6).astype(np.float16)
    v[3, 0, 7], v[4, -1, -1] = np.nan, -np.inf
    before = rng.integers(0, 200, (4, 2, h_kv, page, 17 * d // 32)).astype(np.uint8)
    pages = dev(before)
    kernels.mxfp4_append(pages, dev(k), dev(v), i32(slots))
    with np.errstate(invalid="ignore"):
        want = mxfp4.append(before, k, v, slots)
    assert np.array_equal(host(pages), want)  # the other slots' bytes as they were
    # written slots, one more that nothing wrote, and a negative one
    at = np.concatenate((slots, [-1])).astype(np.int32)
    k_back, v_back = (torch.full((len(at), h_kv, d), 3.0, dtype=torch.float16, device=DEV) for _ in range(2))
    kernels.mxfp4_read_kv(pages, i32(at), k_back, v_back)
    for which, (rows, back) in enumerate(((k, k_back), (v, v_back))):
        expect = np.zeros((len(at), h_kv, d))
        with np.errstate(invalid="ignore"):
            expect[:n] = mxfp4.rounded(rows)
        expect[at < 0] = 0
        assert np.array_equal(host(back).astype(np.float64), expect, equal_nan=True)


def test_every_fp16_value_is_written_as_defined():
    x = np.arange(1 << 16, dtype=np.uint32).astype(np.uint16).view(np.float16)
    rng = np.random.default_rng(3)
    for scale_bits in (0, 0x2c00, 0x5000):  # blocks led by 0, 1/16 and 32, so that every value meets small and large scales
        rows = np.repeat(x[:, None], 32, 1)
        rows[:, 1] = np.uint16(scale_bits).view(np.float16)
        k = rows.reshape(-1, 16, 128)
        slots = rng.permutation(len(k)).astype(np.int32)
        pages = kernels.mxfp4_pages(len(k) // 16, 16, 16, 128)
        kernels.mxfp4_append(pages, dev(k), dev(k[::-1]), i32(slots))
        back = [torch.empty(k.shape, dtype=torch.float16, device=DEV) for _ in range(2)]
        kernels.mxfp4_read_kv(pages, i32(slots), *back)
        with np.errstate(invalid="ignore"):
            want = mxfp4.rounded(k)
        assert np.array_equal(host(back[0]).astype(np.float64), want, equal_nan=True)
        assert np.array_equal(host(back[1]).astype(np.float64), want[::-1], equal_nan=True)


# ---- decode -------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("d, h_q, h_kv, page", [(128, 32, 8, 16), (64, 28, 4, 32), (96, 9, 3, 48), (256, 16, 2, 64), (128, 32, 1, 16),
                                                (128, 40, 1, 128), (64, 2, 2, 16)])
def test_decode(d, h_q, h_kv, page):
    rng = np.random.default_rng(h_q + d)
    stored = [0, 1, 15, 16, 17, 31, 32, 33, 0, 63, 64, 129, 500, 1111]
    pool = Pool(rng, stored, h_kv, page, d)
    q = (1.5 * rng.standard_normal((len(stored), h_q, d))).astype(np.float16)
    out, lse = decode(q, pool, d ** -0.5)
    compare(q, [1] * len(stored), pool, False, out, lse, d ** -0.5)


@pytest.mark.parametrize("d, page, sinks, evicted", [(128, 16, 4, 9), (64, 32, 1, 80), (256, 16, 16, 16), (96, 16, 20, 33)])
def test_decode_over_windows_with_sinks(d, page, sinks, evicted):
    rng = np.random.default_rng(sinks)
    stored = [1, 3, sinks, sinks + 1, sinks + evicted, sinks + evicted + 1, 200, 333, 0]
    pool = Pool(rng, stored, 2, page, d, sinks, evicted)
    q = (1.5 * rng.standard_normal((len(stored), 8, d))).astype(np.float16)
    out, lse = decode(q, pool, d ** -0.5)
    compare(q, [1] * len(stored), pool, False, out, lse, d ** -0.5)


def test_more_sinks_than_stored_tokens_are_all_of_them():
    rng = np.random.default_rng(11)
    stored = [5, 1, 40]
    pool = Pool(rng, stored, 2, 16, 128, 0, 0)
    q = rng.standard_normal((3, 8, 128)).astype(np.float16)
    want, want_lse = decode(q, pool, 0.1)
    for window in (0, 5, 40):
        pool.info = np.stack((pool.info[0], np.minimum(window, stored), np.full(3, 1000))).astype(np.int32)
        out, lse = decode(q, pool, 0.1)
        assert np.array_equal(out, want) and np.array_equal(lse, want_lse), window


@pytest.mark.parametrize("stored", [[20000], [9000, 1, 7000], [4100] * 3])
def test_decode_of_long_sequences_is_split_and_joined(stored):
    rng = np.random.default_rng(len(stored))
    pool = Pool(rng, stored, 2, 16, 128)
    q = (1.5 * rng.standard_normal((len(stored), 8, 128))).astype(np.float16)
    out, lse = decode(q, pool, 0.1)
    compare(q, [1] * len(stored), pool, False, out, lse, 0.1)


@pytest.mark.parametrize("heads, d, stored", [
    (64, 64, [3000, 5000, 100, 0]), (64, 64, [1, 9000]), (64, 64, [2500, 2500, 2500]), (16, 128, [17, 20000, 1, 9000, 4000]),  # chunks that the lengths decide
    (128, 64, [1500, 1600, 1550, 1500]), (128, 64, [1500, 3100, 200, 1500])])  # sequences left whole, and not
def test_decode_whose_chunks_the_device_chooses(heads, d, stored):
    rng = np.random.default_rng(sum(stored))
    pool = Pool(rng, stored, heads, 16, d)
    q = rng.standard_normal((len(stored), heads, d)).astype(np.float16)
    compare(q, [1] * len(stored), pool, False, *decode(q, pool, d ** -0.5), d ** -0.5)


def test_decode_of_many_short_sequences():
    rng = np.random.default_rng(8)
    stored = rng.integers(0, 40, 300)
    pool = Pool(rng, stored.tolist(), 2, 16, 64)
    q = rng.standard_normal((300, 4, 64)).astype(np.float16)
    out, lse = decode(q, pool, 0.125)
    compare(q, [1] * 300, pool, False, out, lse, 0.125)


@pytest.mark.parametrize("batch", [64, 65, 130, 512, 513, 700])
def test_batches_of_every_search_path(batch):
    """A work item finds its sequence by one lane a sequence, by some sequences a lane, or by a search over all."""
    rng = np.random.default_rng(batch)
    stored = (rng.integers(0, 40, batch) * (rng.random(batch) < 0.8)).tolist()
    stored[0], stored[-1] = 0, 33
    pool = Pool(rng, stored, 1, 16, 64)
    q = rng.standard_normal((batch, 2, 64)).astype(np.float16)
    out, lse = decode(q, pool, 0.125)
    compare(q, [1] * batch, pool, False, out, lse, 0.125)
    q_lens = rng.integers(0, 4, batch).tolist()
    q = rng.standard_normal((sum(q_lens), 2, 64)).astype(np.float16)
    out, lse = prefill(q, q_lens, pool, 1, 0.125)
    compare(q, q_lens, pool, True, out, lse, 0.125)


@pytest.mark.parametrize("sm_scale", [-0.1, 0.0, 1.0])
def test_scales_of_either_sign_and_none(sm_scale):
    rng = np.random.default_rng(18)
    pool = Pool(rng, [70, 1, 300], 2, 16, 128)
    q = (0.3 * rng.standard_normal((3, 8, 128))).astype(np.float16)
    out, lse = decode(q, pool, sm_scale)
    compare(q, [1] * 3, pool, False, out, lse, sm_scale)
    q = (0.3 * rng.standard_normal((40, 8, 128))).astype(np.float16)
    out, lse = prefill(q, [30, 1, 9], pool, 1, sm_scale)
    compare(q, [30, 1, 9], pool, True, out, lse, sm_scale)


def test_decode_with_sharp_and_flat_weights():
    """Scores far apart (one key takes all) and all equal; the running maximum rises at the very end of a sequence."""
    rng = np.random.default_rng(9)
    pool = Pool(rng, [700, 700, 700], 1, 16, 128)
    q = np.zeros((3, 4, 128), np.float16)
    q[0] = 12 * rng.standard_normal((4, 128))
    k, v = rows_like(rng, 2, 1, 128), rows_like(rng, 2, 1, 128)
    q[2] = rng.standard_normal((4, 128))
    k[0] = 6 * q[2, 0]
    k[1] = -6 * q[2, 1]
    pool.pages = mxfp4.append(pool.pages, k, v, [pool.slot(2, 699), pool.slot(2, 3)])
    out, lse = decode(q, pool, 128 ** -0.5)
    compare(q, [1] * 3, pool, False, out, lse, 128 ** -0.5)


# ---- prefill ------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("causal", [1, 0])
@pytest.mark.parametrize("d, h_q, h_kv, page", [(128, 8, 2, 16), (64, 7, 1, 32), (96, 3, 3, 16), (256, 4, 2, 48), (128, 17, 1, 64)])
def test_prefill(causal, d, h_q, h_kv, page):
    rng = np.random.default_rng(d + h_q)
    stored = [1, 5, 40, 0, 130, 70, 33, 64, 3]
    q_lens = [1, 5, 17, 2, 130, 0, 40, 1, 6]  # the fourth and the last have queries without keys
    pool = Pool(rng, stored, h_kv, page, d)
    q = (1.5 * rng.standard_normal((sum(q_lens), h_q, d))).astype(np.float16)
    out, lse = prefill(q, q_lens, pool, causal, d ** -0.5)
    compare(q, q_lens, pool, causal, out, lse, d ** -0.5)


@pytest.mark.parametrize("causal", [1, 0])
@pytest.mark.parametrize("q_lens, stored", [([3], [3000]), ([300], [1500]), ([260, 9, 31], [260, 900, 31]), ([5] * 90, [60] * 90)])
def test_prefill_of_long_and_many_sequences(causal, q_lens, stored):
    rng = np.random.default_rng(len(stored) + causal)
    pool = Pool(rng, stored, 2, 16, 128)
    q = (1.5 * rng.standard_normal((sum(q_lens), 4, 128))).astype(np.float16)
    out, lse = prefill(q, q_lens, pool, causal, 0.1)
    compare(q, q_lens, pool, causal, out, lse, 0.1)


@pytest.mark.parametrize("causal", [1, 0])
@pytest.mark.parametrize("d, sinks, evicted", [(128, 4, 13), (64, 16, 40), (256, 1, 5)])
def test_prefill_over_windows_with_sinks(causal, d, sinks, evicted):
    rng = np.random.default_rng(d + sinks)
    stored, q_lens = [120, 7, 45, 200, 60], [9, 7, 30, 1, 44]
    pool = Pool(rng, stored, 2, 16, d, sinks, evicted)
    q = (1.5 * rng.standard_normal((sum(q_lens), 8, d))).astype(np.float16)
    out, lse = prefill(q, q_lens, pool, causal, d ** -0.5)
    compare(q, q_lens, pool, causal, out, lse, d ** -0.5)


def test_prefill_of_one_token_is_decode():
    rng = np.random.default_rng(10)
    stored = [1, 40, 700, 0, 65]
    pool = Pool(rng, stored, 2, 16, 128)
    q = rng.standard_normal((5, 8, 128)).astype(np.float16)
    out, lse = prefill(q, [1] * 5, pool, 1, 0.1)
    compare(q, [1] * 5, pool, True, out, lse, 0.1)


# ---- what is not finite ---------------------------------------------------------------------------------------------


def test_nan_in_places_that_are_not_seen():
    """Behind the end, among the evicted tokens and behind a causal query, NaN rows reach nothing; where they are seen they do."""
    rng = np.random.default_rng(11)
    d, nan = 128, np.full((1, 2, 128), np.nan, np.float16)
    pool = Pool(rng, [40, 100, 130], 2, 16, d, 4, 20)
    hidden = ((0, 40), (0, 47), (1, 4), (1, 23), (2, 10), (2, 130))
    for b, t in hidden:
        pool.pages = mxfp4.append(pool.pages, nan, nan, [pool.slot(b, t)])
    q = rng.standard_normal((3, 8, d)).astype(np.float16)
    out, lse = decode(q, pool, 0.1)
    assert np.isfinite(out).all()
    one = np.ones((1, 2, d), np.float16)
    for b, t in hidden:  # any finite row there gives the same
        pool.pages = mxfp4.append(pool.pages, one, one, [pool.slot(b, t)])
    again, again_lse = decode(q, pool, 0.1)
    assert np.array_equal(out, again) and np.array_equal(lse, again_lse)
    compare(q, [1] * 3, pool, False, out, lse, 0.1)


@pytest.mark.parametrize("d, q_len, stored", [(128, 20, 50), (96, 20, 50), (256, 9, 40), (64, 300, 300)])
def test_nan_values_behind_a_causal_query(d, q_len, stored):
    rng = np.random.default_rng(d)
    pool = Pool(rng, [stored], 1, 16, d)
    at = stored - q_len // 2  # the token of the middle query, roughly
    v = rows_like(rng, 1, 1, d)
    v[0, 0, 35] = np.nan  # one block of 32
    slot = pool.slot(0, at)
    k = mxfp4.rows_of(pool.pages, d)[slot // 16, 0, :, slot % 16][None].astype(np.float16)
    pool.pages = mxfp4.append(pool.pages, k, v, [slot])
    q = rng.standard_normal((q_len, 4, d)).astype(np.float16)
    out, lse = prefill(q, [q_len], pool, 1, 0.1)
    sees = np.arange(q_len) + stored - q_len >= at
    assert np.isnan(out[sees][:, :, 32:64]).all()
    rest = np.ones(d, bool)
    rest[32:64] = False
    assert np.isfinite(out[sees][:, :, rest]).all() and np.isfinite(out[~sees]).all() and np.isfinite(lse).all()


def test_nan_keys_and_queries_stay_with_their_rows():
    rng = np.random.default_rng(12)
    pool = Pool(rng, [50, 50], 2, 16, 128)
    bad = np.zeros((1, 2, 128), np.float16)
    bad[0, 0, 3] = np.inf  # the first head's key
    pool.pages = mxfp4.append(pool.pages, bad, np.ones((1, 2, 128), np.float16), [pool.slot(0, 20)])
    q = rng.standard_normal((2, 8, 128)).astype(np.float16)
    q[1, 5] = np.nan
    out, lse = decode(q, pool, 0.1)
    assert np.isnan(out[0, :4]).all() and np.isfinite(out[0, 4:]).all()
    assert np.isnan(out[1, 5]).all() and np.isfinite(np.delete(out[1], 5, 0)).all()


# ---- memory, streams, graphs ---------------------------------------------------------------------------------------


def test_pools_of_more_than_4_gib():
    rng = np.random.default_rng(13)
    d, h_kv, page = 128, 8, 128
    per_page = 2 * h_kv * page * 17 * d // 32
    total = (9 << 29) // per_page  # 4.5 GiB
    pool = torch.zeros((total, 2, h_kv, page, 17 * d // 32), dtype=torch.uint8, device=DEV)
    ids = np.array([total - 1, 0, total - 3, total // 2], np.int32)
    n = 3 * page + 50
    k, v = rows_like(rng, n, h_kv, d), rows_like(rng, n, h_kv, d)
    slots = (ids[np.arange(n) // page] * page + np.arange(n) % page).astype(np.int32)
    kernels.mxfp4_append(pool, dev(k), dev(v), i32(slots))
    back = [torch.empty((n, h_kv, d), dtype=torch.float16, device=DEV) for _ in range(2)]
    kernels.mxfp4_read_kv(pool, i32(slots), *back)
    assert np.array_equal(host(back[0]).astype(np.float64), mxfp4.rounded(k))
    assert np.array_equal(host(back[1]).astype(np.float64), mxfp4.rounded(v))
    small = Pool(rng, [n], h_kv, page, d)
    small.ids = np.arange(4, dtype=np.int32)
    small.pages = mxfp4.append(mxfp4.empty_pages(4, h_kv, page, d), k, v, np.arange(n))
    q = rng.standard_normal((1, 16, d)).astype(np.float16)
    out, lse = torch.empty((1, 16, d), dtype=torch.float16, device=DEV), torch.empty((1, 16), device=DEV)
    kernels.mxfp4_batch_decode_paged_kv(dev(q), pool, i32([0, 4]), i32(ids), i32([50]), out, lse, 0.1)
    compare(q, [1], small, False, host(out), host(lse), 0.1)
    kernels.mxfp4_batch_prefill_paged_kv(dev(q), i32([0, 1]), pool, i32([0, 4]), i32(ids), i32([50]), out, lse, 1, 0.1)
    compare(q, [1], small, True, host(out), host(lse), 0.1)


def test_calls_on_two_streams_do_not_meet():
    rng = np.random.default_rng(14)
    pools = [Pool(rng, [3000, 50], 2, 16, 128), Pool(rng, [2500, 900], 2, 16, 128)]
    qs = [rng.standard_normal((2, 8, 128)).astype(np.float16) for _ in pools]
    streams = [torch.cuda.Stream() for _ in pools]
    state = [(dev(q), *pool.device(), torch.empty((2, 8, 128), dtype=torch.float16, device=DEV), torch.empty((2, 8), device=DEV))
             for q, pool in zip(qs, pools)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, args in zip(streams, state):
            with torch.cuda.stream(s):
                kernels.mxfp4_batch_decode_paged_kv(*args, 0.1)
    torch.cuda.synchronize()
    for q, pool, args in zip(qs, pools, state):
        compare(q, [1, 1], pool, False, host(args[-2]), host(args[-1]), 0.1)


def test_a_step_can_be_captured():
    """Append and decode of a step in a graph, replayed with other rows and queries between eager calls."""
    rng = np.random.default_rng(15)
    pool = Pool(rng, [2000, 77, 500], 2, 16, 128)
    pages, indptr, ids, info = pool.device()
    slots = np.array([pool.slot(b, n - 1) for b, n in enumerate((2000, 77, 500))], np.int32)
    k, v = (torch.zeros((3, 2, 128), dtype=torch.float16, device=DEV) for _ in range(2))
    q = torch.zeros((3, 8, 128), dtype=torch.float16, device=DEV)
    out, lse = torch.empty((3, 8, 128), dtype=torch.float16, device=DEV), torch.empty((3, 8), device=DEV)
    at = i32(slots)

    def step():
        kernels.mxfp4_append(pages, k, v, at)
        kernels.mxfp4_batch_decode_paged_kv(q, pages, indptr, ids, info, out, lse, 0.1)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(4):
        new_k, new_v = rows_like(rng, 3, 2, 128), rows_like(rng, 3, 2, 128)
        new_q = rng.standard_normal((3, 8, 128)).astype(np.float16)
        k.copy_(dev(new_k))
        v.copy_(dev(new_v))
        q.copy_(dev(new_q))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        pool.pages = mxfp4.append(pool.pages, new_k, new_v, slots)
        replayed = host(out).copy(), host(lse).copy()
        compare(new_q, [1] * 3, pool, False, *replayed, 0.1)
        out.zero_()
        with torch.cuda.stream(stream):
            kernels.mxfp4_batch_decode_paged_kv(q, pages, indptr, ids, info, out, lse, 0.1)
        torch.cuda.synchronize()
        assert np.array_equal(host(out), replayed[0]) and np.array_equal(host(lse), replayed[1])


def test_shapes_that_need_more_and_less_scratch_in_turn():
    """The join's counters are where the next launch of other shapes, or of more rows, looks for them."""
    rng = np.random.default_rng(19)
    pools = [Pool(rng, [6000], 2, 16, 128), Pool(rng, [3000, 2000, 40], 1, 16, 64), Pool(rng, [2500] * 5, 2, 32, 256)]
    qs = [rng.standard_normal((len(p.info), 4 * p.pages.shape[2], p.d)).astype(np.float16) for p in pools]
    for _ in range(2):
        for q, pool in zip(qs, pools):
            out, lse = decode(q, pool, 0.1)
            compare(q, [1] * len(q), pool, False, out, lse, 0.1)
            few = [3] * len(q)
            rows = np.repeat(q, 3, 0)
            out, lse = prefill(rows, few, pool, 1, 0.1)
            compare(rows, few, pool, True, out, lse, 0.1)


def test_results_do_not_depend_on_the_run():
    rng = np.random.default_rng(16)
    pool = Pool(rng, [5000, 1200, 30], 2, 16, 128)
    q = rng.standard_normal((3, 8, 128)).astype(np.float16)
    first = decode(q, pool, 0.1)
    for _ in range(5):
        again = decode(q, pool, 0.1)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


def test_tensor_level_entry_points_read_views_of_a_merged_buffer():
    """The index arrays at offsets of one buffer, as the cache's are; the same bits as by the Python functions."""
    from tvm_amd import dlpack as dl

    rng = np.random.default_rng(17)
    pool = Pool(rng, [300, 17, 90], 2, 16, 128)
    pages, indptr, ids, info = pool.device()
    k, v = rows_like(rng, 3, 2, 128), rows_like(rng, 3, 2, 128)
    slots = np.array([pool.slot(b, n - 1) for b, n in enumerate((300, 17, 90))], np.int32)
    merged = torch.zeros(1024, dtype=torch.int32, device=DEV)
    views, at = [], 4
    for values in (pool.indptr, pool.ids, pool.info, slots, np.array([0, 4, 5, 7], np.int32)):
        merged[at:at + len(values)] = i32(values)
        views.append(dl.view(merged, 4 * at, (len(values),)))
        at += -(-len(values) // 4) * 4
    d_indptr, d_ids, d_info, d_slots, d_q_indptr = views
    dl.call("mxfp4_append", dl.tensor(pages), dl.tensor(dev(k)), dl.tensor(dev(v)), d_slots)
    pool.pages = mxfp4.append(pool.pages, k, v, slots)
    assert np.array_equal(host(pages), pool.pages)
    back = [torch.empty((3, 2, 128), dtype=torch.float16, device=DEV) for _ in range(2)]
    dl.call("mxfp4_read_kv", dl.tensor(pages), d_slots, dl.tensor(back[0]), dl.tensor(back[1]))
    assert np.array_equal(host(back[0]).astype(np.float64), mxfp4.rounded(k)) and np.array_equal(host(back[1]).astype(np.float64), mxfp4.rounded(v))
    q = rng.standard_normal((7, 8, 128)).astype(np.float16)
    d_q = dev(q)
    out, lse = torch.empty((7, 8, 128), dtype=torch.float16, device=DEV), torch.empty((7, 8), device=DEV)
    dl.call("mxfp4_batch_prefill_paged_kv", dl.tensor(d_q), d_q_indptr, dl.tensor(pages), d_indptr, d_ids, d_info, dl.tensor(out), dl.tensor(lse),
            1, 0.1)
    again = prefill(q, [4, 1, 2], pool, 1, 0.1)
    assert np.array_equal(host(out), again[0]) and np.array_equal(host(lse), again[1])
    dl.call("mxfp4_batch_decode_paged_kv", dl.tensor(d_q[:3]), dl.tensor(pages), d_indptr, d_ids, d_info, dl.tensor(out[:3]), dl.tensor(lse[:3]),
            0.1)
    again = decode(q[:3], pool, 0.1)
    assert np.array_equal(host(out[:3]), again[0]) and np.array_equal(host(lse[:3]), again[1])
