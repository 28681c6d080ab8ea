"""Eviction by attention weight as a caller's program runs it, step after step (bounds: tests/test_gpu_eviction.py)."""
import os
import re
import threading
import types

import numpy as np
import pytest
import torch

from oracle import eviction
from tests.gpu_util import DEV, dev, host, i32
from tests.test_gpu_eviction import check_attention, queries
from tvm_amd import kernels

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def readme_example():
    """The readme's example of eviction: what is made once, and a step."""
    text = open(os.path.join(ROOT, "README.md")).read()
    block = next(b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "move_kept_tokens" in b)
    lines = block.split("\n")
    first = next(i for i, line in enumerate(lines) if line.startswith("sums = "))
    return "\n".join(lines[:first + 1]), "\n".join(lines[first + 1:])


class Sequences:
    """What a program keeps: a pool that other sequences have used, page lists, lengths."""

    def __init__(self, rng, lengths, h_kv, page, d, most):
        self.page, self.d, self.stored = page, d, list(lengths)
        each = -(-most // page)
        self.total = each * len(lengths) + 2
        lists = rng.permutation(self.total)[:each * len(lengths)].astype(np.int32)
        self.lists = [lists[i * each:(i + 1) * each] for i in range(len(lengths))]
        self.pages = rng.standard_normal((self.total, 2, h_kv, page, d)).astype(np.float16)
        self.tables()

    def tables(self):
        counts = [-(-n // self.page) for n in self.stored]
        self.ids = self.weight_ids = np.concatenate([l[:c] for l, c in zip(self.lists, counts)])
        self.indptr = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
        self.info = np.array([n - (c - 1) * self.page for n, c in zip(self.stored, counts)], np.int32)

    def next_slots(self):
        return np.array([l[n // self.page] * self.page + n % self.page for l, n in zip(self.lists, self.stored)], np.int32)


def test_the_example_of_the_readme():
    """A token that is stored where an evicted one was begins without weight."""
    rng = np.random.default_rng(60)
    setup, step = readme_example()
    h_q, h_kv, d, page, budget = 32, 8, 128, 16, 300
    s = Sequences(rng, [budget, budget - 20], h_kv, page, d, budget + 1)
    names = {"num_pages": s.total}
    exec(setup, names)
    names["sums"].fill_(5.0)  # what the pool's sequences have received until now
    names["pages"], names["keep"] = dev(s.pages), i32([budget, budget])
    names["kept"] = torch.empty((2, h_kv, budget), dtype=torch.int32, device=DEV)
    for _ in range(30):
        k, v = (rng.standard_normal((2, h_kv, d)).astype(np.float16) for _ in range(2))
        slots, q = s.next_slots(), queries(rng, 2, h_q, d)
        s.sums = host(names["sums"]).copy()
        for i, slot in enumerate(slots):
            s.pages[slot // page, 0, :, slot % page], s.pages[slot // page, 1, :, slot % page] = k[i], v[i]
            s.sums[slot // page, :, slot % page] = 0
        s.stored = [n + 1 for n in s.stored]
        s.tables()
        names.update(k=dev(k), v=dev(v), slots=i32(slots), indptr=i32(s.indptr), ids=i32(s.ids), last_page_len=i32(s.info), q=dev(q),
                     out=torch.empty(q.shape, dtype=torch.float16, device=DEV), lse=torch.empty(q.shape[:2], device=DEV))
        before = {}

        def select(sums, *rest):  # what attention has left, for the oracle
            before["sums"] = host(sums).copy()
            kernels.select_kept_tokens(sums, *rest)

        names["kernels"] = types.SimpleNamespace(**{**vars(kernels), "select_kept_tokens": select})
        exec(step, names)
        check_attention(q, [1, 1], s, False, 0, (host(names["out"]), host(names["lse"]), before["sums"]))
        kept = eviction.select(before["sums"], s.indptr, s.weight_ids, s.info, [budget] * 2, budget, 4, 256)
        assert np.array_equal(host(names["kept"]), kept)
        s.pages, sums = eviction.move(s.pages, before["sums"], s.indptr, s.ids, s.weight_ids, kept)
        assert np.array_equal(host(names["pages"]).view(np.uint16), s.pages.view(np.uint16)) and np.array_equal(host(names["sums"]), sums)
        s.stored = [min(n, budget) for n in s.stored]


class Captured:
    """One decode, choice and move, and one prefill, captured over arrays of fixed size whose contents change from replay to replay."""

    def __init__(self, rng, batch, capacity, queries_at_most, keep, h_q, h_kv, page, d):
        self.batch, self.capacity, self.page, self.d, self.h_q, self.h_kv, self.keep = batch, capacity, page, d, h_q, h_kv, keep
        shape = (capacity + 4, 2, h_kv, page, d)
        self.t = {"pages": torch.zeros(shape, dtype=torch.float16, device=DEV), "sums": torch.zeros((capacity + 4, h_kv, page), device=DEV),
                  "indptr": i32([0] * (batch + 1)), "ids": i32([0] * capacity), "weight_ids": i32([0] * capacity), "info": i32([0] * batch),
                  "q_indptr": i32([0] * (batch + 1)), "q": torch.zeros((queries_at_most, h_q, d), dtype=torch.float16, device=DEV),
                  "one": torch.zeros((batch, h_q, d), dtype=torch.float16, device=DEV), "keep": i32([0] * batch)}
        self.o = {"out": torch.zeros_like(self.t["q"]), "lse": torch.zeros(self.t["q"].shape[:2], device=DEV),
                  "one_out": torch.zeros_like(self.t["one"]), "one_lse": torch.zeros((batch, h_q), device=DEV),
                  "kept": torch.zeros((batch, h_kv, keep), dtype=torch.int32, device=DEV), "after_prefill": torch.zeros_like(self.t["sums"]),
                  "after_decode": torch.zeros_like(self.t["sums"])}

    def calls(self):
        t, o, scale = self.t, self.o, self.d ** -0.5
        kernels.batch_prefill_paged_kv_weights(t["q"], t["q_indptr"], t["pages"], t["indptr"], t["ids"], t["info"], o["out"], o["lse"], t["sums"],
                                               t["weight_ids"], 1, 3, scale)
        o["after_prefill"].copy_(t["sums"])
        kernels.batch_decode_paged_kv_weights(t["one"], t["pages"], t["indptr"], t["ids"], t["info"], o["one_out"], o["one_lse"], t["sums"],
                                              t["weight_ids"], scale)
        o["after_decode"].copy_(t["sums"])
        kernels.select_kept_tokens(t["sums"], t["indptr"], t["weight_ids"], t["info"], t["keep"], o["kept"], 2, 7)
        kernels.move_kept_tokens(t["pages"], t["sums"], t["indptr"], t["ids"], t["weight_ids"], o["kept"])

    def fill(self, rng, stored, q_lens, keep):
        pool = types.SimpleNamespace(d=self.d, page=self.page, stored=list(stored))
        counts = [-(-n // self.page) for n in stored]
        assert sum(counts) <= self.capacity and sum(q_lens) <= len(self.t["q"])
        pool.ids, pool.weight_ids = (rng.permutation(self.capacity + 4)[:self.capacity].astype(np.int32) for _ in range(2))
        pool.indptr = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
        pool.info = np.array([n - (c - 1) * self.page if c else 0 for n, c in zip(stored, counts)], np.int32)
        pool.pages = rng.standard_normal(tuple(self.t["pages"].shape)).astype(np.float16)
        pool.sums = rng.random(tuple(self.t["sums"].shape)).astype(np.float32)
        q, one = queries(rng, len(self.t["q"]), self.h_q, self.d), queries(rng, self.batch, self.h_q, self.d)
        for name, x in dict(pages=pool.pages, sums=pool.sums, indptr=pool.indptr, ids=pool.ids, weight_ids=pool.weight_ids, info=pool.info, q=q, one=one,
                            q_indptr=np.concatenate(([0], np.cumsum(q_lens))).astype(np.int32), keep=np.array(keep, np.int32)).items():
            self.t[name].copy_(dev(x))
        self.o["out"].fill_(7.0)
        self.o["lse"].fill_(7.0)
        return pool, q, one

    def check(self, pool, q, one, q_lens, keep, what):
        o, n = {name: host(x) for name, x in self.o.items()}, sum(q_lens)
        check_attention(q[:n], q_lens, pool, True, 3, (o["out"][:n], o["lse"][:n], o["after_prefill"]), what + ", prefill")
        assert (o["out"][n:] == 7.0).all() and (o["lse"][n:] == 7.0).all()
        pool.sums = o["after_prefill"]
        check_attention(one, [1] * self.batch, pool, False, 0, (o["one_out"], o["one_lse"], o["after_decode"]), what + ", decode")
        kept = eviction.select(o["after_decode"], pool.indptr, pool.weight_ids, pool.info, keep, self.keep, 2, 7)
        assert np.array_equal(o["kept"], kept), what
        pages, sums = eviction.move(pool.pages, o["after_decode"], pool.indptr, pool.ids, pool.weight_ids, kept)
        assert np.array_equal(host(self.t["pages"]).view(np.uint16), pages.view(np.uint16)) and np.array_equal(host(self.t["sums"]), sums), what


@pytest.mark.parametrize("capacity, queries_at_most, steps", [
    (40, 12, [([600], [5], [90]), ([1], [1], [5]), ([0], [0], [9]), ([633], [12], [100]), ([17], [0], [3])]),
    (60, 40, [([100, 200, 300], [9, 0, 31], [50, 60, 7]), ([900, 3, 0], [2, 3, 0], [100, 2, 1]), ([0, 0, 960], [0, 0, 40], [1, 1, 99]), ([1, 1, 1], [1, 1, 1], [1, 0, 1])]),
    (400, 300, [([3000, 20, 1000], [250, 1, 20], [100, 20, 90]), ([0, 6300, 10], [0, 300, 0], [0, 77, 10]), ([2000, 2000, 2000], [1, 1, 1], [100, 99, 98])]),
])
def test_lengths_change_between_replays(capacity, queries_at_most, steps):
    """A launch's shape comes from the arrays' sizes alone: padded tables and queries, sequences that grow, end and begin."""
    rng = np.random.default_rng(capacity)
    c = Captured(rng, len(steps[0][0]), capacity, queries_at_most, 100, 8, 2, 16, 64)
    stream = torch.cuda.Stream()
    c.fill(rng, *steps[0])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        c.calls()  # what the kernels allocate is there
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.calls()
    for i, (stored, q_lens, keep) in enumerate(steps + steps[::-1]):
        torch.cuda.synchronize()
        pool, q, one = c.fill(rng, stored, q_lens, keep)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check(pool, q, one, q_lens, keep, f"replay {i}")


def test_threads_with_streams_of_their_own():
    """Calls of two host threads at once, each with its own stream, scratch memory and shapes."""
    shapes = [(40, 12, [([600], [5], [90]), ([633], [12], [100])]), (400, 300, [([3000, 20, 1000], [250, 1, 20], [100, 20, 90]), ([2000] * 3, [1] * 3, [100] * 3)])]
    failures = []

    def work(n):
        try:
            capacity, most, steps = shapes[n]
            rng, stream = np.random.default_rng(n), torch.cuda.Stream()
            with torch.cuda.stream(stream):
                c = Captured(rng, len(steps[0][0]), capacity, most, 100, 8, 2, 16, 64)
                for i in range(6):
                    stored, q_lens, keep = steps[i % 2]
                    pool, q, one = c.fill(rng, stored, q_lens, keep)
                    c.calls()
                    stream.synchronize()
                    c.check(pool, q, one, q_lens, keep, f"thread {n}, step {i}")
        except BaseException as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
