"""Eviction by attention weight as a caller's program runs it, step after step (bounds: tests/test_gpu_eviction.py)."""
import os
import re
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
