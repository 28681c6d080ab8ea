"""The 4-bit cache object: sequences grow, fork, shrink and end, steps mix prompts and single tokens, and every output is
attention over the rows that the cache holds (oracle/mxfp4.py) and, in steps with prompts, the step's own fp16 rows."""
import numpy as np
import pytest
import torch

from oracle import mxfp4
from tests.gpu_util import DEV, dev, host, i32
from tests.util import assert_close
from tvm_amd import KVError, RopeMode, kernels
from tvm_amd.mxfp4_cache import Mxfp4KVCache

pytestmark = pytest.mark.gpu


def attend(q, k, v, sm_scale):
    """q (heads, d) over k, v (keys, kv heads, d) in 64 bits."""
    out = np.zeros(q.shape)
    for h in range(q.shape[0]):
        kv = h // (q.shape[0] // k.shape[1])
        s = k[:, kv] @ q[h].astype(np.float64) * sm_scale
        w = np.exp(s - s.max())
        out[h] = w @ v[:, kv] / w.sum()
    return out


class Mirror:
    def __init__(self, layers=2, hq=8, hkv=2, d=128, page=16, windows=False, rope=RopeMode.NORMAL):
        self.cache = Mxfp4KVCache([16, 4096, 512, page, int(windows)], layers, hq, hkv, d, rope)
        self.layers, self.hq, self.hkv, self.d, self.rope = layers, hq, hkv, d, rope
        self.rows = {}     # sequence -> per layer [k (n, hkv, d), v], as the cache holds them
        self.windows = {}  # sequence -> (window, sinks)
        self.rng = np.random.default_rng(3)

    def add(self, sid, window=None):
        self.cache.add_sequence(sid)
        self.rows[sid] = [[np.zeros((0, self.hkv, self.d))] * 2 for _ in range(self.layers)]
        self.position = getattr(self, "position", {})
        self.position[sid] = 0
        if window:
            self.cache.enable_sliding_window_for_seq(sid, *window)
            self.windows[sid] = window

    def fork(self, parent, child, at=-1):
        self.cache.fork_sequence(parent, child, at)
        n = self.position[parent] if at == -1 else at
        self.rows[child] = [[x[:n] for x in kv] for kv in self.rows[parent]]
        self.position[child] = n

    def popn(self, sid, n):
        self.cache.popn(sid, n)
        self.position[sid] -= n
        self.rows[sid] = [[x[:len(x) - n] for x in kv] for kv in self.rows[sid]]

    def step(self, *batch):
        ids, lens = [b[0] for b in batch], [b[1] for b in batch]
        self.cache.begin_forward(ids, lens)
        scale = self.d ** -0.5
        append_first = not self.windows and all(n == 1 for n in lens)
        for layer in range(self.layers):
            qkv = dev(self.rng.standard_normal((sum(lens), self.hq + 2 * self.hkv, self.d)).astype(np.float16))
            out = torch.full((sum(lens), self.hq, self.d), 9.0, dtype=torch.float16, device=DEV)
            self.cache.attention_with_fused_qkv(layer, scale, qkv, out)
            # windows restart positions at their own counting: tests with windows use no rotation
            positions = i32([self.position[s] + i for s, n in batch for i in range(n)])
            q, k, v = (torch.empty((sum(lens), h, self.d), dtype=torch.float16, device=DEV) for h in (self.hq, self.hkv, self.hkv))
            kernels.fused_rope(qkv, positions, q, k, v, self.rope == RopeMode.NORMAL)
            q, k, v, out = (host(t).astype(np.float64) for t in (q, k, v, out))
            at = 0
            for sid, n in batch:
                new = [k[at:at + n], v[at:at + n]]
                stored = [mxfp4.rounded(x) for x in new]
                held = self.rows[sid][layer]
                own = stored if append_first else new
                for i in range(n):
                    keys, values = (np.concatenate((h, x[:i + 1])) for h, x in zip(held, own))
                    assert_close(out[at + i].astype(np.float32), attend(q[at + i], keys, values, scale).astype(np.float32),
                                 what=f"sequence {sid}, token {i}, layer {layer}, after {len(held[0])} rows")
                self.rows[sid][layer] = [np.concatenate((h, x)) for h, x in zip(held, stored)]
                at += n
        self.cache.end_forward()
        for sid, n in batch:
            self.position[sid] += n
            if sid in self.windows and len(self.rows[sid][0][0]) > self.windows[sid][0]:
                window, sinks = self.windows[sid]
                self.rows[sid] = [[np.concatenate((x[:sinks], x[len(x) - (window - sinks):])) for x in kv] for kv in self.rows[sid]]


@pytest.mark.parametrize("shape", [dict(), dict(hq=4, hkv=4, d=64, page=32), dict(hq=6, hkv=1, d=96), dict(hq=4, hkv=1, d=256, layers=1),
                                   dict(rope=RopeMode.NONE)])
def test_sequences_grow_fork_shrink_and_end(shape):
    m = Mirror(**shape)
    for sid in (0, 1, 2):
        m.add(sid)
    m.step((0, 37), (1, 5), (2, 1))
    m.step((0, 1), (1, 1), (2, 1))
    m.step((0, 1), (2, 20))           # a prompt chunk beside a decoding sequence
    m.fork(0, 3)
    m.fork(0, 4, 20)                  # in the middle of a page
    m.step((0, 1), (3, 1), (4, 1), (1, 1))
    m.step((3, 3), (4, 9))
    m.popn(3, 2)
    m.popn(2, 17)
    m.popn(0, 17)                     # into rows that forks share: the host cache forks anew and copies a page
    m.step((3, 1), (0, 1), (2, 1))
    m.cache.remove_sequence(1)
    m.step((0, 2), (2, 1), (4, 1))


def test_windows_slide_over_4_bit_rows():
    m = Mirror(windows=True, rope=RopeMode.NONE, layers=1)
    m.add(0, (40, 4))
    m.add(1)
    m.step((0, 30), (1, 50))
    for _ in range(14):
        m.step((0, 1), (1, 1))
    m.step((0, 7), (1, 3))
    for _ in range(3):
        m.step((0, 1), (1, 1))


def test_a_cleared_cache_starts_over():
    m = Mirror(layers=1)
    m.add(0)
    m.step((0, 20))
    m.fork(0, 1, 10)
    m.step((1, 1))
    m.cache.clear()
    assert m.cache.get_num_available_pages() == m.cache.pages[0].shape[0]
    m.rows.clear()
    m.add(0)
    m.step((0, 18))
    m.fork(0, 1, 9)
    m.step((0, 1), (1, 1))


def test_refusals():
    with pytest.raises(KVError, match="INLINE"):
        Mxfp4KVCache([4, 256, 64, 16, 0], 1, 8, 2, 128, RopeMode.INLINE)
    cache = Mxfp4KVCache([4, 256, 64, 16, 0], 1, 8, 2, 128)
    qkv, out = torch.zeros((3, 12, 128), dtype=torch.float16, device=DEV), torch.zeros((3, 8, 128), dtype=torch.float16, device=DEV)
    with pytest.raises(KVError, match="between begin_forward and end_forward"):
        cache.attention_with_fused_qkv(0, 0.1, qkv, out)
    cache.add_sequence(0)
    cache.begin_forward([0], [2])
    with pytest.raises(KVError, match="qkv has shape"):
        cache.attention_with_fused_qkv(0, 0.1, qkv, out[:2])
    with pytest.raises(KVError, match="out has shape"):
        cache.attention_with_fused_qkv(0, 0.1, qkv[:2], out)
    with pytest.raises(KVError):  # the host cache's own check
        cache.add_sequence(0)
