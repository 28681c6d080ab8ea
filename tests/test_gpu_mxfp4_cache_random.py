"""The 4-bit cache object through random verbs: sequences begin, grow by prompts and single tokens, fork, shrink and end, and
every output is attention over the rows that the cache holds."""
import numpy as np
import pytest

from tests.test_gpu_mxfp4_cache import Mirror

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed, shape", [(0, dict(layers=1)), (1, dict(layers=1, hq=3, hkv=3, d=64, page=32)), (2, dict(layers=1, hq=6, hkv=1, d=96)),
                                         (3, dict(layers=1, hq=2, hkv=1, d=256, page=48))])
def test_random_verbs(seed, shape):
    rng = np.random.default_rng(seed)
    m = Mirror(**shape)
    free, m.position = list(range(100)), {}
    for _ in range(60):
        live, what = list(m.position), rng.random()
        if what < 0.12 and len(live) < 8 or not live:
            m.add(free.pop(0))
        elif what < 0.3 and len(live) < 8:
            parent = int(rng.choice(live))
            if m.position[parent] > 0:
                m.fork(parent, free.pop(0), int(rng.integers(1, m.position[parent] + 1)))
        elif what < 0.42:
            sid = int(rng.choice(live))
            if m.position[sid] > 1:
                m.popn(sid, int(rng.integers(1, m.position[sid])))
        elif what < 0.5 and len(live) > 2:
            sid = int(rng.choice(live))
            m.cache.remove_sequence(sid)
            del m.position[sid], m.rows[sid]
        else:
            some = [int(s) for s in rng.permutation(live)[:rng.integers(1, len(live) + 1)]]
            if rng.random() < 0.5:
                m.step(*((s, 1) for s in some))
            else:
                m.step(*((s, int(rng.integers(1, 40))) for s in some))
