"""Eviction by attention weight without a GPU: the oracle's own promises, and what the entry points refuse."""
import numpy as np
import pytest

import tvm_amd
from oracle import eviction


def one_sequence(weights, page=16):
    n = len(weights)
    count = -(-n // page)
    sums = np.full((count, 1, page), 1e9, np.float32)
    sums.reshape(-1)[:n] = weights
    return sums, np.array([0, count]), np.arange(count), np.array([n - (count - 1) * page])


def select(weights, keep, sinks, recent, max_keep=None):
    sums, indptr, ids, info = one_sequence(weights)
    return eviction.select(sums, indptr, ids, info, [keep], max_keep or keep, sinks, recent)[0, 0].tolist()


def test_stayers_keep_their_places_and_recent_tokens_come_last():
    assert select([0, 5, 1, 9, 2, 8, 7, 0], 5, 1, 1) == [0, 5, 6, 3, 7]
    assert select([0, 5, 1, 9, 2, 8, 7, 0], 5, 0, 0) == [5, 1, 6, 3, 4]
    assert select([3, 3, 3, 3, 3, 3], 3, 0, 1) == [0, 1, 5]  # equal ones: the first
    assert select([np.nan, -np.inf, 1.0, -0.0, 0.0], 3, 0, 0) == [3, 4, 2]
    assert select([1, 2], 5, 1, 1) == [0, 1, -1, -1, -1]
    assert select([1, 2, 3], 2, 9, 9) == [1, 2]
    assert select([1, 2, 3], 0, 1, 1, max_keep=2) == [-1, -1]


def test_a_choice_moves_every_token_to_the_front_of_none():
    rng = np.random.default_rng(0)
    for _ in range(50):
        n = int(rng.integers(2, 300))
        keep, sinks, recent = (int(rng.integers(1, n + 3)) for _ in range(3))
        kept = np.array(select(rng.random(n).astype(np.float32), keep, sinks, recent))
        kept = kept[kept >= 0]
        assert len(kept) == min(n, keep) and len(set(kept.tolist())) == len(kept) and (kept >= np.arange(len(kept))).all()


def test_weights_of_the_oracle():
    rng = np.random.default_rng(1)
    pages = rng.standard_normal((3, 2, 1, 16, 8))
    sums = np.zeros((3, 1, 16))
    q = rng.standard_normal((3, 2, 8))
    _, _, got, _, _ = eviction.attention(q, [3], pages, np.array([0, 2]), np.array([2, 0]), np.array([4]), True, 0.3, sums, np.array([1, 2]))
    assert abs(got.sum() - 6) < 1e-12 and got[0].sum() == 0 and got[2, 0, 4:].sum() == 0
    s = q[2, 0] @ np.concatenate((pages[2, 0, 0], pages[0, 0, 0, :4])).T * 0.3
    _, _, last, _, _ = eviction.attention(q[:, :1], [3], pages, np.array([0, 2]), np.array([2, 0]), np.array([4]), True, 0.3, sums,
                                          np.array([1, 2]), observed=1)
    assert np.allclose(np.concatenate((last[1, 0], last[2, 0, :4])), np.exp(s) / np.exp(s).sum())


# ---- refusals: every check comes in front of any device work ------------------------------------------------------

SOME = 4096  # an address that is never read


def decode_args(**changes):
    a = dict(q=SOME, pages=SOME, indptr=SOME, values=SOME, info=SOME, out=SOME, lse=SOME, sums=SOME, weight_values=SOME, scale=1.0, batch=1,
             nnz=1, num_pages=1, h_q=8, h_kv=2, d=128, page=16, stream=None)
    a.update(changes)
    return list(a.values())


def prefill_args(**changes):
    a = dict(q=SOME, q_indptr=SOME, pages=SOME, indptr=SOME, values=SOME, info=SOME, out=SOME, lse=SOME, sums=SOME, weight_values=SOME,
             causal=1, observed=0, scale=1.0, batch=1, total_q=3, nnz=1, num_pages=1, h_q=8, h_kv=2, d=128, page=16, stream=None)
    a.update(changes)
    return list(a.values())


def select_args(**changes):
    a = dict(sums=SOME, indptr=SOME, weight_values=SOME, info=SOME, keep=SOME, kept=SOME, sinks=1, recent=1, batch=1, nnz=1, h_kv=2, page=16,
             max_keep=8, stream=None)
    a.update(changes)
    return list(a.values())


def move_args(**changes):
    a = dict(pages=SOME, sums=SOME, indptr=SOME, values=SOME, weight_values=SOME, kept=SOME, batch=1, nnz=1, num_pages=1, h_kv=2, page=16, d=128,
             bits=16, max_keep=8, stream=None)
    a.update(changes)
    return list(a.values())


ENTRIES = {"batch_decode_paged_kv_weights": decode_args, "batch_prefill_paged_kv_weights": prefill_args, "select_kept_tokens": select_args,
           "move_kept_tokens": move_args}


def refusal(entry, changes):
    lib = tvm_amd.lib()
    code = getattr(lib, "tvmkv_" + entry)(*ENTRIES[entry](**changes))
    return code, lib.tvmkv_last_error().decode()


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("changes, code, text", [
    (dict(page=24), -2, "page_size 24 is not built (16, 32, 64, 128)"),
    (dict(page=0), -2, "page_size 0 is not built"),
    (dict(page=256), -2, "page_size 256 is not built"),
    (dict(h_kv=0), -1, "bad shape"),
    (dict(batch=-1), -1, "bad shape"),
    (dict(nnz=-1), -1, "bad shape"),
    (dict(nnz=1 << 27), -1, "too many pages"),
    (dict(indptr=None), -1, "NULL tensor"),
    (dict(weight_values=None), -1, "NULL page table"),
])
def test_refused_by_every_entry_point(entry, changes, code, text):
    got, message = refusal(entry, changes)
    assert got == code and message.startswith(entry + ":") and text in message


@pytest.mark.parametrize("entry, changes, code, text", [
    (entry, changes, code, text)
    for entry in ("batch_decode_paged_kv_weights", "batch_prefill_paged_kv_weights")
    for changes, code, text in [
        (dict(d=72), -2, "head_dim 72 is not built"), (dict(d=512), -2, "head_dim 512 is not built"), (dict(h_q=9), -1, "bad shape"),
        (dict(h_q=0), -1, "bad shape"), (dict(q=None), -1, "NULL tensor"), (dict(sums=None), -1, "NULL tensor"),
        (dict(lse=None), -1, "NULL tensor"), (dict(info=None), -1, "NULL tensor"), (dict(values=None), -1, "NULL page table"),
        (dict(q=SOME + 2), -1, "aligned to 16 bytes"), (dict(pages=SOME + 8), -1, "aligned to 16 bytes"),
        (dict(out=SOME + 8), -1, "aligned to 16 bytes")]
] + [
    ("batch_prefill_paged_kv_weights", dict(total_q=-1), -1, "bad shape"),
    ("batch_prefill_paged_kv_weights", dict(total_q=1 << 30), -1, "bad shape"),
    ("batch_prefill_paged_kv_weights", dict(observed=-1), -1, "observed is -1"),
    ("batch_prefill_paged_kv_weights", dict(q_indptr=None), -1, "NULL tensor"),
    ("select_kept_tokens", dict(sinks=-1), -1, "bad shape"),
    ("select_kept_tokens", dict(recent=-1), -1, "bad shape"),
    ("select_kept_tokens", dict(max_keep=-1), -1, "bad shape"),
    ("select_kept_tokens", dict(batch=65536), -1, "too many sequences"),
    ("select_kept_tokens", dict(keep=None), -1, "NULL tensor"),
    ("select_kept_tokens", dict(kept=None), -1, "NULL tensor"),
    ("select_kept_tokens", dict(sums=None), -1, "NULL tensor"),
    ("move_kept_tokens", dict(bits=8), -2, "rows of 8 bits"),
    ("move_kept_tokens", dict(d=4), -2, "head_dim 4 is not built"),
    ("move_kept_tokens", dict(d=264), -2, "head_dim 264 is not built"),
    ("move_kept_tokens", dict(pages=None), -1, "NULL tensor"),
    ("move_kept_tokens", dict(kept=None), -1, "NULL tensor"),
    ("move_kept_tokens", dict(values=None), -1, "NULL page table"),
    ("move_kept_tokens", dict(pages=SOME + 8), -1, "aligned to 16 bytes"),
    ("move_kept_tokens", dict(max_keep=-1), -1, "bad shape"),
    ("move_kept_tokens", dict(batch=65536), -1, "too many sequences"),
])
def test_refused(entry, changes, code, text):
    got, message = refusal(entry, changes)
    assert got == code and message.startswith(entry + ":") and text in message


@pytest.mark.parametrize("entry, changes", [
    ("batch_decode_paged_kv_weights", dict(batch=0)), ("batch_prefill_paged_kv_weights", dict(batch=0)),
    ("batch_prefill_paged_kv_weights", dict(total_q=0)), ("select_kept_tokens", dict(batch=0)), ("select_kept_tokens", dict(max_keep=0)),
    ("move_kept_tokens", dict(batch=0)), ("move_kept_tokens", dict(max_keep=0)), ("move_kept_tokens", dict(nnz=0)),
])
def test_nothing_to_do(entry, changes):
    assert refusal(entry, changes)[0] == 0


# ---- the Python face: its checks read shapes and types, so that host tensors do -------------------------------------


def tensors(batch=2, rows=2, h_q=8, h_kv=2, d=64, page=16):
    import torch
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    f16 = lambda *shape: torch.zeros(shape, dtype=torch.float16)
    f32 = lambda *shape: torch.zeros(shape, dtype=torch.float32)
    return {"q": f16(rows, h_q, d), "q_indptr": i32(batch + 1), "pages": f16(5, 2, h_kv, page, d), "page_indptr": i32(batch + 1), "page_values": i32(4),
            "length_info": i32(batch), "output": f16(rows, h_q, d), "lse": f32(rows, h_q), "key_weights": f32(6, h_kv, page),
            "weight_page_values": i32(4), "keep": i32(batch), "kept": i32(batch, h_kv, 8)}


PYTHON = {
    "batch_decode_paged_kv_weights": (["q", "pages", "page_indptr", "page_values", "length_info", "output", "lse", "key_weights",
                                       "weight_page_values"], [0.125]),
    "batch_prefill_paged_kv_weights": (["q", "q_indptr", "pages", "page_indptr", "page_values", "length_info", "output", "lse", "key_weights",
                                        "weight_page_values"], [1, 0, 0.125]),
    "select_kept_tokens": (["key_weights", "page_indptr", "weight_page_values", "length_info", "keep", "kept"], [1, 1]),
    "move_kept_tokens": (["pages", "key_weights", "page_indptr", "page_values", "weight_page_values", "kept"], []),
}


def call(name, t):
    from tvm_amd import kernels
    order, rest = PYTHON[name]
    getattr(kernels, name)(*[t[k] for k in order], *rest)


@pytest.mark.parametrize("name", PYTHON)
def test_host_tensors_are_refused(name):
    with pytest.raises(tvm_amd.KVError, match="device memory"):
        call(name, tensors())


def changes():
    import torch
    attention = ("batch_decode_paged_kv_weights", "batch_prefill_paged_kv_weights")
    for name in attention:
        yield name, dict(q=torch.zeros(2, 8, 64)), "float16"
        yield name, dict(page_values=torch.zeros(4, dtype=torch.int64)), "int32"
        yield name, dict(lse=torch.zeros(2, 8, dtype=torch.float64)), "lse must be float32"
        yield name, dict(lse=torch.zeros(2, 9)), "lse has shape"
        yield name, dict(output=torch.zeros(3, 8, 64, dtype=torch.float16)), "output has shape"
        yield name, dict(pages=torch.zeros(5, 2, 2, 16, 32, dtype=torch.float16)), "pages has shape"
        yield name, dict(pages=torch.zeros(5, 2, 16, 64, dtype=torch.float16)), "pages has shape"
        yield name, dict(length_info=torch.zeros(3, 2, dtype=torch.int32)), "length_info has shape"  # sliding windows
        yield name, dict(weight_page_values=torch.zeros(3, dtype=torch.int32)), "weight_page_values has shape"
        yield name, dict(key_weights=torch.zeros(6, 2, 16, dtype=torch.float16)), "key_weights must be float32"
        yield name, dict(key_weights=torch.zeros(6, 2, 32)), "key_weights has shape"
    yield attention[0], dict(tensors(rows=3), length_info=tensors()["length_info"]), "q has shape"
    yield attention[1], dict(q_indptr=torch.zeros(2, dtype=torch.int32)), "q_indptr has shape"
    yield "select_kept_tokens", dict(key_weights=torch.zeros(6, 2, 16, dtype=torch.float64)), "key_weights must be float32"
    yield "select_kept_tokens", dict(keep=torch.zeros(3, dtype=torch.int32)), "keep has shape"
    yield "select_kept_tokens", dict(length_info=torch.zeros(1, dtype=torch.int32)), "length_info has shape"
    yield "select_kept_tokens", dict(kept=torch.zeros(2, 3, 8, dtype=torch.int32)), "kept has shape"
    yield "select_kept_tokens", dict(kept=torch.zeros(2, 2, 8, dtype=torch.int64)), "int32"
    yield "move_kept_tokens", dict(pages=torch.zeros(5, 2, 2, 16, 64, dtype=torch.bfloat16)), "only float16 and float32"
    yield "move_kept_tokens", dict(pages=torch.zeros(5, 3, 2, 16, 64)), "pages has shape"
    yield "move_kept_tokens", dict(key_weights=torch.zeros(6, 2, 32)), "key_weights has shape"
    yield "move_kept_tokens", dict(weight_page_values=torch.zeros(5, dtype=torch.int32)), "weight_page_values has shape"
    yield "move_kept_tokens", dict(kept=torch.zeros(1, 2, 8, dtype=torch.int32)), "kept has shape"


@pytest.mark.parametrize("name, change, text", list(changes()))
def test_refused_by_the_python_face(name, change, text):
    with pytest.raises(tvm_amd.KVError, match=text):
        call(name, dict(tensors(), **change))


def test_kernels_keep_their_values_in_registers(tmp_path):
    """Nothing that the kernels of eviction hold is spilled, nor by the decode kernels that keep their scores."""
    import os
    import re

    from tests.test_host_support import READELF, ROOT, _kernel_metadata
    library = os.path.join(ROOT, "tvm_amd", "lib", "libtvmkv.so")
    if not (os.path.exists(READELF) and os.path.exists(library)):
        pytest.skip("needs the built library and llvm-readelf")
    kernels = [k for k in _kernel_metadata(library, tmp_path)
               if re.search(r"key_weights_kernel|shared_rows_kernel|merge_and_weigh_kernel|kept_scores_kernel|select_|move_kept_kernel", k[0])
               or ("decode_mfma_kernel" in k[0] and k[0].split("EEEv")[0].endswith("Lb1"))]
    assert len(kernels) == 11 + 6 + 1 + 1 + 6 + 3 + 4
    assert [k for k in kernels if k[1] or k[2]] == []
