"""The 4-bit cache without a GPU: what its format promises, and what its entry points refuse."""
import ctypes

import numpy as np
import pytest

import tvm_amd
from oracle import mxfp4


def finite_halves():
    x = np.arange(1 << 16, dtype=np.uint32).astype(np.uint16).view(np.float16)
    return x[np.isfinite(x)]


def test_every_fp16_value_reads_back_as_fp16():
    x = np.random.default_rng(0).permutation(finite_halves())
    x = x[:len(x) // 32 * 32].reshape(-1, 32)
    for rows in (x, x * np.float16(2.0 ** -12), x * np.float16(2.0 ** -20)):
        y = mxfp4.rounded(rows)
        assert np.array_equal(y.astype(np.float16).astype(np.float64), y)
        # a code is at most half of the widest spacing (2) off; only magnitudes that no scale reaches saturate
        largest = np.abs(rows.astype(np.float64)).max(-1, keepdims=True)
        _, scales = mxfp4.quantise(rows)
        off = np.abs(y - rows.astype(np.float64)) / 2.0 ** (scales.astype(np.float64) - 127)
        assert (off <= 1.0).all(where=largest <= 7.0 * 2.0 ** 13)
        assert np.abs(y).max() <= 49152.0


def test_scales_are_the_smallest_that_reach():
    rows = np.zeros((6, 32), np.float16)
    rows[:, 3] = [7.0, 7.004, -6.0, 3.5, 0.0, 65504.0]
    codes, scales = mxfp4.quantise(rows)
    assert scales[:, 0].tolist() == [127, 128, 127, 126, 127 - 23, 127 + 13]
    assert mxfp4.rounded(rows)[:, 3].tolist() == [6.0, 8.0, -6.0, 3.0, 0.0, 49152.0]


def test_ties_go_to_the_even_code_and_stored_values_stay():
    rows = np.zeros((1, 32), np.float16)
    rows[0, :8] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -5.0]
    assert mxfp4.rounded(rows)[0, :8].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, -4.0]
    again = mxfp4.rounded(np.random.default_rng(1).standard_normal((50, 64)).astype(np.float16))
    assert np.array_equal(mxfp4.rounded(again.astype(np.float16)), again)


def test_blocks_that_are_not_finite_are_nan():
    rows = np.ones((1, 96), np.float16)
    rows[0, 5], rows[0, 70] = np.inf, np.nan
    back = mxfp4.rounded(rows)[0]
    assert np.isnan(back[:32]).all() and (back[32:64] == 1).all() and np.isnan(back[64:]).all()


def test_pages_hold_codes_then_scales():
    k = np.zeros((1, 1, 64), np.float16)
    v = np.zeros((1, 1, 64), np.float16)
    k[0, 0, :3] = [6.0, -0.5, 1.5]
    v[0, 0, 33] = 12.0
    pages = mxfp4.append(mxfp4.empty_pages(2, 1, 16, 64), k, v, [16 + 5]).reshape(2, 2, -1)
    assert pages[0].sum() == 0
    assert pages[1, 0, 5 * 32:5 * 32 + 2].tolist() == [0x97, 0x03] and pages[1, 0, 16 * 32 + 5 * 2:][:2].tolist() == [127, 104]
    assert pages[1, 1, 5 * 32 + 16] == 0x70 and pages[1, 1, 16 * 32 + 5 * 2:][:2].tolist() == [104, 128]


# ---- refusals: every check comes in front of any device work ------------------------------------------------------

SOME = 4096  # an address that is never read


def append_args(**changes):
    a = dict(pages=SOME, k=SOME, v=SOME, map=SOME, n=1, num_pages=1, h_kv=2, page=16, d=128, stream=None)
    a.update(changes)
    return list(a.values())


def decode_args(**changes):
    a = dict(q=SOME, pages=SOME, indptr=SOME, values=SOME, info=SOME, out=SOME, lse=SOME, scale=1.0, batch=1, nnz=1, num_pages=1,
             h_q=8, h_kv=2, d=128, page=16, sliding=0, stream=None)
    a.update(changes)
    return list(a.values())


def prefill_args(**changes):
    a = dict(q=SOME, q_indptr=SOME, pages=SOME, indptr=SOME, values=SOME, info=SOME, out=SOME, lse=SOME, causal=1, scale=1.0, batch=1,
             total_q=3, nnz=1, num_pages=1, h_q=8, h_kv=2, d=128, page=16, sliding=0, stream=None)
    a.update(changes)
    return list(a.values())


ENTRIES = {"mxfp4_append": append_args, "mxfp4_read_kv": lambda **c: [append_args(**c)[i] for i in (0, 3, 1, 2, 4, 5, 6, 7, 8, 9)],
           "mxfp4_batch_decode_paged_kv": decode_args, "mxfp4_batch_prefill_paged_kv": prefill_args}


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("changes, code, text", [
    (dict(d=80), -2, "head_dim 80 is not built"),
    (dict(d=512), -2, "head_dim 512 is not built"),
    (dict(page=24), -2, "page_size must be a multiple of 16, got 24"),
    (dict(page=0), -2, "page_size must be a multiple of 16, got 0"),
    (dict(page=1 << 26, h_kv=4), -2, "a page of 8 GiB or more is not built"),
    (dict(h_kv=0), -1, "bad shape"),
    (dict(pages=None), -1, "NULL tensor"),
    (dict(pages=SOME + 8), -1, "aligned to 16 bytes"),
])
def test_refused_by_every_entry_point(entry, changes, code, text):
    lib = tvm_amd.lib()
    assert getattr(lib, "tvmkv_" + entry)(*ENTRIES[entry](**changes)) == code
    message = lib.tvmkv_last_error().decode()
    assert message.startswith(entry + ":") and text in message


@pytest.mark.parametrize("entry, changes, text", [
    ("mxfp4_append", dict(n=-1), "bad shape"),
    ("mxfp4_append", dict(map=None), "NULL tensor"),
    ("mxfp4_append", dict(v=SOME + 2), "aligned to 16 bytes"),
    ("mxfp4_batch_decode_paged_kv", dict(h_q=9), "bad shape"),
    ("mxfp4_batch_decode_paged_kv", dict(batch=-1), "bad shape"),
    ("mxfp4_batch_decode_paged_kv", dict(nnz=-1), "bad shape"),
    ("mxfp4_batch_decode_paged_kv", dict(values=None), "NULL page table"),
    ("mxfp4_batch_decode_paged_kv", dict(lse=None), "NULL tensor"),
    ("mxfp4_batch_decode_paged_kv", dict(out=SOME + 4), "aligned to 16 bytes"),
    ("mxfp4_batch_prefill_paged_kv", dict(total_q=-1), "bad shape"),
    ("mxfp4_batch_prefill_paged_kv", dict(q_indptr=None), "NULL tensor"),
    ("mxfp4_batch_prefill_paged_kv", dict(values=None), "NULL page table"),
])
def test_refused(entry, changes, text):
    lib = tvm_amd.lib()
    assert getattr(lib, "tvmkv_" + entry)(*ENTRIES[entry](**changes)) == -1
    assert text in lib.tvmkv_last_error().decode()


@pytest.mark.parametrize("entry", ["mxfp4_batch_decode_paged_kv", "mxfp4_batch_prefill_paged_kv"])
def test_attention_refuses_pools_it_cannot_address(entry):
    pages_of_64_gib = (1 << 36) // (2 * 2 * 16 * 68) + 1
    lib = tvm_amd.lib()
    assert getattr(lib, "tvmkv_" + entry)(*ENTRIES[entry](num_pages=pages_of_64_gib)) == -2
    assert "a pool of 64 GiB or more is not built" in lib.tvmkv_last_error().decode()


def test_more_work_items_than_a_launch_has_are_refused():
    lib = tvm_amd.lib()
    assert lib.tvmkv_mxfp4_batch_prefill_paged_kv(*prefill_args(total_q=1 << 30)) == -1
    assert "too many work items" in lib.tvmkv_last_error().decode()


@pytest.mark.parametrize("entry, changes", [("mxfp4_append", dict(n=0, pages=None)), ("mxfp4_read_kv", dict(n=0, pages=None)),
                                            ("mxfp4_batch_decode_paged_kv", dict(batch=0, q=None)),
                                            ("mxfp4_batch_prefill_paged_kv", dict(batch=0, q=None)),
                                            ("mxfp4_batch_prefill_paged_kv", dict(total_q=0, q=None))])
def test_nothing_to_do_is_no_error(entry, changes):
    assert getattr(tvm_amd.lib(), "tvmkv_" + entry)(*ENTRIES[entry](**changes)) == 0


def test_python_entry_points_check_their_tensors():
    torch = pytest.importorskip("torch")
    from tvm_amd import KVError, kernels

    pages = kernels.mxfp4_pages(2, 2, 16, 128, device="cpu")
    assert pages.shape == (2, 2, 2, 16, 68) and pages.dtype == torch.uint8
    rows = torch.zeros((1, 2, 128), dtype=torch.float16)
    slots = torch.zeros(1, dtype=torch.int32)
    for bad, text in (((pages.float(), rows, rows, slots), "must be uint8"), ((pages[0], rows, rows, slots), "expected (num_pages, 2"),
                      ((pages, rows.float(), rows, slots), "float16"), ((pages, rows, rows, slots.long()), "int32"),
                      ((pages, rows, rows[:0], slots), "v_data has shape"), ((pages, rows, rows, slots), "device memory")):
        with pytest.raises(KVError, match=text.replace("(", r"\(")):
            kernels.mxfp4_append(*bad)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    q, lse = torch.zeros((1, 4, 128), dtype=torch.float16), torch.zeros((1, 4))
    for bad, text in (((q, pages, i32(2), i32(1), i32(2), q, lse, 1.0), "length_info has shape"),
                      ((q, pages, i32(2), i32(1), i32(1), q, lse.half(), 1.0), "lse must be float32"),
                      ((q, pages, i32(3), i32(1), i32(2), q, lse, 1.0), "q has shape"),
                      ((q, pages, i32(2), i32(1), i32(1), q[:, :2], lse, 1.0), "output has shape")):
        with pytest.raises(KVError, match=text):
            kernels.mxfp4_batch_decode_paged_kv(*bad)
    with pytest.raises(KVError, match="q_indptr has shape"):
        kernels.mxfp4_batch_prefill_paged_kv(q, i32(3), pages, i32(2), i32(1), i32(1), q, lse, 1, 1.0)


def test_tensor_level_entry_points_check_their_tensors():
    torch = pytest.importorskip("torch")
    from tvm_amd import KVError
    from tvm_amd import dlpack as dl

    f16, i32, f32, u8 = torch.float16, torch.int32, torch.float32, torch.uint8

    def z(*shape, dtype=f16):
        return dl.tensor(torch.zeros(*shape, dtype=dtype))

    pages = z(10, 2, 2, 16, 68, dtype=u8)
    append = dict(pages=pages, k=z(3, 2, 128), v=z(3, 2, 128), pos=z(3, dtype=i32))
    decode = dict(q=z(3, 8, 128), pages=pages, indptr=z(4, dtype=i32), indices=z(7, dtype=i32), info=z(3, dtype=i32), out=z(3, 8, 128),
                  lse=z(3, 8, dtype=f32))
    prefill = dict(q=z(9, 8, 128), q_indptr=z(4, dtype=i32), pages=pages, indptr=z(4, dtype=i32), indices=z(7, dtype=i32),
                   info=z(3, dtype=i32), out=z(9, 8, 128), lse=z(9, 8, dtype=f32))

    def fails(name, args, text, *scalars):
        with pytest.raises(KVError) as e:
            dl.call(name, *args.values(), *scalars, stream=0)
        assert e.value.code == -1 and text in str(e.value), str(e.value)

    fails("mxfp4_append", {**append, "pages": z(10, 2, 2, 16, 128)}, "pages must be uint8")
    fails("mxfp4_append", {**append, "pages": z(10, 2, 2, 16, 64, dtype=u8)}, "pages has shape (10, 2, 2, 16, 64), expected")
    fails("mxfp4_append", {**append, "k": z(3, 2, 128, dtype=f32)}, "k_data must be float16")
    fails("mxfp4_append", {**append, "v": z(2, 2, 128)}, "v_data has shape (2, 2, 128)")
    fails("mxfp4_append", {**append, "pos": None}, "append_position_map is NULL")
    back = {"pages": pages, "pos": append["pos"], "k": append["k"], "v": z(3, 1, 128)}
    fails("mxfp4_read_kv", back, "v_data has shape (3, 1, 128)")
    fails("mxfp4_batch_decode_paged_kv", {**decode, "q": z(4, 8, 128), "out": z(4, 8, 128), "lse": z(4, 8, dtype=f32)}, "q has shape", 0.1)
    fails("mxfp4_batch_decode_paged_kv", {**decode, "info": z(2, 3, dtype=i32)}, "length_info has shape (2, 3), expected (3, batch)", 0.1)
    fails("mxfp4_batch_decode_paged_kv", {**decode, "lse": z(3, 4, dtype=f32)}, "lse has shape (3, 4)", 0.1)
    fails("mxfp4_batch_prefill_paged_kv", {**prefill, "q_indptr": z(5, dtype=i32)}, "qo_indptr has shape (5), expected (batch + 1,)", 1, 0.1)
    fails("mxfp4_batch_prefill_paged_kv", {**prefill, "out": z(9, 8, 64)}, "out has shape", 1, 0.1)


def test_forks_past_the_end_of_a_long_copy_log():
    cache = tvm_amd.Mxfp4KVCache([4, 256, 64, 16, 0], 1, 4, 2, 64, device="cpu")
    pages = cache.pages[0]
    cache.add_sequence(0)
    cache.begin_forward([0], [20])
    cache.end_forward()
    target = None
    for i in range(8300):  # the host cache keeps the last 1024 of its copies when they become more than 8192
        if target is not None:
            pages[source, 0, 0, :8] = i % 251
            pages[target] = 255
        cache.fork_sequence(0, 1, 5)
        (source, target, _), = cache._host.copies_since(10**9)[0]
        assert pages[target].equal(pages[source]), i
        cache.remove_sequence(1)
