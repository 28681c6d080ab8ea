"""Python face of the kernel launchers of libtvmkv.so.

Function names and positional arguments are those of the reference's kernels
(python/tvm/relax/frontend/nn/llm/_page_kernels.py, _decode_kernels.py, _prefill_kernels.py,
position_embedding.py) as the cache calls them (src/runtime/vm/attn_backend.h:239-242,
:392-395, :511-514; src/runtime/vm/paged_kv_cache.cc:728, :1361-1372, :1550, :1718, :2292).
Tensors are torch tensors in device memory; shapes are read from them the way the reference's
``T.match_buffer`` does.  Launches go to torch's current stream.
"""
import ctypes

import torch

from ._lib import KVError, check, lib


def _p(t):
    if t is None:
        return ctypes.c_void_p(0)
    if not t.is_contiguous():
        raise KVError(-1, "kernel arguments must be contiguous")
    if not t.is_cuda:
        raise KVError(-4, "kernel arguments must live in device memory")
    return ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _f16(*tensors):
    for t in tensors:
        if t.dtype != torch.float16:
            raise KVError(-2, f"only float16 K/V/Q data is built, got {t.dtype}")


def _i32(*tensors):
    for t in tensors:
        if t is not None and t.dtype != torch.int32:
            raise KVError(-1, f"index arrays must be int32, got {t.dtype}")


def fused_rope(qkv, position_map, q, k, v, apply_rope, rope_scale=1.0, rope_theta=1e4):
    _f16(qkv, q, k, v)
    _i32(position_map)
    n, _, d = qkv.shape
    check(lib().tvmkv_fused_rope(_p(qkv), _p(position_map), _p(q), _p(k), _p(v), int(apply_rope), n, q.shape[1],
                                 k.shape[1], d, float(rope_scale), float(rope_theta), _stream()))


def fused_rope_scaled(qkv, position_map, q, k, v, apply_rope, rope_scaling, rope_scale=1.0, rope_theta=1e4,
                      rope_ext_factors=None):
    """fused_rope with one of the reference's frequency variants: rope_scaling is the reference's dictionary
    (rope_type llama3 / longrope / yarn and its parameters, position_embedding.py:258-299); rope_ext_factors the
    float32 device tensor of a longrope model (long factors, then short ones)."""
    from .dlpack import RopeScaling
    _f16(qkv, q, k, v)
    _i32(position_map)
    if rope_ext_factors is not None and rope_ext_factors.dtype != torch.float32:
        raise KVError(-1, "rope_ext_factors must be float32")
    n, _, d = qkv.shape
    scaling = RopeScaling.from_dict(rope_scaling)
    check(lib().tvmkv_fused_rope_scaled(_p(qkv), _p(position_map), _p(q), _p(k), _p(v), int(apply_rope),
                                        _p(rope_ext_factors), ctypes.c_void_p(ctypes.addressof(scaling)), n, q.shape[1],
                                        k.shape[1], d, float(rope_scale), float(rope_theta), _stream()))


def fused_rope_append(qkv, position_map, q, k, v, apply_rope, pages, append_position_map, rope_scale=1.0,
                      rope_theta=1e4):
    """fused_rope and tir_kv_cache_transpose_append in one launch.  q=None: the q rows are not written
    (batch_prefill_cached_and_new_kv_fused_q reads and rotates them from qkv)."""
    _f16(qkv, k, v, pages)
    if q is not None:
        _f16(q)
    _i32(position_map, append_position_map)
    n, _, d = qkv.shape
    num_pages, _, hkv, ps, _ = pages.shape
    check(lib().tvmkv_fused_rope_append(_p(qkv), _p(position_map), _p(q), _p(k), _p(v), int(apply_rope), _p(pages),
                                        _p(append_position_map), n, qkv.shape[1] - 2 * k.shape[1], k.shape[1], d,
                                        num_pages, ps, float(rope_scale), float(rope_theta), _stream()))


def tir_kv_cache_transpose_append(pages, k_data, v_data, position_map):
    _f16(pages, k_data, v_data)
    _i32(position_map)
    num_pages, _, hkv, ps, d = pages.shape
    check(lib().tvmkv_kv_cache_transpose_append(_p(pages), _p(k_data), _p(v_data), _p(position_map),
                                                position_map.shape[0], num_pages, hkv, ps, d, _stream()))


def tir_kv_cache_transpose_append_mla(pages, kv_data, position_map):
    _f16(pages, kv_data)
    _i32(position_map)
    num_pages, ps, d = pages.shape
    check(lib().tvmkv_kv_cache_transpose_append_mla(_p(pages), _p(kv_data), _p(position_map),
                                                    position_map.shape[0], num_pages, ps, d, _stream()))


def _scaling_arg(rope_scaling):
    """The reference's rope_scaling dictionary (position_embedding.py:258-299) as the C description, kept
    alive by the caller for the duration of the call; None = the default frequencies."""
    from .dlpack import RopeScaling
    scaling = RopeScaling.from_dict(rope_scaling)
    return scaling, ctypes.c_void_p(ctypes.addressof(scaling))


def batch_prefill_ragged_kv(q, q_indptr, k, v, kv_indptr, q_rope_position, k_rope_pos_offset, output, lse,
                            causal, rotary_mode, rope_scale, rope_theta, sm_scale, rope_scaling=None):
    """rope_scaling: the frequency variant of the in-kernel RoPE (rotary_mode = 1), the reference's dictionary."""
    _f16(q, k, v, output)
    _i32(q_indptr, kv_indptr, q_rope_position, k_rope_pos_offset)
    args = (_p(q), _p(q_indptr), _p(k), _p(v), _p(kv_indptr), _p(q_rope_position), _p(k_rope_pos_offset), _p(output),
            _p(lse), int(causal), int(rotary_mode), float(rope_scale), float(rope_theta), float(sm_scale),
            q_indptr.shape[0] - 1, q.shape[0], q.shape[1], k.shape[1], q.shape[2], v.shape[2])
    if rope_scaling:
        keep, ptr = _scaling_arg(rope_scaling)
        check(lib().tvmkv_batch_prefill_ragged_kv_scaled(*args, ptr, _stream()))
    else:
        check(lib().tvmkv_batch_prefill_ragged_kv(*args, _stream()))


def batch_prefill_paged_kv(q, q_indptr, pages, page_indptr, page_values, length_info, k_rope_pos_offset,
                           q_rope_position, output, lse, causal, rotary_mode, rope_scale, rope_theta, sm_scale,
                           sliding_window_size=1024, merge_into=False, rope_scaling=None):
    """merge_into: output / lse hold an attention state of the same rows; merge into it instead of
    overwriting (one launch for the paged kernel and merge_state_inplace).  rope_scaling: the frequency
    variant of the in-kernel RoPE (rotary_mode = 1), the reference's dictionary."""
    _f16(q, pages, output)
    _i32(q_indptr, page_indptr, page_values, length_info, k_rope_pos_offset, q_rope_position)
    num_pages, _, hkv, ps, d = pages.shape
    args = (_p(q), _p(q_indptr), _p(pages), _p(page_indptr), _p(page_values), _p(length_info), _p(k_rope_pos_offset),
            _p(q_rope_position), _p(output), _p(lse), int(causal), int(rotary_mode), float(rope_scale),
            float(rope_theta), float(sm_scale), q_indptr.shape[0] - 1, q.shape[0], page_values.shape[0], num_pages,
            q.shape[1], hkv, d, ps, int(length_info.dim() == 2), int(sliding_window_size))
    if rope_scaling:
        keep, ptr = _scaling_arg(rope_scaling)
        check(lib().tvmkv_batch_prefill_paged_kv_scaled(*args, int(bool(merge_into)), ptr, _stream()))
    else:
        fn = lib().tvmkv_batch_prefill_paged_kv_merge if merge_into else lib().tvmkv_batch_prefill_paged_kv
        check(fn(*args, _stream()))


def batch_prefill_cached_and_new_kv(q, q_indptr, k, v, pages, page_indptr, page_values, last_page_len, output, lse,
                                    sm_scale):
    """Ragged causal self-attention over the new tokens, paged attention over the cached ones and
    the merge of the two, in one pass."""
    _f16(q, k, v, pages, output)
    _i32(q_indptr, page_indptr, page_values, last_page_len)
    num_pages, _, hkv, ps, d = pages.shape
    check(lib().tvmkv_batch_prefill_cached_and_new_kv(
        _p(q), _p(q_indptr), _p(k), _p(v), _p(pages), _p(page_indptr), _p(page_values), _p(last_page_len),
        _p(output), _p(lse), float(sm_scale), q_indptr.shape[0] - 1, q.shape[0], page_values.shape[0], num_pages,
        q.shape[1], hkv, d, ps, _stream()))


def batch_prefill_cached_and_new_kv_fused_q(qkv, q_rope_position, apply_rope, rope_scale, rope_theta, q_indptr, k, v,
                                            pages, page_indptr, page_values, last_page_len, output, lse, sm_scale):
    """batch_prefill_cached_and_new_kv with the queries read from the fused qkv tensor and rotated inside
    the kernel."""
    _f16(qkv, k, v, pages, output)
    _i32(q_rope_position, q_indptr, page_indptr, page_values, last_page_len)
    num_pages, _, hkv, ps, d = pages.shape
    hq = qkv.shape[1] - 2 * hkv
    check(lib().tvmkv_batch_prefill_cached_and_new_kv_fused_q(
        _p(qkv), _p(q_rope_position), int(apply_rope), float(rope_scale), float(rope_theta), _p(q_indptr), _p(k),
        _p(v), _p(pages), _p(page_indptr), _p(page_values), _p(last_page_len), _p(output), _p(lse), float(sm_scale),
        q_indptr.shape[0] - 1, qkv.shape[0], page_values.shape[0], num_pages, hq, hkv, d, ps, _stream()))


def fused_decode_step(qkv, pages, page_indptr, page_values, last_page_len, q_rope_position, append_position_map,
                      output, lse, apply_rope, rope_scale, rope_theta, sm_scale):
    """One launch for the decode step of a layer: split of qkv, RoPE, append of the new k / v rows and
    decode attention (tvmkv_fused_decode_step); the page table covers the new tokens."""
    _f16(qkv, pages, output)
    _i32(page_indptr, page_values, last_page_len, q_rope_position, append_position_map)
    num_pages, _, hkv, ps, d = pages.shape
    hq = qkv.shape[1] - 2 * hkv
    check(lib().tvmkv_fused_decode_step(
        _p(qkv), _p(pages), _p(page_indptr), _p(page_values), _p(last_page_len), _p(q_rope_position),
        _p(append_position_map), _p(output), _p(lse), int(apply_rope), float(rope_scale), float(rope_theta),
        float(sm_scale), qkv.shape[0], page_values.shape[0], num_pages, hq, hkv, d, ps, _stream()))


def batch_decode_paged_kv(q, pages, page_indptr, page_values, length_info, k_rope_pos_offset, q_rope_position,
                          output, lse, rotary_mode, rope_scale, rope_theta, sm_scale, noalloc=False, rope_scaling=None):
    """noalloc=True calls the entry point that takes its scratch memory from the library's built-in
    per-device array instead of allocating (tvmkv_batch_decode_paged_kv_noalloc).  rope_scaling: the
    frequency variant of the in-kernel RoPE (rotary_mode = 1), the reference's dictionary."""
    _f16(q, pages, output)
    _i32(page_indptr, page_values, length_info, k_rope_pos_offset, q_rope_position)
    num_pages, _, hkv, ps, d = pages.shape
    args = (_p(q), _p(pages), _p(page_indptr), _p(page_values), _p(length_info), _p(k_rope_pos_offset),
            _p(q_rope_position), _p(output), _p(lse), int(rotary_mode), float(rope_scale), float(rope_theta),
            float(sm_scale), q.shape[0], page_values.shape[0], num_pages, q.shape[1], hkv, d, ps,
            int(length_info.dim() == 2))
    if rope_scaling:
        keep, ptr = _scaling_arg(rope_scaling)
        check(lib().tvmkv_batch_decode_paged_kv_scaled(*args, ptr, _stream()))
        return
    entry = lib().tvmkv_batch_decode_paged_kv_noalloc if noalloc else lib().tvmkv_batch_decode_paged_kv
    check(entry(*args, _stream()))


def batch_tree_attn(q, q_indptr, k, v, kv_indptr, q_rope_position, mn_indptr, mask, output, lse, rotary_mode,
                    rope_scale, rope_theta, sm_scale, rope_scaling=None):
    _f16(q, k, v, output)
    _i32(q_indptr, kv_indptr, q_rope_position, mn_indptr, mask)
    args = (_p(q), _p(q_indptr), _p(k), _p(v), _p(kv_indptr), _p(q_rope_position), _p(mn_indptr), _p(mask), _p(output),
            _p(lse), int(rotary_mode), float(rope_scale), float(rope_theta), float(sm_scale), q_indptr.shape[0] - 1,
            q.shape[0], q.shape[1], k.shape[1], q.shape[2])
    if rope_scaling:
        keep, ptr = _scaling_arg(rope_scaling)
        check(lib().tvmkv_batch_tree_attn_scaled(*args, ptr, _stream()))
    else:
        check(lib().tvmkv_batch_tree_attn(*args, _stream()))


def tree_attn_paged_kv(q, q_indptr, pages, page_indptr, page_values, length_info, k_rope_pos_offset,
                       q_rope_position, output, lse, rotary_mode, rope_scale, rope_theta, sm_scale,
                       tree_order_indptr, tree_order):
    _f16(q, pages, output)
    _i32(q_indptr, page_indptr, page_values, length_info, k_rope_pos_offset, q_rope_position, tree_order_indptr,
         tree_order)
    num_pages, _, hkv, ps, d = pages.shape
    check(lib().tvmkv_tree_attn_paged_kv(
        _p(q), _p(q_indptr), _p(pages), _p(page_indptr), _p(page_values), _p(length_info), _p(k_rope_pos_offset),
        _p(q_rope_position), _p(output), _p(lse), int(rotary_mode), float(rope_scale), float(rope_theta),
        float(sm_scale), _p(tree_order_indptr), _p(tree_order), q_indptr.shape[0] - 1, q.shape[0],
        page_values.shape[0], num_pages, q.shape[1], hkv, d, ps, int(length_info.dim() == 2), _stream()))


def batch_prefill_paged_kv_mla(q, q_indptr, pages, page_indptr, page_values, length_info, output, lse, causal,
                               sm_scale):
    _f16(q, pages, output)
    _i32(q_indptr, page_indptr, page_values, length_info)
    num_pages, ps, d_qk = pages.shape
    d_latent = output.shape[2]
    check(lib().tvmkv_batch_prefill_paged_kv_mla(
        _p(q), _p(q_indptr), _p(pages), _p(page_indptr), _p(page_values), _p(length_info), _p(output), _p(lse),
        int(causal), float(sm_scale), q_indptr.shape[0] - 1, q.shape[0], page_values.shape[0], num_pages,
        q.shape[1], d_latent, d_qk - d_latent, ps, _stream()))


def merge_state_inplace(v, s, v_other, s_other):
    _f16(v, v_other)
    n, h, d = v.shape
    check(lib().tvmkv_merge_state_inplace(_p(v), _p(s), _p(v_other), _p(s_other), n, h, d, _stream()))


def copy_single_page(pages, src_page_id, tgt_page_id, copy_length):
    _f16(pages)
    num_pages, _, hkv, ps, d = pages.shape
    check(lib().tvmkv_copy_single_page(_p(pages), src_page_id, tgt_page_id, copy_length, num_pages, hkv, ps, d,
                                       _stream()))


def copy_single_page_mla(pages, src_page_id, tgt_page_id, copy_length):
    _f16(pages)
    num_pages, ps, d = pages.shape
    check(lib().tvmkv_copy_single_page_mla(_p(pages), src_page_id, tgt_page_id, copy_length, num_pages, ps, d,
                                           _stream()))


def tir_kv_cache_debug_get_kv(pages, position_map, k_data, v_data, layer_id):
    _f16(pages, k_data, v_data)
    _i32(position_map)
    num_pages, _, hkv, ps, d = pages.shape
    check(lib().tvmkv_kv_cache_debug_get_kv(_p(pages), _p(position_map), _p(k_data), _p(v_data), layer_id,
                                            position_map.shape[0], num_pages, hkv, ps, d, _stream()))


def tir_kv_cache_debug_get_kv_mla(pages, position_map, kv_data, layer_id):
    _f16(pages, kv_data)
    _i32(position_map)
    num_pages, ps, d = pages.shape
    check(lib().tvmkv_kv_cache_debug_get_kv_mla(_p(pages), _p(position_map), _p(kv_data), layer_id,
                                                position_map.shape[0], num_pages, ps, d, _stream()))


def compact_kv_copy(pages, copy_length_indptr, copy_src_dst_pos, batch_size):
    _f16(pages)
    _i32(copy_length_indptr, copy_src_dst_pos)
    num_pages, _, hkv, ps, d = pages.shape
    check(lib().tvmkv_compact_kv_copy(_p(pages), _p(copy_length_indptr), _p(copy_src_dst_pos), batch_size,
                                      copy_src_dst_pos.shape[1], num_pages, hkv, ps, d, _stream()))


# ---- a cache held in 4 bits (include/tvmkv.h has its format) ----------------------------------------------------


def mxfp4_pages(num_pages, h_kv, page_size, head_dim, device="cuda"):
    """A pool of pages for mxfp4_append and the kernels that read them: 17 * head_dim / 32 bytes a row."""
    return torch.zeros((num_pages, 2, h_kv, page_size, 17 * head_dim // 32), dtype=torch.uint8, device=device)


# These calls take a few microseconds on the device, so that their checks are written to be cheap: one pass over the tensors
# of a kind, shapes compared as they are, addresses as integers.


# (torch.cuda.current_stream builds an object first, 2.8 us; the handle alone takes 0.1)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda device: torch.cuda.current_stream(device).cuda_stream)


def _mxfp4_call(entry, tensors, *rest):
    for t in tensors:
        if not t.is_cuda or not t.is_contiguous():
            _p(t)  # refuses it
    check(entry(*[t.data_ptr() for t in tensors], *rest, _raw_stream(tensors[0].get_device())))


def _mxfp4_pool(pages, head_dim):
    shape = pages.shape
    if pages.dtype != torch.uint8:
        raise KVError(-1, f"pages of 4-bit rows must be uint8, got {pages.dtype}")
    if len(shape) != 5 or shape[1] != 2 or shape[4] * 32 != 17 * head_dim:
        raise KVError(-1, f"pages has shape {tuple(shape)}, expected (num_pages, 2, h_kv, page_size, 17 * {head_dim} / 32)")
    return shape


def _shape(t, name, expected):
    if t.shape != expected:
        raise KVError(-1, f"{name} has shape {tuple(t.shape)}, expected {expected}")


def _mxfp4_rows(entry, pages, k_data, v_data, position_map, tensors):
    _f16(k_data, v_data)
    _i32(position_map)
    d = k_data.shape[-1]
    num_pages, _, hkv, ps, _ = _mxfp4_pool(pages, d)
    n = position_map.shape[0]
    _shape(k_data, "k_data", (n, hkv, d))
    _shape(v_data, "v_data", (n, hkv, d))
    _mxfp4_call(entry, tensors, n, num_pages, hkv, ps, d)


def mxfp4_append(pages, k_data, v_data, position_map):
    """Quantises the rows k_data, v_data (tokens, h_kv, head_dim) into the slots position_map (negative: none)."""
    _mxfp4_rows(lib().tvmkv_mxfp4_append, pages, k_data, v_data, position_map, (pages, k_data, v_data, position_map))


def mxfp4_read_kv(pages, position_map, k_data, v_data):
    """The rows of the slots position_map as fp16, into k_data and v_data (tokens, h_kv, head_dim)."""
    _mxfp4_rows(lib().tvmkv_mxfp4_read_kv, pages, k_data, v_data, position_map, (pages, position_map, k_data, v_data))


def _mxfp4_attention(q, pages, page_indptr, page_values, length_info, output, lse):
    _f16(q, output)
    _i32(page_indptr, page_values, length_info)
    if lse.dtype != torch.float32:
        raise KVError(-1, f"lse must be float32, got {lse.dtype}")
    rows, hq, d = q.shape
    num_pages, _, hkv, ps, _ = _mxfp4_pool(pages, d)
    batch = page_indptr.shape[0] - 1
    _shape(output, "output", (rows, hq, d))
    _shape(lse, "lse", (rows, hq))
    sliding = length_info.dim() == 2
    _shape(length_info, "length_info", (3, batch) if sliding else (batch,))
    return rows, batch, (page_values.shape[0], num_pages, hq, hkv, d, ps, int(sliding))


def mxfp4_batch_decode_paged_kv(q, pages, page_indptr, page_values, length_info, output, lse, sm_scale):
    """batch_decode_paged_kv over 4-bit pages: one query token a sequence, keys stored rotated."""
    rows, batch, sizes = _mxfp4_attention(q, pages, page_indptr, page_values, length_info, output, lse)
    if rows != batch:
        raise KVError(-1, f"q has shape {tuple(q.shape)}, expected {(batch,) + tuple(q.shape[1:])}")
    _mxfp4_call(lib().tvmkv_mxfp4_batch_decode_paged_kv, (q, pages, page_indptr, page_values, length_info, output, lse), sm_scale,
                batch, *sizes)


def mxfp4_batch_prefill_paged_kv(q, q_indptr, pages, page_indptr, page_values, length_info, output, lse, causal, sm_scale):
    """batch_prefill_paged_kv over 4-bit pages: q_indptr (batch + 1) query tokens of each sequence, keys stored rotated."""
    rows, batch, sizes = _mxfp4_attention(q, pages, page_indptr, page_values, length_info, output, lse)
    _i32(q_indptr)
    _shape(q_indptr, "q_indptr", (batch + 1,))
    _mxfp4_call(lib().tvmkv_mxfp4_batch_prefill_paged_kv, (q, q_indptr, pages, page_indptr, page_values, length_info, output, lse),
                causal, sm_scale, batch, rows, *sizes)


# ---- eviction by attention weight (include/tvmkv.h says what the calls compute) -----------------------------------


def key_weight_pages(num_pages, h_kv, page_size, device="cuda"):
    """Sums of the attention weights that stored tokens have received, for the *_weights calls: none yet.

    The calls only add to them, and move_kept_tokens leaves those of the places that it empties.  Whoever stores a token sets the sums of
    its slot to 0 (sums[slots // page_size, :, slots % page_size] = 0), or it begins with those of the token that was there."""
    return torch.zeros((num_pages, h_kv, page_size), dtype=torch.float32, device=device)


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _weights_call(entry, tensors, *rest):
    """tensors: all on one device, which is the current one for the call; None: NULL."""
    index = tensors[0].get_device()  # -1: not in device memory
    pointers = []
    for t in tensors:
        if t is None:
            pointers.append(None)
            continue
        if t.get_device() != index or index < 0 or not t.is_contiguous():
            _p(t)
            raise KVError(-1, f"kernel arguments must be on one device, got {t.device} and {tensors[0].device}")
        pointers.append(t.data_ptr())
    if index == _current_device():
        check(entry(*pointers, *rest, _raw_stream(index)))
    else:
        with torch.cuda.device(index):
            check(entry(*pointers, *rest, _raw_stream(index)))


def _key_weights(key_weights, hkv, ps):
    if key_weights.dtype != torch.float32:
        raise KVError(-1, f"key_weights must be float32, got {key_weights.dtype}")
    if key_weights.dim() != 3 or key_weights.shape[1] != hkv or key_weights.shape[2] != ps:
        raise KVError(-1, f"key_weights has shape {tuple(key_weights.shape)}, expected (num_weight_pages, {hkv}, {ps})")


def _weighed_attention(q, pages, page_indptr, page_values, length_info, output, lse, key_weights, weight_page_values):
    _f16(q, pages, output)
    _i32(page_indptr, page_values, length_info, weight_page_values)
    if lse.dtype != torch.float32:
        raise KVError(-1, f"lse must be float32, got {lse.dtype}")
    rows, hq, d = q.shape
    if pages.dim() != 5 or pages.shape[1] != 2 or pages.shape[4] != d:
        raise KVError(-1, f"pages has shape {tuple(pages.shape)}, expected (num_pages, 2, h_kv, page_size, {d})")
    num_pages, _, hkv, ps, _ = pages.shape
    batch = page_indptr.shape[0] - 1
    _shape(output, "output", (rows, hq, d))
    _shape(lse, "lse", (rows, hq))
    _shape(length_info, "length_info", (batch,))
    _shape(weight_page_values, "weight_page_values", page_values.shape)
    _key_weights(key_weights, hkv, ps)
    return rows, batch, (page_values.shape[0], num_pages, hq, hkv, d, ps)


def batch_decode_paged_kv_weights(q, pages, page_indptr, page_values, length_info, output, lse, key_weights, weight_page_values,
                                  sm_scale):
    """batch_decode_paged_kv, keys stored rotated, that also adds each stored token's attention weight to key_weights
    (num_weight_pages, h_kv, page_size) on the pages weight_page_values, which lie beside page_values."""
    rows, batch, sizes = _weighed_attention(q, pages, page_indptr, page_values, length_info, output, lse, key_weights,
                                            weight_page_values)
    if rows != batch:
        raise KVError(-1, f"q has shape {tuple(q.shape)}, expected {(batch,) + tuple(q.shape[1:])}")
    _weights_call(lib().tvmkv_batch_decode_paged_kv_weights,
                  (q, pages, page_indptr, page_values, length_info, output, lse, key_weights, weight_page_values), sm_scale, batch, *sizes)


def batch_prefill_paged_kv_weights(q, q_indptr, pages, page_indptr, page_values, length_info, output, lse, key_weights,
                                   weight_page_values, causal, observed, sm_scale):
    """batch_prefill_paged_kv, keys stored rotated, that also adds each stored token's attention weight to key_weights; observed > 0:
    that of the last `observed` queries of each sequence only."""
    rows, batch, sizes = _weighed_attention(q, pages, page_indptr, page_values, length_info, output, lse, key_weights,
                                            weight_page_values)
    _i32(q_indptr)
    _shape(q_indptr, "q_indptr", (batch + 1,))
    _weights_call(lib().tvmkv_batch_prefill_paged_kv_weights,
                  (q, q_indptr, pages, page_indptr, page_values, length_info, output, lse, key_weights, weight_page_values), int(causal),
                  int(observed), sm_scale, batch, rows, *sizes)


def select_kept_tokens(key_weights, page_indptr, weight_page_values, length_info, keep, kept, num_sinks, num_recent):
    """Which tokens stay, into kept (batch, h_kv, max_keep): of each sequence keep[b] at most, for each kv head its first num_sinks,
    its last num_recent and those with the largest sums; kept names the token that each place takes, -1 behind the last."""
    _i32(page_indptr, weight_page_values, length_info, keep, kept)
    batch = page_indptr.shape[0] - 1
    if key_weights.dim() != 3 or key_weights.dtype != torch.float32:
        raise KVError(-1, f"key_weights must be float32 (num_weight_pages, h_kv, page_size), got {key_weights.dtype} of shape "
                          f"{tuple(key_weights.shape)}")
    _, hkv, ps = key_weights.shape
    _shape(length_info, "length_info", (batch,))
    _shape(keep, "keep", (batch,))
    if kept.dim() != 3 or kept.shape[:2] != (batch, hkv):
        raise KVError(-1, f"kept has shape {tuple(kept.shape)}, expected ({batch}, {hkv}, max_keep)")
    _weights_call(lib().tvmkv_select_kept_tokens, (key_weights, page_indptr, weight_page_values, length_info, keep, kept), int(num_sinks),
                  int(num_recent), batch, weight_page_values.shape[0], hkv, ps, kept.shape[2])


def move_kept_tokens(pages, key_weights, page_indptr, page_values, weight_page_values, kept):
    """Moves the rows of the tokens `kept`, K, V and (key_weights not None) their sums, to their places at the front of each sequence's
    pages; float16 or float32 pages.  The sums of the places behind them stay as they are (key_weight_pages)."""
    _i32(page_indptr, page_values, weight_page_values, kept)
    if pages.dtype not in (torch.float16, torch.float32):
        raise KVError(-2, f"only float16 and float32 rows are built, got {pages.dtype}")
    if pages.dim() != 5 or pages.shape[1] != 2:
        raise KVError(-1, f"pages has shape {tuple(pages.shape)}, expected (num_pages, 2, h_kv, page_size, head_dim)")
    num_pages, _, hkv, ps, d = pages.shape
    batch = page_indptr.shape[0] - 1
    if key_weights is not None:
        _key_weights(key_weights, hkv, ps)
        _shape(weight_page_values, "weight_page_values", page_values.shape)
    if kept.dim() != 3 or kept.shape[:2] != (batch, hkv):
        raise KVError(-1, f"kept has shape {tuple(kept.shape)}, expected ({batch}, {hkv}, max_keep)")
    _weights_call(lib().tvmkv_move_kept_tokens, (pages, key_weights, page_indptr, page_values, weight_page_values, kept), batch,
                  page_values.shape[0], num_pages, hkv, ps, d, 8 * pages.element_size(), kept.shape[2])
