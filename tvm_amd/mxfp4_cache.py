"""A paged KV cache held in 4 bits, with the verbs of the fp16 cache.

The page pool, the block tree and the step's index arrays are those of the library's cache object in its host-only form
(``vm.builtin.paged_attention_kv_cache_create`` without a device); the rows live in uint8 pools (``kernels.mxfp4_pages``)
that the 4-bit kernels write and read: 4.25 bits an element, 3.76 times the tokens of an fp16 pool of the same size.

    cache = Mxfp4KVCache([64, 1 << 20, 4096, 16, 0], layers, 32, 8, 128)
    cache.add_sequence(0)
    cache.begin_forward([0], [prompt_length])
    for layer in range(layers):
        cache.attention_with_fused_qkv(layer, 128 ** -0.5, qkv[layer], out[layer])   # appends, attends
    cache.end_forward()
"""
import ctypes

import torch

from . import kernels
from .runtime import KVError, RopeMode, get_global_func


class Mxfp4KVCache:
    """cache_config: the reference's (max batch, max total tokens, prefill chunk, page size, sliding windows), page size
    a multiple of 16.  A step that appends one token to every sequence writes it first and attends to the cache alone; in
    the others the new tokens attend to each other's fp16 rows and to the cached 4-bit ones, and are written afterwards.
    Calls run on torch's current stream; token trees are not built."""

    def __init__(self, cache_config, num_layers, num_qo_heads, num_kv_heads, head_dim, rope_mode=RopeMode.NORMAL, rope_scale=1.0,
                 rope_theta=1e4, device="cuda"):
        if rope_mode == RopeMode.INLINE:
            raise KVError(-2, "a 4-bit cache stores rotated keys: rope_mode INLINE is not built")
        if head_dim not in (64, 96, 128, 256):
            raise KVError(-2, f"a 4-bit cache: head_dim {head_dim} is not built (64, 96, 128, 256)")
        if cache_config[3] <= 0 or cache_config[3] % 16 != 0:
            raise KVError(-2, f"a 4-bit cache: page_size must be a multiple of 16, got {cache_config[3]}")
        if num_layers <= 0 or num_kv_heads <= 0 or num_qo_heads <= 0 or num_qo_heads % num_kv_heads != 0:
            raise KVError(-1, f"a 4-bit cache: bad shape: {num_layers} layers, {num_qo_heads} query heads, {num_kv_heads} kv heads")
        self.num_layers, self.num_qo_heads, self.num_kv_heads, self.head_dim = num_layers, num_qo_heads, num_kv_heads, head_dim
        self.rope = (rope_mode == RopeMode.NORMAL, float(rope_scale), float(rope_theta))
        self.sliding_windows = bool(cache_config[4])
        self._host = get_global_func("vm.builtin.paged_attention_kv_cache_create")(
            list(cache_config), [0, num_layers], num_qo_heads, num_kv_heads, head_dim, head_dim, [0] * num_layers, False,
            int(rope_mode), rope_scale, rope_theta, None, "host")
        num_pages, page_size = self._host.flags()["num_total_pages"], cache_config[3]
        self.pages = [kernels.mxfp4_pages(num_pages, num_kv_heads, page_size, head_dim, device) for _ in range(num_layers)]
        self.device = self.pages[0].device
        self._copied = 0  # length of the host cache's copy log when its copies were done last
        self._step = None

    # ---- sequences -----------------------------------------------------------------------------------------------
    def _verb(self, name, *args):
        return get_global_func("vm.builtin." + name)(self._host, *args)

    def clear(self):
        self._step = None
        self._verb("kv_state_clear")
        self._copied = 0

    def add_sequence(self, seq_id):
        self._verb("kv_state_add_sequence", seq_id)

    def remove_sequence(self, seq_id):
        self._verb("kv_state_remove_sequence", seq_id)

    def fork_sequence(self, parent_id, child_id, fork_pos=-1):
        self._verb("kv_state_fork_sequence", parent_id, child_id, fork_pos)
        self._copy_pages()

    def _copy_pages(self):
        """What the host cache asked for since the last time: pages that a sequence no longer shares from some token on."""
        copies, self._copied = self._host.copies_since(self._copied)
        for source, target, _ in copies:
            for pages in self.pages:
                pages[target].copy_(pages[source])

    def popn(self, seq_id, n):
        self._verb("kv_state_popn", seq_id, n)
        self._copy_pages()  # a sequence that ends inside rows that others share is forked anew

    def enable_sliding_window_for_seq(self, seq_id, window, sinks):
        self._verb("attention_kv_cache_enable_sliding_window_for_seq", seq_id, window, sinks)

    def get_num_available_pages(self):
        return self._verb("attention_kv_cache_get_num_available_pages")

    # ---- a step --------------------------------------------------------------------------------------------------
    def begin_forward(self, seq_ids, append_lengths):
        self._step = None  # until the new one is complete
        self._verb("kv_state_begin_forward", seq_ids, append_lengths)
        flags, total, places = self._host.flags(), 0, []

        def place(*arrays):  # one behind the other, the first at a multiple of 16 bytes
            nonlocal total
            total = -(-total // 4) * 4
            places.append((total, [self._host.aux_data(*a) for a in arrays]))
            total += sum(n for _, n in places[-1][1])
            return len(places) - 1

        info = ["last_page_len"] + (["sliding_window_offset", "sink_size"] if self.sliding_windows else [])
        depths = []
        for d in range(flags["num_depths"]):
            qo_indptr = place(("qo_indptr", d))
            ids = place(("page_indices", d))
            if places[ids][1][0][1] > 0:
                depths.append((qo_indptr, place(("page_indptr", d)), ids, place(*((name, d) for name in info))))
        rest = [place((name,)) for name in ("q_rope_position_map", "append_position_map", "cur_append_lengths_indptr",
                                            "k_ragged_rope_pos_offset")]
        merged = torch.empty(total, dtype=torch.int32, pin_memory=self.device.type == "cuda")
        for at, arrays in places:
            for data, n in arrays:
                ctypes.memmove(merged.data_ptr() + 4 * at, data, 4 * n)
                at += n
        one_each = [bool((merged[at:at + n].diff() == 1).all()) for at, n in self._spans(places, [q for q, *_ in depths])]
        merged = merged.to(self.device, non_blocking=True)
        array = [merged[at:at + n] for at, n in self._spans(places, range(len(places)))]
        self._step = {
            "rows": sum(append_lengths), "append_first": bool(flags["append_before_attn"]),
            "depths": [(one, array[q], array[p], array[i], array[f].view(3, -1) if self.sliding_windows else array[f])
                       for one, (q, p, i, f) in zip(one_each, depths)],
            "positions": array[rest[0]], "slots": array[rest[1]], "indptr": array[rest[2]], "key_positions": array[rest[3]]}

    @staticmethod
    def _spans(places, which):
        return [(places[i][0], sum(n for _, n in places[i][1])) for i in which]

    def end_forward(self):
        self._step = None
        self._verb("kv_state_end_forward")

    def attention_with_fused_qkv(self, layer_id, sm_scale, qkv, out):
        """qkv (rows, num_qo_heads + 2 num_kv_heads, head_dim) of the step's tokens: rotates, appends to the layer's pages and
        attends, into out (rows, num_qo_heads, head_dim)."""
        step = self._step
        if step is None:
            raise KVError(-1, "attention_with_fused_qkv belongs between begin_forward and end_forward")
        if not 0 <= layer_id < self.num_layers:
            raise KVError(-1, f"layer id {layer_id} out of range")
        rows, hq, hkv, d = step["rows"], self.num_qo_heads, self.num_kv_heads, self.head_dim
        for name, t, heads in (("qkv", qkv, hq + 2 * hkv), ("out", out, hq)):
            if tuple(t.shape) != (rows, heads, d):
                raise KVError(-1, f"{name} has shape {tuple(t.shape)}, expected {(rows, heads, d)}")
        pages = self.pages[layer_id]
        q, k, v = (torch.empty((rows, heads, d), dtype=torch.float16, device=self.device) for heads in (hq, hkv, hkv))
        kernels.fused_rope(qkv, step["positions"], q, k, v, *self.rope)
        lse = torch.empty((rows, hq), dtype=torch.float32, device=self.device)
        if step["append_first"]:
            kernels.mxfp4_append(pages, k, v, step["slots"])
        else:
            kernels.batch_prefill_ragged_kv(q, step["indptr"], k, v, step["indptr"], step["positions"], step["key_positions"], out, lse, 1,
                                            0, 1.0, 1e4, sm_scale)
        first = step["append_first"]
        for one_each, qo_indptr, page_indptr, page_ids, length_info in step["depths"]:
            o, s = (out, lse) if first else (torch.empty_like(out), torch.empty_like(lse))
            if one_each:
                kernels.mxfp4_batch_decode_paged_kv(q, pages, page_indptr, page_ids, length_info, o, s, sm_scale)
            else:
                kernels.mxfp4_batch_prefill_paged_kv(q, qo_indptr, pages, page_indptr, page_ids, length_info, o, s, 0, sm_scale)
            if not first:
                kernels.merge_state_inplace(out, lse, o, s)
            first = False
        if not step["append_first"]:
            kernels.mxfp4_append(pages, k, v, step["slots"])
