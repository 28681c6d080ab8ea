"""The 4-bit cache object without a GPU: what it refuses, and that a step ends with what made it."""
import pytest

torch = pytest.importorskip("torch")

from tvm_amd import KVError, Mxfp4KVCache  # noqa: E402


def cache_of(**changes):
    shape = dict(cache_config=[4, 256, 64, 16, 0], num_layers=2, num_qo_heads=4, num_kv_heads=2, head_dim=64, device="cpu")
    return Mxfp4KVCache(**{**shape, **changes})


def attend(cache, rows, layer=0):
    f16 = torch.float16
    cache.attention_with_fused_qkv(layer, 0.1, torch.zeros((rows, 8, 64), dtype=f16), torch.zeros((rows, 4, 64), dtype=f16))


def refuses_attention(cache, rows):
    with pytest.raises(KVError, match="between begin_forward and end_forward"):
        attend(cache, rows)


def test_no_step_is_left_after_clear():
    cache = cache_of()
    cache.add_sequence(0)
    cache.begin_forward([0], [3])
    cache.clear()
    refuses_attention(cache, 3)


def test_no_step_is_left_after_a_begin_forward_that_failed():
    cache = cache_of()
    cache.add_sequence(0)
    cache.begin_forward([0], [3])
    with pytest.raises(KVError):
        cache.begin_forward([7], [1])  # no such sequence
    refuses_attention(cache, 3)


def test_no_step_is_left_after_end_forward():
    cache = cache_of()
    refuses_attention(cache, 3)
    cache.add_sequence(0)
    cache.begin_forward([0], [3])
    cache.end_forward()
    refuses_attention(cache, 3)


@pytest.mark.parametrize("layer", [-1, 2])
def test_a_layer_that_the_cache_does_not_have_is_refused(layer):
    cache = cache_of()
    cache.add_sequence(0)
    cache.begin_forward([0], [3])
    with pytest.raises(KVError, match="layer id .* out of range"):
        attend(cache, 3, layer)


@pytest.mark.parametrize("changes, text", [
    (dict(head_dim=80), "head_dim 80 is not built"),
    (dict(cache_config=[4, 256, 64, 24, 0]), "page_size must be a multiple of 16, got 24"),
    (dict(num_qo_heads=5), "5 query heads"),
    (dict(num_layers=0), "0 layers"),
])
def test_shapes_that_the_kernels_do_not_have_are_refused_before_memory_is_taken(changes, text):
    with pytest.raises(KVError, match=text):
        cache_of(**changes)
