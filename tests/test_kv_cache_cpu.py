"""Pages and lengths of the paged cache, on the CPU."""
import pytest
import torch

from sharq_b200.decoder import rope_tables
from sharq_b200.kv_cache import PagedKVCache


def make(sequences=3, max_tokens=40, page_size=8, pages=None, layers=2, **kw):
    cos, sin = rope_tables(max_tokens, 64, 1e4, torch.device("cpu"))
    return PagedKVCache(layers, 2, 64, sequences, max_tokens, cos, sin, page_size, pages, **kw)


def check(cache):
    """Every page belongs to one sequence or is free; the device side says what the host side says."""
    held = [p for pages in cache._held for p in pages]
    assert sorted(held + cache._free) == list(range(cache.k.shape[1]))
    for i, pages in enumerate(cache._held):
        assert cache.table[i, :len(pages)].tolist() == pages
        assert len(pages) >= -(-cache.lengths[i] // cache.page_size)
    assert cache.device_lengths.tolist() == cache.lengths


def test_sequences_grow_and_end():
    cache = make()
    assert cache.k.shape == (2, 15, 2, 8, 64) and cache.k_scale is None
    cache.reserve([5, 16, 0])
    check(cache)
    assert [len(h) for h in cache._held] == [1, 2, 0]
    cache.advance([5, 16, 0])
    cache.reserve([3, 1, 40])
    cache.advance([3, 1, 40])
    check(cache)
    assert cache.lengths == [8, 17, 40] and [len(h) for h in cache._held] == [1, 3, 5]
    cache.free(2)
    check(cache)
    cache.reserve([1, 0, 9])
    cache.advance([1, 0, 9])
    check(cache)
    assert cache.lengths == [9, 17, 9]


def test_what_does_not_fit_changes_nothing():
    cache = make(pages=4)
    cache.reserve([8, 8, 8])
    cache.advance([8, 8, 8])
    table = cache.table.clone()
    with pytest.raises(RuntimeError, match="1 free pages, 2 are needed"):
        cache.reserve([1, 1, 0])
    with pytest.raises(RuntimeError, match="does not fit"):
        cache.reserve([33, 0, 0])
    check(cache)
    assert torch.equal(cache.table, table) and cache.lengths == [8, 8, 8]
    with pytest.raises(ValueError, match="reserved before"):
        cache.advance([0, 0, 1])
    with pytest.raises(ValueError, match="one count"):
        cache.reserve([1, 1])
    with pytest.raises(ValueError, match="one count"):
        cache.reserve([1, 1, -1])


def test_prompt_steps_and_layers():
    cache = make(dtype=torch.float8_e4m3fn, k_scale=torch.rand(2, 2))
    assert cache.v_scale.tolist() == [[1, 1], [1, 1]] and cache.k.dtype == torch.float8_e4m3fn
    cache.reserve([9] * 3)
    positions, sequences = cache.prompt_step(9)
    assert positions.tolist() == list(range(9)) * 3 and sequences.tolist() == [i for i in range(3) for _ in range(9)]
    assert positions.dtype == sequences.dtype == torch.int32
    layer = cache.layer(1, positions, sequences, None)
    assert layer.table.shape == (3, 2) and layer.k.data_ptr() == cache.k[1].data_ptr()
    assert torch.equal(layer.k_scale, cache.k_scale[1]) and layer.k_scale.is_contiguous()


def test_arguments_that_are_refused():
    with pytest.raises(ValueError, match="positive"):
        make(sequences=0)
    with pytest.raises(ValueError, match="bfloat16 or"):
        make(dtype=torch.float16)
    with pytest.raises(ValueError, match="belong to"):
        make(k_scale=torch.ones(2, 2))
    with pytest.raises(ValueError, match="layers, kv_heads"):
        make(dtype=torch.float8_e4m3fn, v_scale=torch.ones(2))
    cos, sin = rope_tables(8, 64, 1e4, torch.device("cpu"))
    with pytest.raises(ValueError, match="rotary tables"):
        PagedKVCache(1, 2, 64, 1, 9, cos, sin)
