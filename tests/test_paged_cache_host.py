"""PagedKVCache's own account on the CPU, with the page plan stood in for."""
import pytest
import torch

from modelcore_amd.cache import PagedKVCache, PagedStep


def make(rows=2, seq_len=64, **kw):
    return PagedKVCache(rows, 1, seq_len, 32, 1, "cpu", torch.float32, **kw)


def captured(cache, n):
    """The step of a capture, without its plan on the device."""
    counts = torch.full((cache.batch_size,), n, dtype=torch.int32)
    return PagedStep(cache, [n] * cache.batch_size, counts, None, True)


def test_a_captured_step_leaves_its_rotary_table_for_the_replays():
    cache = make()
    step = captured(cache, 3)
    step.bound_positions(50)
    captured(cache, 1).bound_positions(20)  # a second graph, of a model with a shorter table
    for _ in range(6):
        cache.note_device_step(3)
    free = cache.pages_free
    with pytest.raises(AssertionError, match="rotary embeddings cache: 21 > 20"):
        cache.note_device_step(3)
    assert cache.lengths == [18, 18] and cache.pages_free == free
    cache.note_device_step(2)
    assert cache.lengths == [20, 20]
    with pytest.raises(AssertionError, match="exceeds cache length"):
        cache.note_device_step(45)
