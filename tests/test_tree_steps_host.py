"""Steps of drafted trees that fail on their way, on the CPU with the operators stood in for."""
import pytest
import torch

from test_tree_cache_host import cache, i32  # noqa: F401  (the fixture)


def test_a_step_whose_trees_fail_keeps_its_pages_in_the_account(cache, monkeypatch):  # noqa: F811
    """Its pages are taken on the device when the nodes' positions are made: where those fail, the cache is not
    begun again before it is reset."""
    from modelcore_amd.kernels import paged
    made = paged.paged_tree

    def fails(*a, **kw):
        raise RuntimeError("out of memory")

    monkeypatch.setattr(paged, "paged_tree", fails)
    with pytest.raises(RuntimeError, match="out of memory"):
        cache.begin_tree([[-1] * 20, [-1]])
    assert cache.pages_free == 7 - 3 and cache.lengths == [0, 0]
    monkeypatch.setattr(paged, "paged_tree", made)
    for again in (lambda: cache.begin(1), lambda: cache.begin_tree([[-1], []]), lambda: cache.release([0]),
                  lambda: cache.note_device_step(1)):
        with pytest.raises(AssertionError, match="has not run"):
            again()
    cache.reset()
    assert cache.pages_free == 7
    step = cache.begin_tree([[-1] * 20, [-1]])
    step.advance(21)
    assert cache.keep(step, torch.zeros(2, 20, dtype=torch.int32), i32([3, 1])) == [3, 1]
