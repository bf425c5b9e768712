"""A paged cache's steps of drafted trees on the CPU, with the operators stood in for, and the host's side of
decoding with drafts."""
import pytest
import torch

from modelcore_amd.cache import PagedKVCache, TreeStep
from modelcore_amd.generate import lookup_drafts


@pytest.fixture
def cache(monkeypatch):
    from modelcore_amd.kernels import paged

    def reserve(table, seqlens, counts, free, count, *, total, page_size):
        z = torch.zeros(total, dtype=torch.int32)
        return paged.PagedPlan(z.long(), z, torch.zeros(len(counts) + 1, dtype=torch.int32), z[:1])

    def tree(parents, cu, held, *, max_seqlen):
        return paged.TreePlan(parents + 100, parents[:, None].long())

    monkeypatch.setattr(paged, "paged_reserve", reserve)
    monkeypatch.setattr(paged, "paged_tree", tree)
    monkeypatch.setattr(paged, "paged_keep", lambda *a: None)
    monkeypatch.setattr(paged, "paged_release", lambda *a, **kw: None)
    return PagedKVCache(2, 1, 64, 32, 1, "cpu", torch.float32, n_pages=7)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def test_a_step_of_trees_moves_the_account_by_what_is_kept(cache):
    step = cache.begin_tree([[-1, 0, 0, 1] * 5, [-1, 0]])
    assert isinstance(step, TreeStep) and step.lens == [20, 2] and step.max_seqlen == 20 and step.uniform is None
    assert cache.pages_free == 7 - 3 and cache.lengths == [0, 0]
    assert step.positions.tolist()[:3] == [99, 100, 100] and step.parents.tolist()[-2:] == [-1, 0]
    with pytest.raises(AssertionError, match="has not run"):
        cache.begin(1)
    with pytest.raises(AssertionError, match="forward has not run"):
        cache.keep(step, torch.zeros(2, 20, dtype=torch.int32), i32([1, 1]))
    with pytest.raises(AssertionError, match="every row's new tokens"):
        step.advance(21)
    step.advance(22)
    for again in (lambda: cache.begin(1), lambda: cache.begin_tree([[-1], []]), lambda: cache.release([0]),
                  lambda: cache.note_device_step(1)):
        with pytest.raises(AssertionError, match="have not been kept"):
            again()
    with pytest.raises(AssertionError, match="run once"):
        step.check_open()
    assert cache.keep(step, torch.zeros(2, 20, dtype=torch.int32), i32([3, 2])) == [3, 2]
    assert cache.lengths == [3, 2] and cache.pages_free == 5
    with pytest.raises(AssertionError, match="not those this cache has begun"):
        cache.keep(step, torch.zeros(2, 20, dtype=torch.int32), i32([3, 2]))
    cache.begin(1).advance(2)
    assert cache.lengths == [4, 3]


def test_counts_past_the_nodes_or_the_list_count_as_those(cache):
    step = cache.begin_tree([[-1] * 6, []])
    step.advance(6)
    assert cache.keep(step, torch.zeros(2, 4, dtype=torch.int32), i32([9, 5])) == [4, 0]
    step = cache.begin_tree([[], [-1]])
    step.advance(1)
    assert cache.keep(step, torch.zeros(2, 4, dtype=torch.int32), i32([-3, 0])) == [0, 0]
    assert cache.lengths == [4, 0] and cache.pages_free == 6


def test_reset_drops_a_step_of_trees(cache):
    step = cache.begin_tree([[-1], [-1]])
    cache.reset()
    with pytest.raises(AssertionError, match="reset"):
        step.advance(2)
    step = cache.begin_tree([[-1], [-1]])
    step.advance(2)
    cache.reset()
    with pytest.raises(AssertionError, match="not those"):
        cache.keep(step, torch.zeros(2, 1, dtype=torch.int32), i32([1, 1]))
    assert cache.pages_free == 7
    cache.begin(1)


def test_trees_that_are_none_are_refused(cache):
    for bad in ([[0], []], [[-1, 1], []], [[-1, 0, 5], []], [[-2], []]):
        with pytest.raises(AssertionError, match="parent is a node before it"):
            cache.begin_tree(bad)
    with pytest.raises(AssertionError, match="token counts"):
        cache.begin_tree([[-1]])
    with pytest.raises(AssertionError, match="exceeds cache length"):
        cache.begin_tree([[-1] * 65, []])
    with pytest.raises(AssertionError, match="pages needed"):
        cache.begin_tree([[-1] * 64, [-1] * 64])
    with pytest.raises(AssertionError, match="1025 nodes"):
        cache.begin_tree([[-1] * 1025, []])
    assert cache.pages_free == 7 and cache._open is None


def test_a_trees_positions_are_bounded_by_its_depth(cache):
    """Rotary tables hold a row's length and its deepest path, however many nodes there are."""
    step = cache.begin_tree([[-1] + [0] * 30 + [30], [-1, 0]])
    assert step.longest == 3
    step.bound_positions(3)
    with pytest.raises(AssertionError, match="rotary embeddings cache: 3 > 2"):
        step.bound_positions(2)
    with pytest.raises(TypeError, match="no last token"):
        step.last


def test_lookup_drafts():
    text = [1, 2, 3, 4, 5, 1, 2, 3, 9, 9, 1, 2]
    # Of [1, 2] the last occurrence before was followed by 3 9 9 1, the one before that by 3 4 5 1.
    assert lookup_drafts(text) == ([3, 9, 9, 1, 4, 5, 1], [0, 1, 2, 3, 1, 5, 6])
    assert lookup_drafts(text, width=1, length=2) == ([3, 9], [0, 1])
    assert lookup_drafts(text, ngram=1) == ([3, 9, 9, 1, 4, 5, 1], [0, 1, 2, 3, 1, 5, 6])
    assert lookup_drafts([7, 7, 7], ngram=1) == ([7, 7], [0, 1])
    for short in ([5], [1, 2], [1, 2, 3]):
        assert lookup_drafts(short) == ([], [])
