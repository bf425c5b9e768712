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


@pytest.fixture
def plans(monkeypatch):
    """paged_reserve without a device: the plans it was asked for; `fail` set, it raises."""
    from modelcore_amd.kernels import paged

    class Plans(list):
        fail = False

    made = Plans()

    def reserve(table, seqlens, counts, free, count, *, total, page_size):
        if made.fail:
            raise RuntimeError("no launch")
        made.append(counts.tolist())
        z = torch.zeros(total, dtype=torch.int32)
        return paged.PagedPlan(z.long(), z, torch.zeros(len(counts) + 1, dtype=torch.int32), z[:1])

    monkeypatch.setattr(paged, "paged_reserve", reserve)
    return made


class Layers(torch.nn.Module):
    """A body that counts its runs and needs no device."""

    def __init__(self):
        super().__init__()
        self.blocks, self.runs = [], 0

    def forward_carry(self, x, kv_cache):
        self.runs += 1
        return x, None


def model_over(layers):
    from modelcore_amd.model import Model
    model = Model.__new__(Model)
    torch.nn.Module.__init__(model)
    model.embedding, model.body, model.unembedding = torch.nn.Identity(), layers, lambda x, h: x
    model._check_paged = lambda idx, kv_cache: None
    return model


def test_a_step_that_is_not_its_caches_open_one_runs_no_layer(plans):
    """Run before, or begun before a reset: its slots may be other rows' by now. Nothing is launched, and
    the step that is open stays so."""
    cache, layers = make(), Layers()
    model = model_over(layers)
    first = cache.begin(2)
    ids = torch.zeros(1, 4, 1)
    model(ids, kv_cache=first)
    assert layers.runs == 1 and cache.lengths == [2, 2] == cache.cache_seqlens.tolist()
    for open_one in (False, True):
        step = cache.begin(2) if open_one else None
        for run in (lambda: model(ids, kv_cache=first), lambda: model.last_logits(ids, first, None)):
            with pytest.raises(AssertionError, match="run once"):
                run()
        assert layers.runs == 1 and cache.lengths == [2, 2] == cache.cache_seqlens.tolist()
        assert cache._open is step
    cache.reset()
    anew = cache.begin(1)
    with pytest.raises(AssertionError, match="reset"):
        model(ids, kv_cache=step)
    with pytest.raises(AssertionError, match="reset"):
        step.advance(4)
    assert layers.runs == 1 and cache.lengths == [0, 0]
    model(ids[:, :2], kv_cache=anew)
    assert layers.runs == 2 and cache.lengths == [1, 1] == cache.cache_seqlens.tolist()


def test_a_plan_that_fails_leaves_the_account(plans):
    cache = make()
    plans.fail = True
    with pytest.raises(RuntimeError, match="no launch"):
        cache.begin([20, 3])
    assert cache.pages_free == cache.n_pages and cache.lengths == [0, 0]
    plans.fail = False
    step = cache.begin([20, 3])
    assert cache.pages_free == cache.n_pages - 3 and plans == [[20, 3]] and step.total == 23
