"""Decoding with drafted tokens on the CPU, with the model and the operators stood in for: how many guesses each
step takes."""
import pytest
import torch

from modelcore_amd import sampling
from modelcore_amd.generate import DraftedDecoder
from test_tree_cache_host import cache  # noqa: F401  (two rows of 64 positions, seven pages of 16)


class Model:
    def __init__(self):
        self.trees = []

    def get_device(self):
        return torch.device("cpu")

    def last_logits(self, ids, step, _):
        step.advance(ids.shape[1])
        return torch.zeros(len(step.lens), 5)

    def forward(self, ids, kv_cache):
        self.trees.append((kv_cache.lens, kv_cache.parents.tolist(), ids[0].tolist()))
        kv_cache.advance(ids.shape[1])
        return torch.zeros(1, ids.shape[1], 5)


@pytest.fixture
def decoder(cache, monkeypatch):  # noqa: F811
    def verify(logits, ids, parents, cu, numbers, *, temperature, max_seqlen):
        n = len(cache.lengths)  # no guess is accepted, and 9 comes next
        kept = torch.zeros(n, max_seqlen, dtype=torch.int32)
        return sampling.Verified(kept, torch.ones(n, dtype=torch.int32), torch.full((n, max_seqlen), 9))

    monkeypatch.setattr(sampling, "verify_drafts", verify)

    class Manager:
        @staticmethod
        def new_paged_kv_cache(model, **kw):
            return cache

    def make(prompts, drafter):
        model = Model()
        return DraftedDecoder(model, Manager, prompts, max_tokens=50, drafter=drafter), model

    return make


def chain(n):
    return list(range(100, 100 + n)), list(range(n))


def test_more_guesses_than_the_free_pages_hold_are_shortened_alike(decoder):
    dec, model = decoder([[1] * 16, [2] * 30], lambda tokens: chain(40 if tokens[0] == 1 else 2))
    # Pages: one and two of seven. Row 0 would take three more and row 1 (30 + 3 tokens) one.
    assert dec.cache.pages_free == 4
    assert dec.step() == [[9], [9]]
    assert model.trees[-1] == ([41, 3], [-1, *range(40), -1, 0, 1], [9, *range(100, 140), 9, 100, 101])
    assert dec.cache.lengths == [17, 31] and dec.cache.pages_free == 3
    dec.cache.pages_free = 1  # as if another row had the others
    assert dec.step() == [[9], [9]]
    # Row 0 has 15 positions left in its page and row 1 one: a page more is row 1's, so both may have 14 guesses.
    assert model.trees[-1][0] == [15, 3]
    assert dec.step() == [[9], [9]]
    assert model.trees[-1][0] == [14, 3] and dec.cache.lengths == [19, 33]  # the page goes to row 1's last token
    assert dec.cache.pages_free == 0
    assert dec.step() == [[9], [9]]
    assert model.trees[-1][0] == [13, 3] and dec.cache.lengths == [20, 34]


def test_pages_for_the_last_tokens_alone(decoder):
    dec, model = decoder([[1] * 31, [2] * 31], lambda tokens: chain(7))
    dec.cache.pages_free = 0
    assert dec.step() == [[9], [9]]
    assert model.trees[-1] == ([1, 1], [-1, -1], [9, 9]) and dec.cache.lengths == [32, 32]
    with pytest.raises(AssertionError, match="2 pages needed, 0 of 7 free"):
        dec.step()
    dec.cache.pages_free = 1
    with pytest.raises(AssertionError, match="2 pages needed, 1 of 7 free"):
        dec.step()
    dec.finish([0])
    dec.step()
    assert model.trees[-1][0] == [0, 8]


def test_more_guesses_than_a_tree_has_room_for(decoder, monkeypatch):
    from modelcore_amd.kernels import paged
    dec, model = decoder([[1], [2]], lambda tokens: chain(60))
    monkeypatch.setattr(paged, "MAX_TREE_NODES", 11)
    dec.step()
    assert model.trees[-1][0] == [11, 11]
    assert model.trees[-1][1][:11] == [-1, *range(10)]


def test_a_drafter_of_thousands(decoder):
    dec, model = decoder([[1], [2]], lambda tokens: ([3] * 2000, [0] * 2000))
    dec.step()
    # 62 positions behind the root, of four pages a row; seven pages in all.
    assert model.trees[-1][0] == [47, 47]
