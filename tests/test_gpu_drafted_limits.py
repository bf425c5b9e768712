"""Decoding with more drafted tokens than pages, positions or a tree have room for, on the GPU."""
import pytest
import torch

from modelcore_amd.model import ModelManager
from modelcore_amd.runtime import Runtime
from test_gpu_tree_model import DEV, awake, config

pytestmark = pytest.mark.gpu


def test_a_full_pool_and_an_eager_drafter_change_nothing():
    """The likeliest tokens, whatever the guesses and however few pages there are for them."""
    mgr = ModelManager(Runtime(torch.float32))
    model = awake(mgr.create_model(config(D=64), device=DEV, seed=0))
    prompts = [[5, 6, 7] * 5, [9] * 8, [3, 1, 4, 1, 5]]

    def run(drafter, **kw):
        dec = mgr.new_drafted_decoder(model, prompts, max_tokens=40, drafter=drafter, **kw)
        steps = 0
        while min(map(len, dec.tokens)) < 20 + 15 and steps < 60:
            done = [b for b, t in enumerate(dec.tokens) if dec.running[b] and len(t) >= 20 + len(prompts[b])]
            dec.finish(done)
            if not any(dec.running):
                break
            dec.step()
            steps += 1
        dec.finish(range(3))
        assert dec.cache.pages_free == dec.cache.free_count.item() == dec.cache.n_pages
        return [t[:20 + len(p)] for t, p in zip(dec.tokens, prompts)]

    want = run(lambda t: ([], []))
    right = {tuple(p): r for p, r in zip(prompts, want)}

    def known(tokens):  # a chain of what comes next, and hundreds of others
        full = next(r for p, r in right.items() if tuple(tokens[:len(p)]) == p)
        ahead = full[len(tokens):]
        return ahead + [11] * 1500, list(range(len(ahead))) + [0] * 1500

    for kw in (dict(), dict(n_pages=7), dict(n_pages=8, page_size=16), dict(n_pages=3, page_size=64)):
        assert run(known, **kw) == want
