"""A model over drafted trees on the GPU: plan, pre-attention step, attention, verification and keeping as a
serving loop runs them together."""
import random

import pytest
import torch

import _tree
from modelcore_amd.generate import lookup_drafts
from modelcore_amd.model import ModelManager
from modelcore_amd.runtime import Runtime
from modelcore_amd.sampling import verify_drafts
from test_gpu_paged_model import config, ids_of
from test_model_host import awake

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def alone(model, tokens):
    """Logits behind the last of `tokens`, without a cache."""
    return model(torch.tensor([tokens], device=DEV))[0, -1]


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("dtype,D,shared,atol", [(torch.float32, 64, False, 1e-4), (torch.float32, 32, True, 1e-4),
                                                 (torch.bfloat16, 128, True, 0.06), (torch.bfloat16, 64, False, 0.06)])
def test_a_server_of_trees(dtype, D, shared, atol, fused):
    """Rows with trees beside rows that sit out, windows in every second layer: the logits of every node against its
    path alone, and again after a path of each tree was kept. The tolerances are those of the mixed rows' test."""
    mgr = ModelManager(Runtime(dtype))
    model = awake(mgr.create_model(config(D=D, window=20, shared=shared), device=DEV, seed=0))
    model.set_fused_epilogue(fused)
    rng = random.Random(D)
    rows = [[rng.randrange(500) for _ in range(n)] for n in (30, 3, 61, 16)]
    with torch.inference_mode():
        cache = mgr.new_paged_kv_cache(model, batch_size=4, seq_len=200, n_pages=34, page_size=16)
        model(ids_of(rows), kv_cache=cache.begin([len(r) for r in rows]))
        for turn in range(4):
            sizes = [[7, 1, 40, 0], [12, 12, 12, 12], [0, 33, 5, 2], [1, 1, 1, 1]][turn]
            trees = [_tree.random_parents(rng, n, 0.1) for n in sizes]
            tokens = [[rng.randrange(500) for _ in t] for t in trees]
            step = cache.begin_tree(trees)
            assert step.plan.refused.item() == 0
            logits = model(ids_of(tokens), kv_cache=step)[0]
            at, kept = 0, []
            for b, up in enumerate(map(_tree.ancestors, trees)):
                for i, path in enumerate(up):
                    want = alone(model, rows[b] + [tokens[b][j] for j in path])
                    torch.testing.assert_close(logits[at + i], want, atol=atol, rtol=0)
                at += len(up)
                kept.append(rng.choice(up) if up else [])
            longest = max(map(len, kept))
            took = cache.keep(step, torch.tensor([k + [-1] * (longest - len(k)) for k in kept], dtype=torch.int32, device=DEV),
                              torch.tensor([len(k) for k in kept], dtype=torch.int32, device=DEV))
            assert took == [len(k) for k in kept]
            for b, path in enumerate(kept):
                rows[b] += [tokens[b][j] for j in path]
            assert cache.cache_seqlens.tolist() == cache.lengths == [len(r) for r in rows]
            assert cache.free_count.item() == cache.pages_free
        # A token of each row behind what it has kept, as a sequence.
        logits = model(ids_of([[7]] * 4), kv_cache=cache.begin(1))[0]
        for b in range(4):
            torch.testing.assert_close(logits[b], alone(model, rows[b] + [7]), atol=atol, rtol=0)
        cache.release(range(4))
    assert cache.free_count.item() == cache.pages_free == 34
    assert sorted(cache.free_pages.tolist()) == list(range(34))


@torch.inference_mode()
def likeliest(model, tokens, n):
    """Every token after the first n is the likeliest there, up to twice what two runs' logits differ by."""
    logits = model(torch.tensor([tokens[:-1]], device=DEV))[0, n - 1:]
    got = logits.gather(1, torch.tensor(tokens[n:], device=DEV)[:, None])[:, 0]
    assert bool((got >= logits.amax(-1) - 2e-4).all())


def test_drafted_decoding_is_the_models_own():
    """Greedy decoding with guesses from the text, with the right ones, with wrong ones and with none, rows that end
    among others: each token is the model's likeliest, and right guesses are accepted whole."""
    mgr = ModelManager(Runtime(torch.float32))
    model = awake(mgr.create_model(config(D=64, window=40), device=DEV, seed=0))
    rng = random.Random(1)
    prompts = [[rng.randrange(500) for _ in range(n)] for n in (20, 1, 50)]
    prompts[1] = [3, 4, 5] * 6
    known = {}

    def decode(drafter, steps, **kw):
        dec = mgr.new_drafted_decoder(model, prompts, max_tokens=60, drafter=drafter, **kw)
        gained = [dec.step() for _ in range(steps)]
        assert all(len(x) >= 1 for g in gained for x in g)
        for row, p, parts in zip(dec.tokens, prompts, zip(*gained)):
            assert len(row) == len(p) + 1 + sum(map(len, parts))
            likeliest(model, row, len(p))
        assert dec.cache.free_count.item() == dec.cache.pages_free
        return dec

    plain = decode(lambda t: ([], []), 24)
    assert all(len(r) == len(p) + 25 for r, p in zip(plain.tokens, prompts))
    for r, p in zip(plain.tokens, prompts):
        known[tuple(p)] = r

    def right(tokens):
        full = next(r for p, r in known.items() if tokens[:len(p)] == list(p))
        ahead = full[len(tokens):len(tokens) + 3]
        return [11, *ahead, 499], [0, *([0] + list(range(2, 1 + len(ahead))))[:len(ahead)], 0]

    good = decode(right, 5)
    for r, want, p in zip(good.tokens, plain.tokens, prompts):
        assert len(r) == len(p) + 1 + 5 * 4 and r == want[:len(r)]
    decode(lambda t: ([t[-1]] * 6, [0, 0, 1, 2, 2, 5]), 10)
    dec = decode(lookup_drafts, 8, page_size=32)
    dec.finish([1])
    gained = dec.step()
    assert gained[1] == [] and gained[0] and gained[2]
    dec.finish([0, 1, 2])
    assert dec.cache.pages_free == dec.cache.free_count.item() == dec.cache.n_pages
    assert dec.step() == [[], [], []]


def test_drafts_at_the_end_of_a_rows_room():
    """Guesses past the positions a row has are left out, and a row without room is refused before a launch."""
    mgr = ModelManager(Runtime(torch.float32))
    model = awake(mgr.create_model(config(D=64), device=DEV, seed=0))
    dec = mgr.new_drafted_decoder(model, [[1, 2, 3, 4]], max_tokens=6, drafter=lambda t: ([5] * 9, [0] * 9))
    n = 0
    while dec.cache.lengths[0] < 10:
        n += len(dec.step()[0])
    assert n == 6 and dec.cache.lengths == [10]
    with pytest.raises(AssertionError, match="exceeds cache length"):
        dec.step()


def test_sampled_drafts_follow_the_seed():
    mgr = ModelManager(Runtime(torch.bfloat16))
    model = awake(mgr.create_model(config(D=128), device=DEV, seed=0))
    prompts = [[5, 6, 7] * 5, [9] * 8]

    def run(seed):
        dec = mgr.new_drafted_decoder(model, prompts, max_tokens=80, temperature=0.8, seed=seed)
        for _ in range(12):
            dec.step()
        return dec.tokens

    assert run(1) == run(1) != run(2)


def test_a_step_of_trees_is_not_captured():
    mgr = ModelManager(Runtime(torch.bfloat16))
    model = awake(mgr.create_model(config(D=128), device=DEV, seed=0))
    cache = mgr.new_paged_kv_cache(model, batch_size=1, seq_len=40)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=DEV)
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            x.add_(1)
            cache.begin_tree([[-1]])
    torch.cuda.synchronize()
    assert cache.pages_free == cache.n_pages and cache._open is None


def test_a_layer_in_one_graph():
    """A whole step behind the cache's account, pages to verification, as one graph over tensors that a caller keeps:
    each replay against the same calls without it."""
    from modelcore_amd.kernels.flash_attn import flash_attn
    from modelcore_amd.kernels.paged import paged_keep, paged_reserve, paged_tree
    from modelcore_amd.kernels.qk_epilogue import rope_norm_scale_append_paged
    B, n, H, H_kv, D, page, V = 3, 9, 8, 2, 128, 16, 600
    g = torch.Generator(device=DEV).manual_seed(3)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    head = randn(V, H * D) * 0.05
    cos, sin = torch.cos(randn(300, D // 2)).bfloat16(), torch.sin(randn(300, D // 2)).bfloat16()
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 3, 5, 5] * B, dtype=torch.int32, device=DEV)
    new = torch.full((B,), n, dtype=torch.int32, device=DEV)
    qkv, tokens, numbers = randn(B * n, H + 2 * H_kv, D).bfloat16(), torch.zeros(B * n, dtype=torch.long, device=DEV), randn(B * n)

    def state():
        i = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        k = torch.zeros(30, page, H_kv, D, dtype=torch.bfloat16, device=DEV)
        return [torch.full((B, 12), -1, dtype=torch.int32, device=DEV), i(0, 0, 0),
                torch.arange(30, dtype=torch.int32, device=DEV), i(30), k, k.clone()]

    def step(s):
        table, held, free, count, k, v = s
        plan = paged_reserve(table, held, new, free, count, total=B * n, page_size=page)
        tree = paged_tree(parents, plan.cu_seqlens, held, max_seqlen=n)
        q = rope_norm_scale_append_paged(qkv[:, :H], cos, sin, tree.positions, qkv[:, H:H + H_kv], qkv[:, H + H_kv:], k, v, plan.slots)
        y = flash_attn.flash_attn_paged_tree_with_kvcache(q.view(B, n, H, D), k, v, tree_masks=tree.masks.view(B, n, 1),
                                                          block_table=table, cache_seqlens=held)
        logits = y.reshape(B * n, H * D).float() @ head.t()
        done = verify_drafts(logits, tokens, parents, plan.cu_seqlens, numbers, draft_probs=None, max_seqlen=n)
        paged_keep(k, v, table, held, new, done.kept, done.counts, free, count)
        return [y, *done]

    a, b = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a)
    torch.cuda.current_stream().wait_stream(side)
    step(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(a)
    for turn in range(6):
        qkv.copy_(randn(*qkv.shape))
        tokens.copy_(torch.randint(0, V, tokens.shape, generator=g, device=DEV))
        numbers.copy_(torch.rand(numbers.shape, generator=g, device=DEV) * (0.002 if turn % 2 else 1))
        graph.replay()
        want = step(b)
        torch.cuda.synchronize()
        for x, y in zip(out + a, want + b):
            assert torch.equal(x, y)
    assert b[1].tolist() > [7, 7, 7]
