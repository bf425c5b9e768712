"""A model over a paged cache on the GPU: the page plan, the pre-attention step and the attention over
pages as a server runs them together, against the reference's goldens and the contiguous cache."""
import pytest
import torch

import _goldens
from modelcore_amd.model import ComponentSpec, ModelConfig, ModelManager
from modelcore_amd.runtime import Runtime
from test_model_host import awake

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def ids_of(rows):
    return torch.tensor([t for r in rows for t in r], dtype=torch.long, device=DEV)[None]


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("name", _goldens.GOLDENS)
def test_goldens_from_pages(name, fused):
    """A prompt's first tokens, then token by token, gives the reference's logits; rows of other lengths
    beside it change nothing."""
    mgr = ModelManager(Runtime(torch.float32))
    model, idx, logits = _goldens.build(name, mgr, DEV)
    model.set_fused_epilogue(fused)
    idx = idx.to(DEV)
    B, T = idx.shape
    with torch.no_grad():
        cache = mgr.new_paged_kv_cache(model, batch_size=B + 1, seq_len=T + 20, page_size=16)
        other = [3, 1, 4, 1, 5, 9, 2]
        rows = [idx[b, :5].tolist() for b in range(B)]
        out = model(ids_of(rows + [other]), kv_cache=cache.begin([5] * B + [7]))
        parts = [out[0, :5 * B].view(B, 5, -1)]
        for t in range(5, T):
            rows = [[int(idx[b, t])] for b in range(B)]
            if t % 3 == 0:
                out = model(ids_of(rows), kv_cache=cache.begin([1] * B + [0]))
            else:
                out = model(ids_of(rows + [[t]]), kv_cache=cache.begin(1))
            parts.append(out[0, :B].view(B, 1, -1))
    torch.testing.assert_close(torch.cat(parts, dim=1).cpu(), logits, atol=1e-4, rtol=0)


def config(H=8, H_kv=2, D=64, window=-1, layers=3, shared=False):
    blocks = [ComponentSpec("block", {
        "layer_idx": i, "features": [],
        "mixer": ComponentSpec("attention", {
            "n_head": H, "n_kv_head": H_kv, "head_dim": D, "window": window if i % 2 else -1,
            "kv_slot": min(i, layers - 2) if shared else None, "produces_kv": not (shared and i == layers - 1),
            "features": []}),
        "ffn": ComponentSpec("gated_mlp", {"activation": "silu", "hidden_dim": 256})})
        for i in range(layers)]
    return ModelConfig(sequence_len=512, vocab_size=500, n_embd=256, pad_vocab_size_to=64,
                       shared={"rope": ComponentSpec("rotary", {"head_dim": D, "over_compute": 1}),
                               "norm": ComponentSpec("rms_norm", {"eps": None})},
                       input=ComponentSpec("token_embedding", {"smear": False}),
                       body=ComponentSpec("stack", {"blocks": blocks, "features": []}),
                       output=ComponentSpec("lm_head", {"softcap": 15}))


@pytest.mark.parametrize("dtype,D,shared,atol", [(torch.float32, 64, False, 1e-4), (torch.float32, 32, True, 1e-4),
                                                 (torch.bfloat16, 128, True, 0.06), (torch.bfloat16, 64, False, 0.06)])
def test_a_server_of_mixed_rows(dtype, D, shared, atol):
    """Requests arrive, read their prompts in chunks beside others that decode, end, and give their pages
    to the next: every logit against that request alone on a contiguous cache."""
    mgr = ModelManager(Runtime(dtype))
    model = awake(mgr.create_model(config(D=D, window=40, shared=shared), device=DEV, seed=0))
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 500, (n,), generator=g).tolist() for n in (70, 5, 33, 16, 120, 1, 47)]
    steps, chunk, rows = 9, 32, 3
    with torch.inference_mode():
        want = []
        for p in prompts:  # alone, in the same chunks
            c = mgr.new_kv_cache(model, batch_size=1, seq_len=200)
            todo, out = p + [(7 * i + len(p)) % 500 for i in range(steps)], []
            at = 0
            while at < len(todo):
                n = min(chunk, len(p) - at) if at < len(p) else 1
                out.append(model(torch.tensor([todo[at:at + n]], device=DEV), kv_cache=c)[0])
                at += n
            want.append(torch.cat(out))
        cache = mgr.new_paged_kv_cache(model, batch_size=rows, seq_len=200, n_pages=24, page_size=16)
        slots, queue, got = [None] * rows, list(range(len(prompts))), {i: [] for i in range(len(prompts))}
        while queue or any(s is not None for s in slots):
            for r in range(rows):
                if slots[r] is None and queue:
                    i = queue.pop(0)
                    slots[r] = [i, 0, prompts[i] + [(7 * j + len(prompts[i])) % 500 for j in range(steps)]]
            parts = []
            for s in slots:
                if s is None:
                    parts.append([])
                    continue
                i, at, todo = s
                n = min(chunk, len(prompts[i]) - at) if at < len(prompts[i]) else 1
                parts.append(todo[at:at + n])
            step = cache.begin([len(p) for p in parts])
            assert step.plan.refused.item() == 0
            logits = model(ids_of(parts), kv_cache=step)[0]
            at, ended = 0, []
            for r, p in enumerate(parts):
                if slots[r] is None:
                    continue
                got[slots[r][0]].append(logits[at:at + len(p)])
                at += len(p)
                slots[r][1] += len(p)
                if slots[r][1] == len(slots[r][2]):
                    ended.append(r)
                    slots[r] = None
            assert cache.cache_seqlens.tolist() == cache.lengths
            assert cache.free_count.item() == cache.pages_free
            cache.release(ended)
    assert cache.pages_free == cache.n_pages == cache.free_count.item()
    assert sorted(cache.free_pages.tolist()) == list(range(24))
    for i, w in enumerate(want):
        torch.testing.assert_close(torch.cat(got[i]), w, atol=atol, rtol=0)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 128)])
def test_a_captured_step_replays(dtype, D):
    """Single tokens for every row as one graph: each replay reserves its own pages on the device and gives
    the eager step's logits, with eager work in between."""
    mgr = ModelManager(Runtime(dtype))
    model = awake(mgr.create_model(config(D=D, window=20), device=DEV, seed=0))
    model.cache_inference_weights()
    B = 3
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 500, (40, 1, B), generator=g).to(DEV)
    prompt = torch.randint(0, 500, (1, 30 * B), generator=g).to(DEV)

    def make():
        cache = mgr.new_paged_kv_cache(model, batch_size=B, seq_len=80, n_pages=15, page_size=16)
        model(prompt, kv_cache=cache.begin(30))
        return cache

    with torch.inference_mode():
        eager, cache = make(), make()
        want = [model(ids[i], kv_cache=eager.begin(1)).clone() for i in range(40)]
        column = ids[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [model(column, kv_cache=cache.begin(1)).clone()]  # warm-up: a real step
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = model(column, kv_cache=cache.begin(1))
        for i in range(1, 40):
            column.copy_(ids[i])
            cache.note_device_step(1)
            graph.replay()
            got.append(out.clone())
            if i % 7 == 0:
                torch.cuda.synchronize()
                make()
    assert cache.cache_seqlens.tolist() == cache.lengths == [70] * B
    assert cache.free_count.item() == cache.pages_free == 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with pytest.raises(AssertionError, match="exceeds cache length"):
        cache.note_device_step(11)


def test_last_logits_and_refusals():
    mgr = ModelManager(Runtime(torch.float32))
    model = awake(mgr.create_model(config(), device=DEV, seed=0))
    with torch.inference_mode():
        cache = mgr.new_paged_kv_cache(model, batch_size=3, seq_len=600, n_pages=45)
        ids = torch.arange(12, device=DEV)[None]
        step = cache.begin([5, 0, 7])
        last = model.last_logits(ids, step, None)
        assert cache.lengths == [5, 0, 7] and last.shape == (2, 500)
        cache.reset()
        full = model(ids, kv_cache=cache.begin([5, 0, 7]))[0, [4, 11]]
        torch.testing.assert_close(last, full, atol=1e-4, rtol=0)
        step = cache.begin(1)
        with pytest.raises(AssertionError, match="has not run"):
            cache.begin(1)
        with pytest.raises(AssertionError, match="has not run"):
            cache.release([0])
        with pytest.raises(AssertionError, match="one \\(1, total\\) sequence"):
            model(ids[:, :2], kv_cache=step)
        with pytest.raises(AssertionError, match="one \\(1, total\\) sequence"):
            model(ids[0, :3, None], kv_cache=step)
        model(ids[:, :3], kv_cache=step)
        with pytest.raises(AssertionError, match="run once"):
            step.advance(3)
        with pytest.raises(AssertionError, match="exceeds cache length"):
            cache.begin([595, 0, 0])
        with pytest.raises(AssertionError, match="pages needed"):
            cache.begin([500, 0, 500])
        with pytest.raises(AssertionError, match="rotary"):
            model(torch.zeros(1, 508, dtype=torch.long, device=DEV), kv_cache=cache.begin([508, 0, 0]))
        cache.reset()
        for lens in ([1, 1], [1, 1, -1]):
            with pytest.raises(AssertionError):
                cache.begin(lens)
        with pytest.raises(AssertionError):
            cache.release([1, 1])
        with pytest.raises(AssertionError):
            cache.release([3])
        assert cache.pages_free == 45
