"""Steps of a paged cache at their edges: replays where the eager step would raise, steps of no tokens."""
import pytest
import torch

from modelcore_amd.model import ModelManager
from modelcore_amd.runtime import Runtime
from test_gpu_paged_model import DEV, config
from test_model_host import awake

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fused", [True, False])
def test_replays_stop_at_the_rotary_table(fused):
    """The cache is longer than the table of 512 positions: the host raises before the replay that would
    pass it, with nothing moved, and the replays up to it give the eager step's logits."""
    mgr = ModelManager(Runtime(torch.float32))
    model = awake(mgr.create_model(config(layers=2), device=DEV, seed=0))
    model.set_fused_epilogue(fused)
    model.cache_inference_weights()
    prompt = torch.arange(2 * 507, device=DEV)[None] % 500
    ids = torch.arange(12, device=DEV).view(6, 1, 2)
    with torch.inference_mode():
        caches = [mgr.new_paged_kv_cache(model, batch_size=2, seq_len=600) for _ in range(2)]
        for c in caches:
            model(prompt, kv_cache=c.begin(507))
        eager, cache = caches
        want = [model(ids[i], kv_cache=eager.begin(1)).clone() for i in range(5)]
        column = ids[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [model(column, kv_cache=cache.begin(1)).clone()]
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = model(column, kv_cache=cache.begin(1))
        for i in range(1, 5):
            column.copy_(ids[i])
            cache.note_device_step(1)
            graph.replay()
            got.append(out.clone())
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        before = cache.pages_free
        with pytest.raises(AssertionError, match="rotary"):
            cache.note_device_step(1)
        assert cache.lengths == [512, 512] == cache.cache_seqlens.tolist()
        assert cache.pages_free == before == cache.free_count.item()
        cache.release([0, 1])  # the table's positions are the next requests'
        cache.note_device_step(1)
        graph.replay()
        assert out.isfinite().all() and cache.cache_seqlens.tolist() == [1, 1]


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_of_no_tokens(dtype, fused):
    mgr = ModelManager(Runtime(dtype))
    model = awake(mgr.create_model(config(layers=2), device=DEV, seed=0))
    model.set_fused_epilogue(fused)
    none = torch.zeros(1, 0, dtype=torch.long, device=DEV)
    with torch.inference_mode():
        cache = mgr.new_paged_kv_cache(model, batch_size=2, seq_len=64)
        model(torch.arange(6, device=DEV)[None], kv_cache=cache.begin(3))
        assert model(none, kv_cache=cache.begin(0)).shape == (1, 0, 500)
        assert model.last_logits(none, cache.begin([0, 0]), None).shape == (0, 500)
        assert cache.lengths == [3, 3] == cache.cache_seqlens.tolist()
        model(torch.arange(2, device=DEV)[None], kv_cache=cache.begin(1))
        assert cache.lengths == [4, 4]
