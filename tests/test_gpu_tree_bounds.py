"""Attention of drafted trees over the longest rows and of the widest trees, on the GPU."""
import random

import pytest
import torch

import _tree
from _paged_blocks import close
from modelcore_amd.kernels.flash_attn import flash_attn
from test_gpu_tree_attention import Call

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,T,D,n", [
    (F32, 70, 32, 140_000_000), (F32, 70, 32, 1 << 28), (F32, 70, 128, 1 << 26), (F32, 3, 32, 1 << 28), (F32, 1, 8, (1 << 30) - 64),
    (BF, 70, 64, 1 << 29), (BF, 40, 32, (1 << 30) - 64), (BF, 3, 64, 1 << 29)])
@pytest.mark.parametrize("where", [0, 0.5, 0.96, 1])
def test_one_key_among_hundreds_of_millions(dtype, T, D, n, where):
    """A row on pages that repeat, cut into as many ranges as one KV head has workgroups: the one key that is like the
    queries, at its start, in its middle, near its end or its last, gives its value to every node."""
    page, pool = 16, 96
    g = torch.Generator().manual_seed(7)
    k = torch.zeros(pool, page, 1, D, dtype=dtype, device=DEV)
    v = torch.randn(pool, page, 1, D, generator=g).to(dtype).to(DEV)
    table = (torch.arange(-(-(n + T) // page), device=DEV) % (pool - 1)).int()[None]
    at = int(where * (n - 1))
    table[0, at // page] = pool - 1  # a page of its own
    like = torch.ones(D, dtype=dtype)
    k[pool - 1, at % page, 0] = like.to(DEV)
    q = (like * (200 / D ** 0.5)).expand(1, T, 1, D).to(DEV)  # 200 more than the other keys' scores
    words = -(-T // 64)
    masks = torch.tensor([_tree.words_of(nodes, words) for nodes in _tree.ancestors([i - 1 for i in range(T)])],
                         dtype=torch.int64, device=DEV)[None]
    y = flash_attn.flash_attn_paged_tree_with_kvcache(
        q, k, v, tree_masks=masks, block_table=table, cache_seqlens=torch.tensor([n], dtype=torch.int32, device=DEV))
    # The others weigh at most 2^30 exp(-199); a weight and the sum are each rounded, and so is the mean.
    want = v[pool - 1, at % page, 0].double().cpu().expand(1, T, 1, D)
    close(y, want, torch.finfo(dtype).eps * want.abs() + 2.0 ** -24)


@pytest.mark.parametrize("window", [0, 5, 100, 190])
@pytest.mark.parametrize("T,H,H_kv,D,dtype", [(1024, 2, 1, 64, BF), (400, 4, 1, 128, BF), (500, 2, 2, 32, F32), (330, 4, 1, 128, F32)])
def test_wide_trees_behind_narrow_windows(T, H, H_kv, D, dtype, window):
    """Keys cut into ranges of which most lie among the nodes: a chain, whose nodes see those just before them, and a
    tree, whose nodes see some far before them."""
    rng = random.Random(T)
    near = [max(-1, i - rng.choice([1, 1, 2])) for i in range(T)]
    far = [-1] + [rng.randrange(i) for i in range(1, T)]
    Call([700, 60], [_tree.ancestors(near), _tree.ancestors(far)], H, H_kv, D, 64, dtype, window, max_pages=64).check()
