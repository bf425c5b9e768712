"""Checked mode of what a paged cache keeps of drafted trees, through its entry point."""
import pytest
import torch

from modelcore_amd.kernels import flash_attn as fa
from modelcore_amd.kernels.paged import paged_keep

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_checked_mode_names_what_is_wrong_and_moves_nothing():
    pools = [torch.randn(1, 9, 16, 2, 8, device=DEV) for _ in range(2)]
    before = [p.clone() for p in pools]
    table, held = i32([[3, 0, 8, -1], [5, -1, -1, -1]]), i32([20, 16])
    free, count = i32([7, 6, 1, 2, 4, -1, -1, -1, -1]), i32([5])

    def keep(new, kept, counts, held=held):
        paged_keep(*pools, table, held, i32(new), i32(kept), i32(counts), free, count)

    fa.set_checked(True)
    try:
        for bad, words in (((([25, 0], [[0, 3, 24]] * 2, [4, 0])), "keeps 4 of its 25"),
                           ((([25, 0], [[0, 24, 3]] * 2, [3, 0])), "not ascending"),
                           ((([25, 0], [[0, 3, 25]] * 2, [3, 0])), "not ascending"),
                           ((([44, 0], [[0, 3, 24]] * 2, [3, 0])), "page -1 of row 0"),
                           ((([45, 0], [[0, 3, 24]] * 2, [3, 0])), r"\[20, 65\) of row 0 fall outside"),
                           ((([25, 0], [[0, 3, 24]] * 2, [3, 0], i32([20, 70]))), r"\[70, 70\) of row 1 fall outside")):
            with pytest.raises(IndexError, match="paged_keep: .*" + words):
                keep(*bad)
        assert all(torch.equal(x, y) for x, y in zip(pools, before))
        assert held.tolist() == [20, 16] and count.tolist() == [5] and table.tolist()[0] == [3, 0, 8, -1]
        keep([25, 0], [[0, 3, 24]] * 2, [3, 0])
    finally:
        fa.set_checked(False)
    # Row 0 kept nodes at 20, 23 and 44: its third page has none left.
    assert held.tolist() == [23, 16] and table.tolist() == [[3, 0, -1, -1], [5, -1, -1, -1]]
    assert count.tolist() == [6] and free.tolist()[:6] == [7, 6, 1, 2, 4, 8]
    for x, y in zip(pools, before):
        y[:, 0, 21 - 16], y[:, 0, 22 - 16] = y[:, 0, 23 - 16].clone(), y[:, 8, 44 - 32].clone()
        assert torch.equal(x, y)
