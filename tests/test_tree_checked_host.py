"""What checked mode says of the nodes that a paged cache is to keep, on the CPU."""
import pytest
import torch

from modelcore_amd.kernels import paged


@pytest.fixture(autouse=True)
def no_capture(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def check(table, held, new, kept, counts, page=16, n_pages=9):
    paged._check_keep(i32(table), i32(held), i32(new), i32(kept), i32(counts), page, n_pages)


GOOD = dict(table=[[3, 0, 8, -1], [5, -1, -1, -1], [-1, -1, -1, -1]], held=[20, 16, 0], new=[25, 0, 0],
            kept=[[0, 3, 24], [-1, -1, -1], [-1, -1, -1]], counts=[3, 0, 0])


def test_rows_that_are_in_order():
    check(**GOOD)
    check(**{**GOOD, "counts": [0, 0, 0], "kept": [[7, 7, 7]] * 3})  # past the counts nothing is looked at
    check(**{**GOOD, "held": [39, 15, 0], "new": [1, 1, 0], "counts": [1, 1, 0], "kept": [[0] * 3] * 3})
    check([[0, 1]], [32], [0], [[]], [0])  # a full line, and no nodes
    check([[0, 1]], [30], [2], [[0, 1]], [2])


@pytest.mark.parametrize("change,words", [
    (dict(counts=[4, 0, 0]), "row 0 keeps 4 of its 25 nodes"),
    (dict(counts=[3, 1, 0]), "row 1 keeps 1 of its 0 nodes"),
    (dict(counts=[3, 0, -1]), "row 2 keeps -1 of its 0 nodes"),
    (dict(new=[2, 0, 0]), "row 0 keeps 3 of its 2 nodes"),
    (dict(new=[25, -2, 0], counts=[3, 1, 0]), "row 1 keeps 1 of its -2 nodes"),
    (dict(kept=[[0, 3, 25]] * 3), "not ascending nodes"),
    (dict(kept=[[0, 3, 3]] * 3), "not ascending nodes"),
    (dict(kept=[[5, 3, 8]] * 3), "not ascending nodes"),
    (dict(kept=[[0, 0, 8]] * 3), "not ascending nodes"),
    (dict(kept=[[-1, 3, 8]] * 3), "not ascending nodes"),
    (dict(held=[-1, 16, 0]), r"positions \[-1, 24\) of row 0 fall outside the 64"),
    (dict(held=[40, 16, 0]), r"positions \[40, 65\) of row 0 fall outside the 64"),
    # Rows without nodes: past the line's end, at a page's end and within one.
    (dict(held=[20, 80, 0]), r"positions \[80, 80\) of row 1 fall outside the 64"),
    (dict(held=[20, 70, 0]), r"positions \[70, 70\) of row 1 fall outside the 64"),
    (dict(held=[20, 65, 0], new=[25, -3, 0]), r"positions \[65, 65\) of row 1 fall outside the 64"),
    (dict(table=[[3, 9, 8, -1], [5, -1, -1, -1], [-1] * 4]), "page 9 of row 0 is not one of the pool's 9"),
    (dict(table=[[3, 0, -1, -1], [5, -1, -1, -1], [-1] * 4]), "page -1 of row 0"),
    (dict(held=[20, 17, 0]), "page -1 of row 1"),
])
def test_rows_that_are_not(change, words):
    with pytest.raises(IndexError, match=words):
        check(**{**GOOD, **change})
