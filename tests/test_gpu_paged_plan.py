"""Page plans on the GPU whose inputs are not what a cache that only ever moves planned rows would hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("rows", [3, 1500])
def test_a_row_longer_than_its_pages_gives_back_those_it_has(rows):
    """A row that was refused and moved on all the same holds fewer pages than its length says: only pages
    go onto the stack, in order, and the plan after it deals each of them once."""
    from modelcore_amd.kernels.paged import paged_release, paged_reserve
    width, n_pages = 4, 4 * rows
    table = [[-1] * width for _ in range(rows)]
    lens, ids = [0] * rows, iter(range(n_pages))
    for b in range(rows):  # every other row has one page less than its length needs
        lens[b] = 16 * (1 + b % 3)
        for i in range(1 + b % 3 - (b % 2)):
            table[b][i] = next(ids)
    table[0][0] = n_pages + 5  # no page of the pool either
    held = [p for line in table for p in line if 0 <= p < n_pages]
    free = sorted(set(range(n_pages)) - set(held))
    count = len(free)
    dt, dl = i32(table), i32(lens)
    df, dc = i32(free + [-7] * (n_pages - count)), i32([count])
    done = list(range(rows))[::-1]
    paged_release(dt, dl, i32(done), df, dc, page_size=16)
    back = [p for b in done for p in table[b] if 0 <= p < n_pages]
    assert dc.tolist() == [count + len(back)]
    assert df.tolist()[:count + len(back)] == free + back
    assert (dt == -1).all() and (dl == 0).all()
    new = [40 if b % 2 else 3 for b in range(rows)]
    plan = paged_reserve(dt, dl, i32(new), df, dc, total=sum(new), page_size=16)
    slots = plan.slots.tolist()
    given = [s for s in slots if s >= 0]
    assert len(set(given)) == len(given) and all(s < 16 * n_pages for s in given)
    assert (plan.refused.item() == 0) == (len(given) == len(slots))


@pytest.mark.parametrize("tokens", [20, 3000])  # in one launch, and in two
@pytest.mark.parametrize("bad", [-1, 7000, 2 ** 31 - 1])
def test_numbers_on_the_stack_that_are_no_pages(tokens, bad):
    """Their tokens get no slot, the table -1, and `refused` says that something was not given."""
    from modelcore_amd.kernels.paged import paged_reserve
    rows, pages = 3, 600
    free = list(range(pages))
    need = -(-tokens // 16)
    free[pages - 1 - need] = bad  # the first page of the second row
    table = torch.full((rows, need + 2), -1, dtype=torch.int32, device=DEV)
    count = i32([pages])
    plan = paged_reserve(table, i32([0] * rows), i32([tokens] * rows), i32(free), count,
                         total=rows * tokens, page_size=16)
    want = []
    for b in range(rows):
        for t in range(tokens):
            page = free[pages - 1 - b * need - t // 16]
            want.append(page * 16 + t % 16 if 0 <= page < pages else -1)
    assert plan.slots.tolist() == want
    assert plan.refused.tolist() == [1] and count.tolist() == [pages - rows * need]
    assert table[1].tolist()[:2] == [-1, free[pages - 2 - need] if need > 1 else -1]


def test_checked_mode_finds_pages_that_would_be_given_twice():
    """Rows whose lines share pages, pages that are free already, numbers that are no pages: refused before
    anything is launched, where checked mode is on."""
    from modelcore_amd.kernels import flash_attn as fa
    from modelcore_amd.kernels.paged import paged_release
    free, count = i32([9, 8, 7, 6, 5] + [-1] * 5), i32([5])
    lens = [20, 16, 40, 0]
    lines = [[0, 1, -1], [0, -1, -1], [2, 3, 4], [2, -1, -1]]

    def release(rows, lines):
        table, n = i32(lines), i32(lens)
        paged_release(table, n, i32(rows), free, count, page_size=16)
        return table, n
    fa.set_checked(True)
    try:
        for rows in ([0], [2, 1], [0, 1]):
            with pytest.raises(ValueError, match="page 0 of row . is also held by rows"):
                release(rows, lines)
        with pytest.raises(ValueError, match="page 6 of row 1 is also free"):
            release([1], [lines[0], [6, -1, -1]] + lines[2:])
        with pytest.raises(IndexError, match="page 10 of row 1 is not one of the pool"):
            release([1], [lines[0], [10, -1, -1]] + lines[2:])
        assert count.tolist() == [5]
        table, n = release([2, 3, 2, 77], lines)  # what row 3 names, it does not hold
        assert count.tolist() == [8] and free.tolist()[5:8] == [2, 3, 4]
        assert n.tolist() == [20, 16, 0, 0] and table.tolist()[2] == [-1] * 3
    finally:
        fa.set_checked(False)


@pytest.mark.parametrize("rows", [5, 1100])
def test_entries_without_a_page_beside_a_full_stack(rows):
    """The lines say more pages than the stack has room for: those there are fill it, in order."""
    from modelcore_amd.kernels.paged import paged_release
    n_pages = 2 * rows
    g = torch.Generator().manual_seed(rows)
    ids = torch.randperm(n_pages, generator=g).tolist()
    table = [[-1, ids[2 * b], -1, n_pages, ids[2 * b + 1]] for b in range(rows - 1)] + [ids[-2:] + [-1] * 3]
    dt, dl = i32(table), i32([80] * (rows - 1) + [32])
    df, dc = i32([-7] * n_pages), i32([0])
    paged_release(dt, dl, i32(list(range(rows))), df, dc, page_size=16)
    assert df.tolist() == ids and dc.tolist() == [n_pages]
    assert (dt == -1).all() and (dl == 0).all()
