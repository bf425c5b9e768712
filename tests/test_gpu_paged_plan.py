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
