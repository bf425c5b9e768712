"""The plan of drafted trees and the acceptance of their nodes in a paged cache, on the GPU against plain
Python."""
import random

import pytest
import torch

import _tree
from modelcore_amd.kernels.paged import paged_keep, paged_reserve, paged_tree

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def check_plan(parents, lens, held, longest, pad=0):
    words = max(1, -(-longest // 64))
    got = paged_tree(i32(parents + [-1] * pad), i32(offsets(lens)), i32(held), max_seqlen=longest)
    pos, masks = _tree.plan(parents, lens, held, words)
    assert got.positions.tolist() == pos + [-1] * pad
    assert got.masks.shape == (len(parents) + pad, words)
    assert got.masks.tolist() == masks + [[0] * words] * pad


@pytest.mark.parametrize("lens", [[1], [0, 3, 0], [64], [65, 1, 63], [7] * 40, [200, 129, 0, 128], [1024, 5]])
@pytest.mark.parametrize("kind", ["random", "chain", "star", "forest"])
def test_plan(lens, kind):
    rng = random.Random(len(lens) * 7 + sum(lens))
    parents = []
    for n in lens:
        parents += {"chain": [i - 1 for i in range(n)], "star": [-1 if i == 0 else 0 for i in range(n)],
                    "random": _tree.random_parents(rng, n), "forest": _tree.random_parents(rng, n, 0.3)}[kind]
    check_plan(parents, lens, [rng.randrange(5000) for _ in lens], max(lens), pad=3)


def test_plan_of_chains_that_do_not_go_down():
    """A parent that is the node itself, after it, or below -1: the node and all that climb through it."""
    check_plan([-1, 0, 2, 2, 5, 1, -2, 6, 1, 100], [10], [9], 10)
    check_plan([0, 0, 1], [3], [0], 3)
    check_plan([-1, 0, -1, 0, 1], [2, 3], [-4, 2 ** 31 - 2], 3)


@pytest.mark.parametrize("seed", range(4))
def test_wide_plans_of_chains_that_do_not_go_down(seed):
    """The same among hundreds of nodes, near and far from those that climb through them."""
    rng = random.Random(seed)
    lens, parents = [300, 1, 1000, 130], []
    for n in lens:
        row = [i - 1 if rng.random() < 0.8 else rng.randrange(max(0, i - 90), i) if i else -1 for i in range(n)]
        for _ in range(n // 100):
            i = rng.randrange(n)
            row[i] = rng.choice([i, i + 1, n, -2, 2 ** 31 - 1, -2 ** 31])
        parents += row
    check_plan(parents, lens, [rng.randrange(5000) for _ in lens], 1000, pad=70)


def test_plan_positions_past_31_bits_are_none():
    got = paged_tree(i32([-1, 0, 1]), i32([0, 3]), i32([2 ** 31 - 2]), max_seqlen=3)
    assert got.positions.tolist() == [2 ** 31 - 2, 2 ** 31 - 1, -1]
    assert got.masks.tolist() == [[1], [3], [0]]


def test_plan_of_more_nodes_than_words():
    """Nodes past max_seqlen's words have no place."""
    n = 70
    got = paged_tree(i32([i - 1 for i in range(n)]), i32([0, n]), i32([3]), max_seqlen=64)
    assert got.positions.tolist() == list(range(3, 67)) + [-1] * 6
    assert got.masks[64:].tolist() == [[0]] * 6
    assert got.masks[63].tolist() == [-1]


def test_plan_of_nothing():
    assert paged_tree(i32([]), i32([0, 0]), i32([3]), max_seqlen=0).masks.shape == (0, 1)
    assert paged_tree(i32([]), i32([0]), i32([]), max_seqlen=5).positions.numel() == 0


# -----------------------------------------------------------------------------------------------
# Keeping
# -----------------------------------------------------------------------------------------------
def check_keep(held, new, kept, counts, page=16, slots=2, heads=2, dim=8, dtype=torch.bfloat16, spare=5, lost=(),
               in_free=(), wide=0, view=False, width=None, seed=0):
    """One call against the lists' form; `lost`: (row, entry) of the table that are none of the pool."""
    rng = random.Random(seed)
    pages = [max(-(-(max(s, 0) + max(t, 0)) // page), 0) for s, t in zip(held, new)]
    n_pages = sum(pages) + spare
    order = list(range(n_pages))
    rng.shuffle(order)
    width = width or max(pages + [0]) + 1
    table = [[order.pop() for _ in range(min(p, width))] + [-1] * (width - min(p, width)) for p in pages]
    for b, e, x in lost:
        table[b][e] = x
    free = order + [-7] * (n_pages - len(order))
    count = [len(order)]
    shape = (slots, n_pages, page, heads, dim)
    if view:  # pools that are every second page and slot of larger ones
        k, v = (torch.randn(2 * slots, 2 * n_pages, page, heads, dim, device=DEV).to(dtype)[::2, ::2]
                for _ in range(2))
    else:
        k, v = (torch.randn(shape, device=DEV).to(dtype) for _ in range(2))
    want_k, want_v = k.cpu().clone(), v.cpu().clone()
    places = [{(p, o): (p, o) for p in range(n_pages) for o in range(page)}]
    t2, h2, f2, c2 = [list(x) for x in table], list(held), list(free), list(count)
    _tree.keep(places, t2, h2, new, kept, counts, f2, c2, page)
    for (p, o), (ps, os_) in places[0].items():
        if (p, o) != (ps, os_):
            want_k[:, p, o], want_v[:, p, o] = k[:, ps, os_].cpu(), v[:, ps, os_].cpu()
    tg, hg, fg, cg = i32(table), i32(held), i32(free), i32(count)
    if wide:
        big = torch.full((len(held), width + wide), 99, dtype=torch.int32, device=DEV)
        big[:, :width] = tg
        tg = big[:, :width]
    paged_keep(k, v, tg, hg, i32(new), torch.tensor(kept, dtype=torch.int32, device=DEV).reshape(len(held), -1),
               i32(counts), fg, cg)
    bits = {torch.bfloat16: torch.int16, torch.float32: torch.int32}[dtype]
    assert torch.equal(k.cpu().contiguous().view(bits), want_k.view(bits))
    assert torch.equal(v.cpu().contiguous().view(bits), want_v.view(bits))
    assert tg.tolist() == t2 and hg.tolist() == h2
    assert cg.tolist() == c2 and fg.tolist()[:c2[0]] == f2[:c2[0]]
    if wide:
        assert bool((big[:, width:] == 99).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("page", [16, 64])
def test_keep(page, dtype):
    check_keep([0, 15, 16, 200, 1], [5, 9, 33, 64, 1],
               [[0, 2, 4, -1], [0, 1, 2, 3], [0, 8, 20, 32], [3, 4, 5, 60], [0, -1, -1, -1]],
               [3, 4, 4, 4, 1], page, dtype=dtype)


@pytest.mark.parametrize("seed", range(6))
def test_keep_at_random(seed):
    """Random trees and paths among them, sources that are other nodes' places among them."""
    rng = random.Random(seed)
    rows = rng.choice([1, 3, 40])
    new = [rng.choice([0, 1, rng.randrange(1, 70)]) for _ in range(rows)]
    kept, counts = [], []
    for n in new:
        path = sorted(rng.sample(range(n), rng.randrange(n + 1)))
        counts.append(len(path))
        kept.append(path + [-1] * (70 - len(path)))
    heads, dim = rng.choice([(1, 8), (3, 40), (4, 128), (12, 64)])
    check_keep([rng.randrange(100) for _ in range(rows)], new, kept, counts, rng.choice([16, 32, 128]),
               rng.choice([1, 3]), heads, dim, rng.choice([torch.bfloat16, torch.float32]),
               wide=rng.choice([0, 3]), view=rng.random() < 0.5, seed=seed)


def test_keep_gives_back_many_pages():
    """More rows than the tables' workgroup has threads, each with pages to give."""
    rng = random.Random(3)
    rows = 1300
    new = [rng.randrange(1, 60) for _ in range(rows)]
    kept = [[0] for _ in range(rows)]
    check_keep([rng.randrange(40) for _ in range(rows)], new, kept, [rng.randrange(2) for _ in range(rows)], heads=1,
               slots=1)


def test_keep_passes_over_what_it_should_not_follow():
    """Counts past the nodes or the list, nodes out of order or outside the row, rows that do not fit, entries that
    are no page."""
    check_keep([3, 3, 3, 3], [6, 6, 6, 6], [[0, 9, 2], [0, 0, 1], [5, -3, 4], [0, 3, 5]], [9, 3, 3, -2])
    check_keep([3, -1, 100], [6, 4, 40], [[0, 2], [0, 1], [0, 1]], [2, 2, 2], width=8)
    # A row that was refused: the pages of its nodes are not there.
    check_keep([14, 20], [30, 30], [[0, 5, 9], [0, 5, 9]], [3, 3], lost=[(0, 1, -1), (0, 2, -1)])
    # Pages that were lost in the middle.
    check_keep([14, 20], [60, 60], [[0, 5, 40], [0, 30, 59]], [3, 3], lost=[(0, 2, 5000), (1, 2, -1)])


def test_keep_one_slot_and_no_rows():
    table, held, free, count = i32([[1, -1]]), i32([4]), i32([0, 2, -1]), i32([2])
    k = torch.arange(3 * 16, device=DEV, dtype=torch.float32).view(3, 16, 1, 1).expand(3, 16, 2, 4).contiguous()
    v = -k
    paged_keep(k, v, table, held, i32([5]), i32([[0, 3]]), i32([2]), free, count)
    assert k[1, :, 0, 0].tolist() == [16, 17, 18, 19, 20, 23, *range(22, 32)]
    assert v[1, 5, 1, 3] == -23
    assert held.tolist() == [6]
    paged_keep(k, v, table[:0], held[:0], i32([]), i32([]).view(0, 2), i32([]), free, count)


def test_keep_refuses_what_it_cannot_follow():
    pool = torch.zeros(2, 6, 16, 2, 8, dtype=torch.bfloat16, device=DEV)
    good = dict(k_pages=pool, v_pages=pool.clone(), block_table=i32([[1, -1]]), cache_seqlens=i32([4]), new_lens=i32([3]),
                kept=i32([[0, 2]]), counts=i32([2]), free_pages=i32([0, 2, 3, 4, 5, -1]), free_count=i32([5]))
    heads_first = pool.transpose(2, 3).contiguous().transpose(2, 3)
    apart = torch.zeros(2, 12, 16, 2, 8, dtype=torch.bfloat16, device=DEV)[:, ::2]
    for kw, error, words in (
            (dict(k_pages=heads_first), ValueError, "each page of k_pages must be contiguous"),
            (dict(v_pages=pool[..., ::2].repeat_interleave(1, -1)), ValueError, "must both be"),
            (dict(k_pages=pool[..., ::2], v_pages=pool[..., ::2]), ValueError, "contiguous"),
            (dict(v_pages=apart), ValueError, "same strides"), (dict(v_pages=pool.float()), TypeError, "v_pages is"),
            (dict(k_pages=pool[:, :5], v_pages=pool[:, :5]), ValueError, "must both be"),
            (dict(k_pages=pool[0, 0], v_pages=pool[0, 0]), ValueError, "must both be"),
            (dict(k_pages=pool.half(), v_pages=pool.half()), TypeError, "bfloat16 or float32"),
            (dict(counts=i32([2, 1])), ValueError, "counts must be"), (dict(new_lens=i32([3]).long()), ValueError, "new_lens"),
            (dict(kept=i32([0, 2])), ValueError, "kept must be"), (dict(kept=i32([[0], [1]])), ValueError, "kept must be"),
            (dict(free_count=i32([5, 5])), ValueError, "free_count"), (dict(block_table=i32([1, -1])), ValueError, "block_table"),
            (dict(kept=torch.zeros(1, 2, dtype=torch.int32)), ValueError, "kept is on cpu")):
        with pytest.raises(error, match=words):
            paged_keep(**{**good, **kw})
    assert good["cache_seqlens"].tolist() == [4] and good["free_count"].tolist() == [5]
    paged_keep(**good)
    assert good["cache_seqlens"].tolist() == [6]


def test_reserve_tree_and_keep_in_a_captured_graph():
    """The bookkeeping of a step of trees replayed, lengths moving on from replay to replay, against the same
    steps without a graph."""
    rows, n, page, n_pages = 3, 21, 16, 40
    parents = [-1 if i == 0 else (i - 1) // 4 for i in range(n)]
    kept = i32([[0, 2, 9], [0, 4, 18], [0, 1, 5]])
    counts, new = i32([3, 1, 2]), i32([n] * rows)

    def state():
        g = torch.Generator(device=DEV).manual_seed(5)
        return dict(table=torch.full((rows, 8), -1, dtype=torch.int32, device=DEV), held=i32([0, 0, 0]),
                    free=torch.arange(n_pages, dtype=torch.int32, device=DEV), count=i32([n_pages]),
                    k=torch.randn(2, n_pages, page, 2, 16, generator=g, device=DEV),
                    v=torch.randn(2, n_pages, page, 2, 16, generator=g, device=DEV))

    def step(s):
        plan = paged_reserve(s["table"], s["held"], new, s["free"], s["count"], total=rows * n, page_size=page)
        tree = paged_tree(i32_parents, plan.cu_seqlens, s["held"], max_seqlen=n)
        paged_keep(s["k"], s["v"], s["table"], s["held"], new, kept, counts, s["free"], s["count"])
        return plan, tree

    i32_parents = i32(parents * rows)
    a, b = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a)
    torch.cuda.current_stream().wait_stream(side)
    step(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan, tree = step(a)
    for _ in range(6):
        graph.replay()
        want_plan, want_tree = step(b)
        for x, y in zip((*plan, *tree, *a.values()), (*want_plan, *want_tree, *b.values())):
            assert torch.equal(x, y)
    assert b["held"].tolist() == [21, 7, 14]
