"""The verification of drafted tokens where logits are large or far apart, against the walk in 64 bits."""
import random

import pytest
import torch

from test_gpu_verify import check, drafted

pytestmark = pytest.mark.gpu
LOWEST, LARGEST = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max


def trees(seed, lens, V, logits, drawn):
    """Trees over `logits`, (total, V): guesses, or drafts, of which half are a node's largest logits."""
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    parents = [-1 if i == 0 else rng.randrange(max(0, i - 3), i) for n in lens for i in range(n)]
    total = sum(lens)
    best = [torch.nonzero(x == x.max()).flatten().tolist() for x in logits]
    likely, at = [], 0
    tokens = torch.randint(0, V, (total,), generator=g)
    for n in lens:
        for i in range(1, n):
            up = at + parents[at + i]
            if rng.random() < 0.5:
                tokens[at + i] = rng.choice(best[up])
        at += n
    probs = torch.rand(total, V, generator=g) / V
    for row, tokens_of in zip(probs, best):
        row[tokens_of] += 0.7 / len(tokens_of)
    probs /= probs.sum(1, keepdim=True)
    return tokens, parents, lens, torch.rand(total, generator=g), probs if drawn else None


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [50, 9000])  # one chunk of the vocabulary, and several
@pytest.mark.parametrize("temperature", [1e-3, 1e-8, 1e-12, 1e-16, 1e-20, 1e-30, 1e-44])
def test_small_temperatures(temperature, V, drawn):
    """The largest logits share all of it, whatever their size over the temperature."""
    longest = 0
    for seed, (spread, off) in enumerate([(4.0, 20.3), (0.5, -7.7), (300.0, 0.0)]):
        g = torch.Generator().manual_seed(seed)
        lens = [5, 1, 7, 3, 6]
        logits = (torch.randn(sum(lens), V, generator=g) * spread).round(decimals=1) + off
        for row in logits[::2]:  # ties, the chunks' borders and the ends among them
            row[[0, V // 2, V - 1, min(4095, V - 1), min(4096, V - 1)]] = row.max()
        tokens, parents, lens, numbers, probs = trees(seed, lens, V, logits, drawn)
        longest = max(longest, *check(logits, tokens, parents, lens, numbers, temperature, probs))
    assert longest > 1  # a draft is accepted somewhere


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [50, 9000])
@pytest.mark.parametrize("size", [1e5, 1e12, 1e20, -1e20, 3e38])
def test_large_logits(size, V, drawn):
    g = torch.Generator().manual_seed(3)
    lens = [5, 1, 7, 3, 6]
    logits = size * (1 - torch.randint(0, 4, (sum(lens), V), generator=g) / 16)
    tokens, parents, lens, numbers, probs = trees(4, lens, V, logits, drawn)
    check(logits, tokens, parents, lens, numbers, 1.0, probs)
    check(logits, tokens, parents, lens, numbers, 0.3, probs)


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [50, 9000])
def test_rows_of_the_lowest_and_largest_values(V, drawn):
    """A row that is masked as a whole by the type's lowest value is a flat one; one behind such a mask is as without."""
    g = torch.Generator().manual_seed(5)
    lens = [6, 4, 5]
    logits = torch.full((sum(lens), V), LOWEST)
    for fill in (LOWEST, LARGEST):
        logits[:] = fill
        tokens, parents, _, numbers, probs = trees(6, lens, V, logits, drawn)
        check(logits, tokens, parents, lens, numbers, 1.0, probs)
        check(logits, tokens, parents, lens, numbers, 1e-9, probs)
    logits[:] = LOWEST
    for row in logits:
        row[torch.randperm(V, generator=g)[:7]] = torch.randn(7, generator=g)
    tokens, parents, _, numbers, probs = trees(7, lens, V, logits, drawn)
    check(logits, tokens, parents, lens, numbers, 1.0, probs)
    logits[:, V // 3] = LARGEST
    tokens, parents, _, numbers, probs = trees(8, lens, V, logits, drawn)
    check(logits, tokens, parents, lens, numbers, 1.0, probs)


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [50, 9000])
@pytest.mark.parametrize("far", [LOWEST, -1e30, -1e5, -900.0])
def test_a_number_of_zero_takes_nothing_that_has_no_probability(far, V, drawn):
    """exp of a finite logit so far below the largest is 0 in 64 bits: such a token is neither accepted nor drawn."""
    g = torch.Generator().manual_seed(9)
    lens = [5, 1, 4, 6]
    logits = torch.randn(sum(lens), V, generator=g)
    logits[:, :V // 2] = far
    logits[1::3, :V - 3] = far
    tokens, parents, _, _, probs = trees(10, lens, V, logits, drawn)
    tokens[2::2] %= V // 2
    for u in (0.0, 2.0 ** -24):
        check(logits, tokens, parents, lens, torch.full((sum(lens),), u), 1.0, probs, least=1.0 if u == 0 else 0.5)


@pytest.mark.parametrize("V,lens", [(400, [130, 200, 90, 300]), (5000, [100, 70])])
@pytest.mark.parametrize("seed", range(3))
def test_wide_stars_of_drawn_drafts(seed, V, lens):
    """Up to hundreds of children of one node, most of them refused: a remainder's sum after each."""
    check(*drafted(seed, lens, V, 1.0, drawn=True, tree="star", off=3.0, spread=3.0), least=1.0)
