"""The verification of drafted tokens on the GPU, against the walk in plain Python and 64 bits."""
import math
import random

import pytest
import torch

import _tree
from modelcore_amd.sampling import PhiloxSampler, verify_drafts

pytestmark = pytest.mark.gpu
DEV = "cuda"
# The kernel's weights are within 2^-30 of exact ones, its 64-bit sums far nearer: a walk whose numbers stay
# further than this from every border has one answer.
NEAR = 1e-8


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def check(logits, tokens, parents, lens, numbers, temperature, probs=None, longest=None, least=0.9, pad=0):
    """One call on rows of lens nodes; tensors on the CPU, (total, ..). At least a share `least` of the rows has to be
    far from every border."""
    longest = longest or max([1] + lens)
    cu = offsets(lens)
    got = verify_drafts(logits.to(DEV), tokens.to(DEV), i32(parents + [-1] * pad), i32(cu), numbers.to(DEV),
                        temperature=temperature, draft_probs=None if probs is None else probs.to(DEV), max_seqlen=longest)
    kept, counts, out = (t.cpu() for t in got)
    assert kept.shape == out.shape == (len(lens), longest)
    assert kept.dtype == counts.dtype == torch.int32 and out.dtype == torch.int64
    clear = 0
    rows = []
    for b, n in enumerate(lens):
        n = min(n, longest)
        at = slice(cu[b], cu[b] + n)
        t = float(torch.tensor(temperature, dtype=torch.float32))
        want_kept, want, near = _tree.verify(logits[at].float().tolist(), tokens[at].tolist(), parents[at], numbers[at].tolist(),
                                             t, None if probs is None else probs[at].tolist())
        rows.append(len(want))
        if near < NEAR:
            continue
        clear += 1
        c = len(want)
        assert counts[b] == c, (b, counts[b], want_kept)
        assert kept[b].tolist() == want_kept + [-1] * (longest - c), b
        assert out[b].tolist() == want + [-1] * (longest - c), b
    assert clear >= least * len(lens)
    return rows


def drafted(seed, lens, V, temperature=1.0, drawn=False, spread=2.0, off=0.5, tree="random"):
    """Logits, drafts by a model that is a little off, and numbers."""
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    total = sum(lens)
    parents = []
    for n in lens:
        parents += {"random": [-1 if i == 0 else rng.randrange(max(0, i - 5), i) for i in range(n)],
                    "chain": [i - 1 for i in range(n)], "star": [-1 if i == 0 else 0 for i in range(n)]}[tree]
    logits = torch.randn(total, V, generator=g) * spread
    near = logits + torch.randn(total, V, generator=g) * off
    probs = torch.softmax(near / (temperature or 1.0), -1)
    tokens = torch.randint(0, V, (total,), generator=g)
    cu = offsets(lens)
    for b, n in enumerate(lens):
        tried = {}
        for i in range(1, n):
            up = cu[b] + parents[cu[b] + i]
            if drawn:
                tokens[cu[b] + i] = torch.multinomial(probs[up], 1, generator=g)[0]
            else:
                k = tried[up] = tried.get(up, -1) + 1
                tokens[cu[b] + i] = near[up].topk(min(k + 1, V)).indices[-1]
    numbers = torch.rand(total, generator=g)
    return logits, tokens, parents, lens, numbers, temperature, probs if drawn else None


@pytest.mark.parametrize("V", [1, 2, 7, 63, 64, 65, 100, 1000, 1025, 4099])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
def test_guesses(V, temperature):
    rows = check(*drafted(V, [5, 1, 9, 0, 3], V, temperature))
    assert rows[3] == 0 and min(rows[:3]) >= 1


@pytest.mark.parametrize("V", [1, 2, 7, 63, 64, 65, 100, 1000, 1025, 4099])
@pytest.mark.parametrize("tree", ["random", "chain", "star"])
def test_drafts_of_a_model(V, tree):
    check(*drafted(V + 1, [5, 1, 9, 0, 12, 3], V, 0.8, drawn=True, tree=tree, off=1.0))


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("spread", [0.0, 0.2, 4.0, 30.0])
def test_flat_and_peaked(spread, drawn):
    """A whole vocabulary as likely, and one token that has nearly all."""
    rows = check(*drafted(17, [4] * 24, 5000, 1.0, drawn=drawn, spread=spread, off=0.3), least=0.8)
    assert max(rows) > 1 or not drawn and spread < 4  # a guess of a flat vocabulary has 1 in 5000


def test_a_whole_vocabulary():
    for drawn in (False, True):
        check(*drafted(3, [3, 4], 32768, 1.0, drawn=drawn))
    check(*drafted(4, [2, 3], 128256, 0.6))


def test_many_rows_and_wide_trees():
    check(*drafted(5, [random.Random(5).randrange(6) for _ in range(300)], 97, 0.9))
    check(*drafted(6, [1024, 200], 50, 1.0, tree="star", off=3.0))
    check(*drafted(7, [130], 40, 1.0, drawn=True, tree="star", off=1.5, spread=1.0), least=0.0)


@pytest.mark.parametrize("drawn", [False, True])
def test_numbers_at_their_ends(drawn):
    """0 accepts what has any probability and draws the first token that has; the largest below 1 the last."""
    args = list(drafted(8, [6] * 8, 300, 1.0, drawn=drawn))
    args[0][:, :40] = -math.inf
    args[0][:, 280:] = -math.inf
    if drawn:
        args[6][:, :40] = 0
    for u in (0.0, 1 - 2.0 ** -24):
        args[4] = torch.full_like(args[4], u)
        check(*args, least=0.0 if u else 1.0)
        kept, counts, out = verify_drafts(args[0].to(DEV), args[1].to(DEV), i32(args[2]), i32(offsets(args[3])), args[4].to(DEV),
                                          draft_probs=None if not drawn else args[6].to(DEV), max_seqlen=6)
        last = out.gather(1, (counts - 1)[:, None].long())
        assert bool(((last >= 40) & (last < 280)).all())


def test_the_same_guess_twice():
    """A token that was refused has no probability left when it is tried again."""
    logits = torch.log(torch.tensor([[0.5, 0.3, 0.2]])).repeat(4, 1)
    tokens, parents = torch.tensor([0, 1, 1, 2]), [-1, 0, 0, 0]
    for u, want in (([0.1, 0.9, 0.0, 0.5], [0]), ([0.1, 0.9, 0.0, 0.2], [2, 0]), ([0.9, 0.9, 0.0, 0.5], [0]),
                    ([0.1, 0.2, 0.0, 0.2], [1, 0])):
        numbers = torch.tensor(u)
        check(logits, tokens, parents, [4], numbers, 1.0, least=1.0)
        got = verify_drafts(logits.to(DEV), tokens.to(DEV), i32(parents), i32([0, 4]), numbers.to(DEV), max_seqlen=4)
        assert got.tokens[0, :len(want)].tolist() == want


def test_odd_logits():
    """NaN and -inf have no probability, +inf all of it; a node with none at all ends its row with token 0."""
    inf, nan = math.inf, math.nan
    logits = torch.tensor([[0.0, nan, 1.0, -inf, 2.0], [inf, 0.0, nan, inf, 5.0], [-inf, nan, -inf, -inf, nan],
                           [nan, 1.0, 1.0, 0.0, -inf]])
    for t in (0.0, 1.0):
        for u in (0.05, 0.4, 0.8):
            for x in range(5):
                # Four rows of a root and a child x.
                check(logits.repeat_interleave(2, 0), torch.tensor([0, x] * 4), [-1, 0] * 4, [2] * 4,
                      torch.tensor([u, 0.45] * 4), t, least=1.0)


def test_tokens_outside_the_vocabulary_are_passed_over():
    for x in (-1, 9, 2 ** 40):
        for probs in (None, torch.full((3, 9), 1 / 9)):
            check(torch.zeros(3, 9), torch.tensor([x, x, 4]), [-1, 0, 0], [3], torch.tensor([0.35, 0.0, 0.05]), 1.0, probs, least=1.0)


def test_layouts():
    """Rows behind the last, a max_seqlen past and short of the rows, logits that are columns of wider ones,
    half-precision ones."""
    logits, tokens, parents, lens, numbers, t, probs = drafted(12, [4, 6, 2], 200, 0.9, drawn=True)
    pad = torch.zeros(3, 200)
    check(torch.cat([logits, pad]), torch.cat([tokens, tokens[:3]]), parents, lens, torch.cat([numbers, numbers[:3]]), t,
          torch.cat([probs, pad]), longest=9, pad=3)
    check(logits, tokens, parents, lens, numbers, t, probs, longest=3)
    wide = torch.cat([logits, logits.flip(0)], 1).to(DEV)
    args = (tokens.to(DEV), i32(parents), i32(offsets(lens)), numbers.to(DEV))
    want = verify_drafts(logits.to(DEV), *args, temperature=t, draft_probs=probs.to(DEV), max_seqlen=6)
    wide_probs = torch.cat([probs, probs], 1).to(DEV)
    for a, p in ((wide[:, :200], wide_probs[:, :200]), (logits.t().contiguous().to(DEV).t(), probs.t().contiguous().to(DEV).t())):
        for x, y in zip(verify_drafts(a, *args, temperature=t, draft_probs=p, max_seqlen=6), want):
            assert torch.equal(x, y)
    half = logits.to(torch.bfloat16)
    check(half, tokens, parents, lens, numbers, t, probs)
    got = verify_drafts(logits[:0].to(DEV), tokens[:0].to(DEV), i32([]), i32([0, 0]), numbers[:0].to(DEV), max_seqlen=2)
    assert got.counts.tolist() == [0] and got.tokens.tolist() == [[-1, -1]]
    assert verify_drafts(logits[:0].to(DEV), tokens[:0].to(DEV), i32([]), i32([0]), numbers[:0].to(DEV), max_seqlen=2).counts.numel() == 0


def test_greedy_is_the_sampler_at_temperature_zero():
    logits = torch.randn(50, 1000, generator=torch.Generator().manual_seed(1)).round(decimals=1).to(DEV)
    want = PhiloxSampler(50, DEV)(logits, temperature=0.0)
    got = verify_drafts(logits, torch.zeros(50, dtype=torch.int64, device=DEV), i32([-1] * 50), i32(list(range(51))),
                        torch.zeros(50, device=DEV), temperature=0.0, max_seqlen=1)
    assert torch.equal(got.tokens, want)


@pytest.mark.parametrize("drawn", [False, True])
def test_emitted_tokens_have_the_targets_distribution(drawn):
    """20000 rows whose first token is drafted twice: the first token after the root is a draw from the target's
    softmax whatever the drafts. A token's count has a standard deviation of at most sqrt(n p); five of them,
    for each of eight tokens, is passed by chance once in 200000 runs, and the seed is fixed."""
    g = torch.Generator().manual_seed(9)
    n, V = 20000, 8
    logits = torch.randn(V, generator=g)
    q = torch.softmax(torch.randn(V, generator=g), -1)
    p = torch.softmax(logits, -1)
    drafts = torch.multinomial(q, 2 * n, replacement=True, generator=g).view(n, 2) if drawn \
        else torch.tensor([[2, 5]]).repeat(n, 1)
    tokens = torch.cat([torch.zeros(n, 1, dtype=torch.int64), drafts], 1).reshape(-1)
    got = verify_drafts(logits.repeat(3 * n, 1).to(DEV), tokens.to(DEV), i32([-1, 0, 0] * n), i32([3 * b for b in range(n + 1)]),
                        torch.rand(3 * n, generator=g).to(DEV), draft_probs=q.repeat(3 * n, 1).to(DEV) if drawn else None,
                        max_seqlen=3)
    seen = torch.bincount(got.tokens[:, 0].cpu(), minlength=V).double()
    assert bool(((seen - n * p).abs() <= 5 * (n * p).sqrt()).all()), (seen / n, p)
    accepted = float((got.counts == 2).sum())
    if drawn:  # at least what the first draft alone is accepted with, sum min(p, q)
        assert accepted >= n * float(torch.minimum(p, q).sum()) - 5 * n ** 0.5
    else:  # as often as the target draws one of the two guesses
        assert abs(accepted - n * float(p[2] + p[5])) <= 5 * (n * float(p[2] + p[5])) ** 0.5


def test_captured_and_replayed():
    """Replays on other logits and numbers, two graphs that were captured one after the other among them."""
    a, b = (drafted(s, [5, 3, 8], 3000, 0.8, drawn=True) for s in (20, 21))
    held = [[t.clone().to(DEV) for t in (x[0], x[1], x[4], x[6])] for x in (a, b)]
    fixed = [(i32(x[2]), i32(offsets(x[3]))) for x in (a, b)]

    def body(i):
        logits, tokens, numbers, probs = held[i]
        return verify_drafts(logits, tokens, fixed[i][0], fixed[i][1], numbers, temperature=0.8, draft_probs=probs, max_seqlen=8)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body(0), body(1)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(body(i))
        graphs.append(graph)
    for k in range(4):
        for i in range(2):
            x = drafted(30 + 2 * k + i, [5, 3, 8], 3000, 0.8, drawn=True)
            for t, y in zip(held[i], (x[0], x[1], x[4], x[6])):
                t.copy_(y)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i in range(2):
            for x, y in zip(outs[i], body(i)):
                assert torch.equal(x, y)


@pytest.mark.parametrize("seed", range(10))
def test_at_random(seed):
    rng = random.Random(seed)
    lens = [rng.randrange(12) for _ in range(rng.randrange(1, 9))]
    drawn = rng.random() < 0.5
    check(*drafted(seed + 50, lens, rng.choice([rng.randrange(1, 300), rng.randrange(300, 9000)]),
                   rng.choice([0.0, 1.0, 0.37, 1.6]), drawn, rng.choice([0.5, 2.0, 5.0]), rng.choice([0.1, 1.0]),
                   rng.choice(["random", "chain", "star"])), least=0.8)


def test_vocabularies_of_more_chunks_than_are_kept():
    """Past 64 chunks of 4096 logits a lane has several of them."""
    for drawn in (False, True):
        check(*drafted(40, [2, 2, 3], 300001, 1.0, drawn=drawn, off=2.0), least=0.3)
