"""The paged attention's rules replayed on the host over calls at random, and the 64-bit form's bounds against
what they are to find."""
import random

import pytest
import torch

import _paged
from _paged_blocks import Rules, attend, close, rounds_weights

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("cus", [304, 256, 32])
def test_every_block_is_done_once(cus):
    rng = random.Random(cus)
    halved = 0
    for _ in range(6000):
        dtype, D = rng.choice([(BF, 128), (BF, 64), (BF, 256), (F32, 64), (F32, 128), (F32, 256), (BF, 24)])
        G, H_kv = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 33, 64]), rng.choice([1, 2, 3, 4, 8, 16, 32])
        n, longest, deep = rng.choice([1, 3, 7, 20, 64, 65, 130, 256, 257]), rng.choice([3, 40, 300]), \
            rng.choice([10, 700, 5000])
        rows = [(rng.choice([0, 1, 2, rng.randint(1, longest)]), rng.randint(0, deep)) for _ in range(n)]
        rows[0] = (longest, rng.choice([deep, -1, 2 ** 31 - 1, 6000]))
        halved += Rules(rows, G * H_kv, H_kv, D, dtype, 5400, rng.choice([-1, -1, -1, 500]), cus).check() > 0
    assert halved > 100


def made(T, G, D, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(T, 2 * G, D, generator=g).to(BF)
    k, v = (torch.randn(n + T, 2, D, generator=g).to(BF) for _ in range(2))
    return q, k, v


@pytest.mark.parametrize("window", [-1, 0, 30])
def test_two_forms_of_one_definition(window):
    q, k, v = made(9, 3, 40, 60)
    a, _ = attend(q, k, v, 60, window)
    b, tol = _paged.attend(q, k, v, 60, window)
    assert ((a - b).abs() <= 2.0 ** -45 * (1 + a.abs())).all()
    assert (attend(q, k, v, 60, window)[1] < tol).all()  # 54 pairs of head dim 40: weights in two terms


def weighted(q, k, v, pos, terms):
    """The kernels' rounding of weights to `terms` bf16 terms, all else in 64 bits but the output's."""
    T, H, D = q.shape
    G = H // k.shape[1]
    kk = k.double().repeat_interleave(G, 1).permute(1, 2, 0).contiguous()
    vv = v.double().repeat_interleave(G, 1).transpose(0, 1).contiguous()
    s = q.double().transpose(0, 1) @ kk / D ** 0.5
    s = s.masked_fill((pos + torch.arange(T))[:, None] < torch.arange(k.shape[0])[None], float("-inf"))
    w = torch.exp(s - s.amax(-1, keepdim=True))
    held, left = torch.zeros_like(w), w
    for _ in range(terms):
        held = held + left.to(BF).double()
        left = w - held
    return (held @ vv / w.sum(-1, keepdim=True)).transpose(0, 1).to(BF)


@pytest.mark.parametrize("T,G,D,n", [(1, 4, 128, 300), (7, 4, 64, 500), (40, 2, 64, 200), (20, 2, 96, 700)])
def test_a_term_that_is_dropped_is_found(T, G, D, n):
    """Two terms hold the bound, one does not: a kernel that leaves the second products out fails."""
    assert not rounds_weights(T, G, D, BF)
    q, k, v = made(T, G, D, n)
    want, tol = attend(q, k, v, n)
    close(weighted(q, k, v, n, 2), want, tol)
    with pytest.raises(AssertionError, match="off, worst"):
        close(weighted(q, k, v, n, 1), want, tol)


def test_one_term_holds_the_bound_of_the_rows_that_have_one():
    q, k, v = made(60, 2, 128, 400)
    assert rounds_weights(60, 2, 128, BF)
    want, tol = attend(q, k, v, 400)
    close(weighted(q, k, v, 400, 1), want, tol)
