"""How exact attention of drafted trees in bf16 is: weights are held to 16 bits, whichever kernel a row takes."""
import math
import random

import pytest
import torch

import _tree
from test_gpu_tree_attention import BF, Call, trees

pytestmark = pytest.mark.gpu


def attend(q, k, v, seen):
    """q (H, D) over the keys `seen`: the output in 64 bits and how far it may be off. As _tree.attend, but that a
    weight has two bf16 terms: what the first, rounded by at most 2^-8, leaves is rounded by 2^-8 again, so a
    weight is off by 2^-16."""
    H, D = q.shape
    G, n, step = H // k.shape[1], len(seen), 2.0 ** -24
    kk, vv = (t[seen].double().repeat_interleave(G, 1) for t in (k, v))
    scale = 1 / math.sqrt(D)
    s = torch.matmul(kk.transpose(0, 1), q.double()[:, :, None])[..., 0] * scale
    size = torch.matmul(kk.abs().transpose(0, 1), q.double().abs()[:, :, None])[..., 0].amax(1) * scale
    w = torch.softmax(s, 1)
    out, mean = (torch.matmul(w[:, None], x.transpose(0, 1))[:, 0] for x in (vv, vv.abs()))
    d = (D + 4) * step * size + 8 * step * (1 + size)
    more = torch.expm1(2 * d + 2.0 ** -16 + (n + 64) * step)[:, None]
    return out, more * mean + torch.finfo(BF).eps / 2 * out.abs() * (1 + more)


def check(call):
    y = call.run()
    for b, (p, t) in enumerate(zip(call.pos, call.new)):
        kk, vv = call.pool.rows(b, p + t)
        for i in range(t):
            want, tol = attend(call.q[call.cu[b] + i], kk, vv, _tree.seen_keys(p, i, call.bits[b][i], call.window))
            off = (y[call.cu[b] + i].double() - want).abs()
            assert bool((off <= tol).all()), f"row {b} node {i}: worst {float((off / tol).max()):.3f} of the bound"


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("H,H_kv,T", [(8, 2, 5), (8, 2, 16), (6, 2, 21), (8, 2, 40), (4, 1, 64), (1, 1, 200)])
def test_weights_of_two_terms(H, H_kv, T, D):
    """Blocks of 32, 64 and 128 pairs, rows within one range and over several."""
    rng = random.Random(T * D)
    check(Call([300, 70], trees(rng, [T, T]), H, H_kv, D, 16, BF))
    check(Call([1700, 33], trees(rng, [T, 3]), H, H_kv, D, 32, BF, max_pages=128))


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("neighbour", [1, 20, 90])
def test_a_wider_row_beside_it_costs_a_row_nothing(neighbour, D):
    """A chain of five, alone and beside trees that send the call to another kernel."""
    rng = random.Random(neighbour)
    check(Call([400, 200], [_tree.ancestors([-1, 0, 1, 2, 3]), *trees(rng, [neighbour])], 4, 1, D, 16, BF))


@pytest.mark.parametrize("window", [0, 20, 300])
def test_windows(window):
    rng = random.Random(window)
    for D in (64, 128):
        check(Call([900, 41], trees(rng, [30, 17]), 8, 2, D, 16, BF, window, max_pages=80))
