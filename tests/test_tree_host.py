"""Decoding with drafted trees on the CPU host: what the library and the Python entry points refuse before
anything is launched, and the tests' own plain forms against brute force."""
import itertools
import random

import pytest
import torch

import _tree
from modelcore_amd import _ext
from modelcore_amd.kernels.flash_attn import flash_attn
from modelcore_amd.kernels.paged import paged_keep, paged_tree
from modelcore_amd.sampling import verify_drafts

FAKE = 1 << 20  # never dereferenced: the checks fail first


def refused(status, code, words):
    assert status == code and words in _ext.lib().mcamd_last_error(), (status, _ext.lib().mcamd_last_error())


def attention(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, masks=FAKE, words=1, n_rows=2, total=7, longest=5, H=8, H_kv=2, D=128, page=16,
             cu=FAKE, scratch=None, nbytes=0, dtype=_ext.BF16)
    a.update(kw)
    return _ext.lib().mcamd_flash_attn_paged_tree_with_kvcache(
        a["q"], a["k"], a["v"], FAKE, FAKE, FAKE, 8, FAKE, a["cu"], a["masks"], a["words"], FAKE, a["n_rows"], a["total"],
        a["longest"], a["H"], a["H_kv"], a["D"], 20, a["page"], a["page"] * a["H_kv"] * a["D"], 8, -1, a["dtype"],
        a["scratch"], a["nbytes"], None)


@pytest.mark.parametrize("kw,code,words", [
    (dict(words=0), _ext.EINVAL, b"1 to 16 words"),
    (dict(words=17), _ext.EINVAL, b"1 to 16 words"),
    (dict(longest=65), _ext.EINVAL, b"1 to 16 words"),
    (dict(masks=FAKE + 4), _ext.EINVAL, b"8-byte aligned"),
    (dict(masks=None), _ext.EINVAL, b"null"),
    (dict(k=None), _ext.EINVAL, b"both k and v"),
    (dict(page=24), _ext.EINVAL, b"power of two"),
    (dict(D=264), _ext.EUNSUPPORTED, b"at most 256"),
    (dict(H=9), _ext.EINVAL, b"multiple"),
    (dict(q=FAKE + 8), _ext.EINVAL, b"16-byte"),
    (dict(cu=None), _ext.EINVAL, b"cu_seqlens"),
    (dict(scratch=FAKE + 8, nbytes=1 << 30), _ext.EINVAL, b"aligned"),
])
def test_attention_refuses(kw, code, words):
    refused(attention(**kw), code, words)


def test_attention_of_nothing_is_no_launch():
    assert attention(n_rows=0, total=0, masks=None) == _ext.OK
    assert attention(total=0, masks=None) == _ext.OK


def test_scratch():
    """Of use where keys can be cut into ranges, and only there; rows of few pairs have that of sequences."""
    lib = _ext.lib()
    few = (60, 300, 8, 32, 8, 128, 600, 16, 1024, _ext.BF16)
    assert lib.mcamd_paged_tree_scratch_bytes(*few) == lib.mcamd_paged_scratch_bytes(*few) > 0
    for D in (64, 96, 128, 256):
        for T, dtype in ((16, _ext.BF16), (64, _ext.BF16), (16, _ext.F32)):
            assert lib.mcamd_paged_tree_scratch_bytes(4, 4 * T, T, 16, 4, D, 512, 64, -1, dtype) > 0
            assert lib.mcamd_paged_tree_scratch_bytes(4, 4 * T, T, 16, 4, D, 1, 16, -1, dtype) == 0
    assert lib.mcamd_paged_tree_scratch_bytes(0, 0, 0, 8, 2, 128, 8, 16, -1, _ext.BF16) == 0


def test_plan_refuses():
    lib = _ext.lib()

    def plan(n_rows=2, total=5, words=1, parents=FAKE, masks=FAKE):
        return lib.mcamd_paged_tree(parents, FAKE, FAKE, FAKE, masks, n_rows, total, words, None)

    refused(plan(n_rows=-1), _ext.EINVAL, b"negative")
    refused(plan(total=-1), _ext.EINVAL, b"negative")
    refused(plan(words=0), _ext.EINVAL, b"1 to 16")
    refused(plan(words=17), _ext.EINVAL, b"1 to 16")
    refused(plan(n_rows=0), _ext.EINVAL, b"without a row")
    refused(plan(parents=None), _ext.EINVAL, b"null")
    refused(plan(masks=FAKE + 4), _ext.EINVAL, b"aligned")
    refused(plan(total=0x7fffffff), _ext.EUNSUPPORTED, b"31 bits")
    assert plan(total=0) == _ext.OK


def test_keep_refuses():
    lib = _ext.lib()

    def keep(k=FAKE, slots=2, slot_stride=20 * 16 * 256, table=FAKE, stride=8, kept=FAKE, most=4, n_rows=2, max_pages=8,
             n_pages=20, page=16, page_stride=16 * 256, row=256, dtype=_ext.BF16):
        return lib.mcamd_paged_keep(k, FAKE, slots, slot_stride, table, stride, FAKE, FAKE, kept, most, FAKE, FAKE, FAKE,
                                    n_rows, max_pages, n_pages, page, page_stride, row, dtype, None)

    for kw, code, words in ((dict(dtype=5), _ext.EINVAL, b"dtype"), (dict(slots=-1), _ext.EINVAL, b"positive"),
                            (dict(n_rows=-1), _ext.EINVAL, b"positive"), (dict(row=0), _ext.EINVAL, b"positive"),
                            (dict(max_pages=0), _ext.EINVAL, b"positive"), (dict(most=-1), _ext.EINVAL, b"positive"),
                            (dict(page=20), _ext.EINVAL, b"power of two"), (dict(stride=7), _ext.EINVAL, b"table_stride"),
                            (dict(n_rows=65536), _ext.EUNSUPPORTED, b"65535"), (dict(slots=32768), _ext.EUNSUPPORTED, b"slots"),
                            (dict(n_pages=1 << 28), _ext.EUNSUPPORTED, b"31 bits"),
                            (dict(page_stride=16 * 256 - 8), _ext.EINVAL, b"page_stride"),
                            (dict(slot_stride=20 * 16 * 256 - 8), _ext.EINVAL, b"slot_stride"),
                            (dict(row=4, page_stride=16 * 4), _ext.EINVAL, b"16-byte"), (dict(k=FAKE + 2), _ext.EINVAL, b"16-byte"),
                            (dict(k=None), _ext.EINVAL, b"null"), (dict(table=None), _ext.EINVAL, b"null"),
                            (dict(kept=None), _ext.EINVAL, b"null")):
        refused(keep(**kw), code, words)
    assert keep(n_rows=0) == _ext.OK


def test_verify_refuses():
    lib = _ext.lib()
    most = 1 << 23  # tokens of a vocabulary whose remainder is summed

    def verify(logits=FAKE, ls=100, probs=None, ps=0, cu=FAKE, n_rows=2, total=5, longest=4, V=100, t=1.0, scratch=FAKE,
               nbytes=1 << 40):
        return lib.mcamd_verify_drafts(logits, ls, probs, ps, FAKE, FAKE, cu, FAKE, FAKE, FAKE, FAKE, n_rows, total, longest,
                                       V, t, scratch, nbytes, None)

    need = lib.mcamd_verify_drafts_scratch_bytes(5, 100)
    assert need > 0 and lib.mcamd_verify_drafts_scratch_bytes(0, 100) == 0

    for kw, code, words in ((dict(n_rows=-1), _ext.EINVAL, b"n_rows"), (dict(total=-1), _ext.EINVAL, b"total"),
                            (dict(longest=0), _ext.EINVAL, b"max_seqlen"), (dict(longest=1025), _ext.EUNSUPPORTED, b"1024"),
                            (dict(V=0), _ext.EINVAL, b"vocab"), (dict(V=1 << 31, ls=1 << 31), _ext.EINVAL, b"vocab"),
                            (dict(t=-1.0), _ext.EINVAL, b"temperature"), (dict(t=float("nan")), _ext.EINVAL, b"temperature"),
                            (dict(t=float("inf")), _ext.EINVAL, b"temperature"), (dict(ls=99), _ext.EINVAL, b"stride"),
                            (dict(probs=FAKE, ps=99), _ext.EINVAL, b"stride"), (dict(logits=None), _ext.EINVAL, b"null"),
                            (dict(cu=None), _ext.EINVAL, b"null"), (dict(total=0x7fffffff), _ext.EUNSUPPORTED, b"31 bits"),
                            (dict(V=most + 1, ls=most + 1, probs=FAKE, ps=most + 1), _ext.EUNSUPPORTED, b"2^23"),
                            (dict(V=1 << 30, ls=1 << 30, total=1 << 10), _ext.EUNSUPPORTED, b"grid"),
                            (dict(scratch=FAKE + 8), _ext.EINVAL, b"aligned"), (dict(scratch=None), _ext.EWORKSPACE, b"scratch"),
                            (dict(nbytes=need - 1), _ext.EWORKSPACE, b"scratch")):
        refused(verify(**kw), code, words)
    assert verify(n_rows=0) == _ext.OK


def test_cpu_tensors_are_refused():
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="paged_tree"):
        paged_tree(i, i, i[:2], max_seqlen=3)
    with pytest.raises(RuntimeError, match="paged_keep"):
        paged_keep(torch.zeros(1, 3, 16, 1, 8), torch.zeros(1, 3, 16, 1, 8), torch.zeros(1, 3, dtype=torch.int32), i[:1], i[:1],
                   i[None], i[:1], i, i[:1])
    with pytest.raises(RuntimeError, match="verify_drafts"):
        verify_drafts(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), i, i[:2], torch.zeros(3), max_seqlen=3)
    with pytest.raises(RuntimeError, match="flash_attn_paged_tree_with_kvcache"):
        flash_attn.flash_attn_paged_tree_with_kvcache(torch.zeros(1, 1, 1, 8), None, None)


# -----------------------------------------------------------------------------------------------
# The plain forms
# -----------------------------------------------------------------------------------------------
def test_plain_plan():
    rng = random.Random(0)
    for n in (1, 5, 70):
        parents = _tree.random_parents(rng, n, 0.2)
        pos, masks = _tree.plan(parents, [n], [7], 2)
        for i in range(n):
            assert pos[i] == 7 + (pos[parents[i]] - 6 if parents[i] >= 0 else 0)
            for j in range(n):
                bit = (masks[i][j // 64] >> (j % 64)) & 1
                up = j == i or (parents[i] >= 0 and (masks[parents[i]][j // 64] >> (j % 64)) & 1)
                assert bit == up


def test_plain_windows():
    """Who sees whom by distance along the path."""
    parents = [-1, 0, 0, 1, 3, 2]
    up = _tree.ancestors(parents)
    for window in range(8):
        for i in range(6):
            path = list(range(4)) + [4 + j for j in up[i]]
            assert _tree.seen_keys(4, i, up[i], window) == path[-(window + 1):]


def test_plain_walk_is_a_draw_from_the_target():
    """All outcomes of two drafts and their numbers on a grid: the first emitted token's frequencies are p, exactly up
    to the grid, for drafts drawn from q and for guesses."""
    p, q = [0.5, 0.3, 0.2], [0.25, 0.5, 0.25]
    import math
    logits = [[math.log(x) for x in p]] * 3
    grid = [(i + 0.5) / 40 for i in range(40)]
    for drawn in (False, True):
        freq = [0.0] * 3
        for x, y in itertools.product(range(3), repeat=2) if drawn else [(1, 2)]:
            share = q[x] * q[y] if drawn else 1.0
            for u in itertools.product(grid, repeat=3):
                _, out, _ = _tree.verify(logits, [0, x, y], [-1, 0, 0], list(u), 1.0, [q] * 3 if drawn else None)
                freq[out[0]] += share / 40 ** 3
        # A border of each of the three numbers falls inside a step of the grid.
        assert all(abs(f - x) < 3 / 40 for f, x in zip(freq, p)), freq
