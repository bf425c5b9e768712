"""The paged KV cache's operators on the GPU against plain 64-bit forms: pages and slots, the
pre-attention step by slot, and attention over pages for single tokens, chunks and mixtures of them."""
import random

import pytest
import torch

from _paged import Pool, attend, release, reserve, rotated

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _op():
    from modelcore_amd.kernels.flash_attn import flash_attn
    return flash_attn.flash_attn_paged_with_kvcache


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g).to(dtype)


def close(got, want, tol, what=""):
    off = (got.detach().cpu().double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((off - tol)[bad].max()):.3e} past"


def same_bits(a, b):
    view = {BF: torch.int16, F32: torch.int32}[a.dtype]
    return torch.equal(a.cpu().contiguous().view(view), b.cpu().contiguous().view(view))


def run_attention(pos, new, H, H_kv, D, page, dtype, window=-1, packed=None, append=True, seed=0,
                  stale=float("nan"), pad=0):
    """One call on rows at `pos` with `new` tokens each, checked against the 64-bit form, its appends
    bit for bit; returns the output."""
    g = torch.Generator().manual_seed(seed + 1)
    pool = Pool([p + t for p, t in zip(pos, new)], page, H_kv, D, dtype, seed=seed, stale=stale)
    n = sum(new)
    q = randn(g, n + pad, H, D, dtype=dtype)
    kp, vp = pool.k.clone(), pool.v.clone()
    k, v = torch.randn(n + pad, H_kv, D, generator=g).to(dtype), randn(g, n + pad, H_kv, D, dtype=dtype)
    at = 0
    for b, (p, t) in enumerate(zip(pos, new)):
        for i in range(t):
            where = pool.place(b, p + i)
            if append:  # what the pages hold there before the call is nobody's
                kp[where], vp[where] = stale, stale
                pool.k[where], pool.v[where] = k[at + i], v[at + i]
        at += t
    kg, vg = kp.to(DEV), vp.to(DEV)
    packed = packed if packed is not None else len(set(new)) > 1 or pad > 0
    kw = {}
    shape = (len(pos), new[0]) if not packed else (n + pad,)
    if packed:
        cu = [0]
        for t in new:
            cu.append(cu[-1] + t)
        kw = {"cu_seqlens": i32(cu), "max_seqlen": max(new)}
    if append:
        kw.update(k=k.to(DEV).view(*shape, H_kv, D), v=v.to(DEV).view(*shape, H_kv, D))
    y = _op()(q.to(DEV).view(*shape, H, D), kg, vg, block_table=pool.table.to(DEV),
              cache_seqlens=i32(pos), causal=True, window_size=(window, 0), **kw)
    torch.cuda.synchronize()
    assert same_bits(kg, pool.k) and same_bits(vg, pool.v), "the pages"
    y = y.view(-1, H, D)[:n]
    at = 0
    for b, (p, t) in enumerate(zip(pos, new)):
        if t == 0:
            continue
        kk, vv = pool.rows(b, p + t)
        want, tol = attend(q[at:at + t], kk, vv, p, window)
        close(y[at:at + t], want, tol, f"row {b} at {p} + {t}")
        at += t
    return y


# -----------------------------------------------------------------------------------------------
# Attention
# -----------------------------------------------------------------------------------------------
HEADS = [(1, 1, 64), (12, 12, 64), (16, 4, 128), (32, 8, 128), (6, 2, 96), (8, 8, 256), (5, 1, 40),
         (7, 1, 128), (24, 2, 128), (64, 1, 128), (3, 3, 32), (4, 2, 8), (40, 2, 192), (15, 3, 160)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,H_kv,D", HEADS)
def test_single_tokens(H, H_kv, D, dtype):
    run_attention([0, 15, 16, 17, 63, 130, 1, 300], [1] * 8, H, H_kv, D, 16, dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("window", [-1, 0, 1, 15, 16, 100])
def test_single_tokens_pages_and_windows(page, window):
    run_attention([0, 31, 32, 95, 257, 511], [1] * 6, 8, 2, 128, page, BF, window)
    run_attention([5, 33, 200], [1] * 3, 4, 4, 64, page, F32, window)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,H_kv,D", HEADS)
def test_chunks(H, H_kv, D, dtype):
    run_attention([0, 37, 128], [67] * 3, H, H_kv, D, 32, dtype)


@pytest.mark.parametrize("T", [2, 3, 8, 9, 31, 33, 64, 65, 129, 257])
@pytest.mark.parametrize("window", [-1, 0, 40])
def test_chunk_lengths(T, window):
    run_attention([0, 50], [T] * 2, 4, 1, 128, 16, BF, window, seed=T)
    run_attention([17], [T], 2, 2, 64, 16, F32, window, seed=T)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 40])
def test_windows_wider_than_any_row(window):
    run_attention([40, 0, 300], [1, 70, 9], 4, 2, 128, 16, BF, window)
    run_attention([40, 0, 300], [1, 70, 9], 4, 2, 64, 16, F32, window)


@pytest.mark.parametrize("dtype,H,H_kv,D", [(BF, 8, 2, 128), (BF, 6, 6, 64), (F32, 4, 2, 128), (BF, 4, 1, 256)])
@pytest.mark.parametrize("window", [-1, 33])
def test_mixed_rows(dtype, H, H_kv, D, window):
    """Rows with one token, with none, with a few and with many, in one call; tokens past the last row
    are nobody's."""
    run_attention([40, 0, 700, 9, 0, 333, 16, 64], [1, 150, 1, 0, 5, 1, 90, 2], H, H_kv, D, 16, dtype,
                  window, pad=7)


def test_many_rows():
    """More rows than the lanes of a wave, and than four of them, of mixed lengths."""
    new = [(1, 0, 3, 1, 20, 1, 1)[b % 7] for b in range(300)]
    run_attention([(b * 29) % 70 for b in range(300)], new, 4, 2, 64, 16, BF)
    run_attention([(b * 29) % 70 for b in range(300)], new, 4, 1, 128, 16, BF)
    run_attention([(b * 13) % 50 for b in range(100)], [1] * 100, 4, 1, 128, 16, BF)


@pytest.mark.parametrize("dtype,H,H_kv,D", [(BF, 8, 2, 128), (BF, 4, 4, 64), (F32, 4, 2, 64), (BF, 2, 1, 256)])
def test_long_rows_are_cut(dtype, H, H_kv, D):
    """One row of many keys, alone and beside short ones: its keys are cut into ranges and merged."""
    run_attention([6000], [1], H, H_kv, D, 64, dtype)
    run_attention([3000, 5, 900], [1, 1, 1], H, H_kv, D, 16, dtype)
    run_attention([4000], [3], H, H_kv, D, 64, dtype)
    run_attention([2500], [40], H, H_kv, D, 16, dtype)
    run_attention([2500, 10, 1500], [30, 1, 1], H, H_kv, D, 16, dtype)
    run_attention([2100], [1], H, H_kv, D, 16, dtype, window=1500)


@pytest.mark.parametrize("dtype,H,H_kv,D", [(BF, 8, 2, 128), (BF, 8, 2, 64), (F32, 8, 2, 64), (BF, 6, 2, 96)])
def test_long_chunks_of_few_rows(dtype, H, H_kv, D):
    """Blocks of many pairs that are cut, rows that end inside one, more new tokens than one launch appends."""
    run_attention([1900], [150], H, H_kv, D, 16, dtype)
    run_attention([1500, 0, 300], [200, 33, 90], H, H_kv, D, 32, dtype, pad=3)
    run_attention([1800], [70], H, H_kv, D, 16, dtype, window=1200)
    run_attention([30, 200, 900, 0, 5], [1, 400, 2, 0, 130], H, H_kv, D, 16, dtype)


@pytest.mark.parametrize("dtype,H,H_kv,D", [(BF, 32, 32, 128), (BF, 64, 32, 64), (F32, 32, 32, 64), (BF, 48, 24, 128)])
def test_the_deepest_blocks_are_halved(dtype, H, H_kv, D):
    """More blocks than may be cut at will, fewer than the chip takes at once: the deepest in two."""
    run_attention([900, 20, 700, 0, 350], [40, 33, 64, 50, 35], H, H_kv, D, 16, dtype)
    run_attention([30, 1200, 0, 640, 5, 1100], [1, 40, 45, 36, 1, 34], H, H_kv, D, 64, dtype, seed=1)
    run_attention([600, 500, 9], [290, 40, 1], H, H_kv, D, 16, dtype, seed=2, append=False)
    run_attention([900, 20, 800, 0, 350], [40, 33, 64, 50, 35], H, H_kv, D, 16, dtype, window=600)


def test_halved_blocks_beside_a_row_that_does_not_fit():
    """Its outputs are NaN, the others' those of a call without it, and the same again."""
    g = torch.Generator().manual_seed(24)
    new, pos = [40, 33, 64, 50], [900, 700, 1100, 5]
    pool = Pool([p + t for p, t in zip(pos, new)], 16, 32, 128, BF, stale=1.0)
    q = randn(g, sum(new), 32, 128, dtype=BF)
    kg, vg, table = pool.k.to(DEV), pool.v.to(DEV), pool.table.to(DEV)
    cu = i32([0, 40, 73, 137, 187])

    def call(pos):
        return _op()(q.to(DEV), kg, vg, block_table=table, cache_seqlens=i32(pos), cu_seqlens=cu, max_seqlen=64,
                     causal=True).cpu()
    for lost in (2 ** 31 - 1, -1, 16 * pool.table.shape[1] - 49):
        y = call([900, 700, 1100, lost])
        assert y[137:].isnan().all() and torch.equal(y[:137], call([900, 700, 1100, lost])[:137])
        for b in range(3):
            a, e = [0, 40, 73][b], [40, 73, 137][b]
            want, tol = attend(q[a:e], *pool.rows(b, pos[b] + new[b]), pos[b], -1)
            close(y[a:e], want, tol)


@pytest.mark.parametrize("dtype,T", [(BF, 7), (F32, 1)])
def test_many_rows_of_a_few_tokens_are_cut(dtype, T):
    """More pairs than the merge has workgroups for."""
    run_attention([500 + 3 * b for b in range(90)], [T - b % 2 if T > 1 else 1 for b in range(90)], 16, 4, 64, 16,
                  dtype, packed=True)


@pytest.mark.parametrize("seed", range(48))
def test_random_calls(seed):
    """Rows, heads, pages, windows and lengths at random, every third seed of bf16 / 128."""
    rng = random.Random(seed)
    dtype = rng.choice([BF, BF, F32])
    D = rng.choice([8, 16, 24, 40, 64, 64, 72, 96, 128, 136, 192, 256])
    if seed % 3 == 0:
        dtype, D = BF, 128
    G = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16, 64])
    H_kv = rng.choice([1, 2, 3, 4, 8]) if G < 16 else 1
    rows = rng.choice([1, 2, 5, 9, 30, 70])
    deep = rng.choice([30, 200, 900, 2500 if rows < 9 else 300])
    pos = [rng.randint(0, deep) for _ in range(rows)]
    kind = rng.choice(["ones", "same", "mixed", "mixed", "mixed"])
    if kind == "ones":
        new = [1] * rows
    elif kind == "same":
        new = [rng.randint(1, 300 // rows + 1)] * rows
    else:
        new = [rng.choice([0, 1, 1, 1, rng.randint(2, 9), rng.randint(1, 240 // rows + 2)]) for _ in range(rows)]
    if sum(new) == 0:
        new[0] = 1
    run_attention(pos, new, G * H_kv, H_kv, D, rng.choice([16, 16, 32, 64, 256 if rows > 5 else 1024]), dtype,
                  window=rng.choice([-1, -1, 0, 5, 33, 300]), append=rng.random() < 0.8, seed=seed,
                  pad=rng.choice([0, 0, 3]), packed=True if rng.random() < 0.3 else None)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (F32, 64)])
def test_without_append(dtype, D):
    run_attention([30, 100, 0], [1, 20, 5], 4, 2, D, 16, dtype, append=False)
    run_attention([30, 100], [1, 1], 4, 2, D, 16, dtype, append=False)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("stale", [float("nan"), float("inf"), torch.finfo(BF).min])
def test_what_no_row_holds_reaches_no_output(dtype, D, stale):
    """Pages of no row, and the rest of a row's last page, hold anything at all."""
    run_attention([3, 17, 40], [1, 1, 1], 4, 2, D, 16, dtype, stale=stale)
    run_attention([3, 17, 40], [5, 40, 1], 4, 2, D, 16, dtype, stale=stale)
    run_attention([600, 2], [70, 3], 4, 2, D, 16, dtype, stale=stale, window=90)


def _call(pool, q, pos, k=None, v=None, window=-1, kg=None, vg=None, table=None):
    """Uniform rows, q (B, T, H, D)."""
    kg = pool.k.to(DEV) if kg is None else kg
    vg = pool.v.to(DEV) if vg is None else vg
    return _op()(q.to(DEV), kg, vg, k=None if k is None else k.to(DEV),
                 v=None if v is None else v.to(DEV),
                 block_table=(pool.table if table is None else table).to(DEV),
                 cache_seqlens=i32(pos), causal=True, window_size=(window, 0)).cpu()


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (F32, 64)])
@pytest.mark.parametrize("T", [4, 40, 200])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_masked_values_that_are_not_finite(dtype, D, T, value):
    """An infinity or NaN in V reaches the queries that see its key, and no other."""
    g = torch.Generator().manual_seed(T)
    pos, bad = 70, 70 + T // 2
    pool = Pool([pos + T], 16, 2, D, dtype)
    q = randn(g, 1, T, 8, D, dtype=dtype)
    p, o = pool.place(0, bad)
    pool.v[p, o, 1, 3] = value
    y = _call(pool, q, [pos])
    clean = pool.v.clone()
    clean[p, o, 1, 3] = 0
    kk, vv = pool.k, clean
    pool.v = clean
    kk, vv = pool.rows(0, pos + T)
    want, tol = attend(q[0], kk, vv, pos, -1)
    seen = torch.zeros(T, 8, D, dtype=torch.bool)
    seen[T // 2:, 4:, 3] = True
    assert not y[0][seen].isfinite().any()
    close(torch.where(seen, 0, y[0]), torch.where(seen, 0, want), tol)
    # behind a window it is seen by the first window + 1 queries from its own on
    pool.v = pool.v.clone()
    pool.v[p, o, 1, 3] = value
    y = _call(pool, q, [pos], window=3)
    seen[T // 2 + 4:] = False
    want, tol = attend(q[0], kk, vv, pos, 3)
    assert not y[0][seen].isfinite().any()
    close(torch.where(seen, 0, y[0]), torch.where(seen, 0, want), tol)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (F32, 64)])
@pytest.mark.parametrize("T", [1, 40, 200])
def test_extreme_scores(dtype, D, T):
    """Scores far apart, up to where the weights of all keys but one vanish, and equal ones."""
    g = torch.Generator().manual_seed(5)
    pool = Pool([100 + T], 16, 2, D, dtype)
    pool.k[torch.isfinite(pool.k)] *= 30
    q = randn(g, 1, T, 4, D, dtype=dtype) * 4
    y = _call(pool, q, [100])
    kk, vv = pool.rows(0, 100 + T)
    want, tol = attend(q[0], kk, vv, 100, -1)
    close(y[0], want, tol)
    pool.k[torch.isfinite(pool.k)] = 0
    y = _call(pool, q, [100])
    want, tol = attend(q[0], *pool.rows(0, 100 + T), 100, -1)
    close(y[0], want, tol)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (F32, 64)])
@pytest.mark.parametrize("T", [1, 30, 300])
def test_pages_and_positions_outside(dtype, D, T):
    """A row past its line of the table is NaN and appends nothing; a page outside the pool makes the
    queries that see its keys NaN and keeps their tokens out; other rows are as they are alone."""
    g = torch.Generator().manual_seed(9)
    pos = [40, 40, 40, 40, 40]
    pool = Pool([340] * 5, 16, 2, D, dtype, stale=1.0)
    room = pool.table.shape[1] * 16
    q, k, v = (randn(g, 5, T, h, D, dtype=dtype) for h in (4, 2, 2))
    alone = _call(pool, q, pos, k, v)
    table = pool.table.clone()
    table[1, 0] = pool.n_pages      # one past the pool
    table[2, 0] = -1
    table[3, (40 + T // 2) // 16] = 2 ** 31 - 1
    kg, vg = pool.k.to(DEV), pool.v.to(DEV)
    pos[4] = room - T + 1
    y = _call(pool, q, pos, k, v, kg=kg, vg=vg, table=table)
    assert torch.equal(y[0], alone[0])
    for b in (1, 2, 4):
        assert y[b].isnan().all(), b
    first = (40 + T // 2) // 16 * 16  # the first key in the lost page
    ok = max(0, first - 40)
    assert torch.equal(y[3, :ok], alone[3, :ok]) or \
        torch.allclose(y[3, :ok].float(), alone[3, :ok].float(), atol=3e-2, rtol=0)
    assert y[3, ok:].isnan().all()
    held = {int(x) for x in pool.table[3, 40 // 16:(40 + T - 1) // 16 + 1]}
    for b in (4,):  # nothing of row 4 was written where its table leads
        for p in pool.table[b].tolist():
            if p >= 0:
                assert same_bits(kg[p], pool.k[p])
    lost = int(pool.table[3, (40 + T // 2) // 16])
    assert lost in held and same_bits(kg[lost], pool.k[lost])
    pos[4] = -1
    y = _call(pool, q, pos, k, v, table=table)
    assert y[4].isnan().all() and torch.equal(y[0], alone[0])


def test_checked_mode_raises_before_launching():
    from modelcore_amd.kernels import flash_attn as fa
    pool = Pool([40], 16, 2, 64, BF, stale=1.0)
    q = torch.zeros(1, 1, 2, 64, dtype=BF)
    fa.set_checked(True)
    try:
        _call(pool, q, [39])
        with pytest.raises(IndexError, match="line of the block table"):
            _call(pool, q, [16 * pool.table.shape[1]])
        with pytest.raises(IndexError, match="not one of the pool"):
            _call(pool, q, [50])
    finally:
        fa.set_checked(False)


def test_rows_that_read_the_same_pages():
    pool = Pool([200], 16, 2, 128, BF)
    g = torch.Generator().manual_seed(3)
    q = randn(g, 5, 1, 8, 128, dtype=BF)
    y = _call(pool, q, [199, 50, 199, 16, 0], table=pool.table.expand(5, -1))
    for b, p in enumerate([199, 50, 199, 16, 0]):
        want, tol = attend(q[b], *pool.rows(0, p + 1), p, -1)
        close(y[b], want, tol)


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_strides(T, dtype):
    """Slots of a pool of several, pages further apart than their size, a table cut out of a wider one,
    queries and new keys that are views of one projection."""
    g = torch.Generator().manual_seed(4)
    pool = Pool([90 + T, 20 + T], 16, 2, 64, dtype)
    n = pool.n_pages
    wide_k, wide_v = torch.full((n, 3, 16, 2, 64), 7, dtype=dtype), torch.full((n, 3, 16, 2, 64), 7, dtype=dtype)
    wide_k[:, 1], wide_v[:, 1] = pool.k, pool.v
    kg, vg = wide_k.to(DEV), wide_v.to(DEV)
    table = torch.full((2, pool.table.shape[1] + 9), 5, dtype=torch.int32)
    table[:, 4:4 + pool.table.shape[1]] = pool.table
    qkv = randn(g, 2, T, 8, 64, dtype=dtype)
    dq = qkv.to(DEV)
    y = _op()(dq[:, :, :4], kg[:, 1], vg[:, 1], k=dq[:, :, 4:6], v=dq[:, :, 6:],
              block_table=table.to(DEV)[:, 4:4 + pool.table.shape[1]],
              cache_seqlens=i32([90, 77, 20])[::2], causal=True)
    for b, p in enumerate((90, 20)):
        for t in range(T):
            where = pool.place(b, p + t)
            pool.k[where], pool.v[where] = qkv[b, t, 4:6], qkv[b, t, 6:]
        want, tol = attend(qkv[b, :, :4], *pool.rows(b, p + T), p, -1)
        close(y[b], want, tol)
    wide_k[:, 1], wide_v[:, 1] = pool.k, pool.v
    assert same_bits(kg, wide_k) and same_bits(vg, wide_v)


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (F32, 128)])
def test_offsets_past_32_bits(T, dtype, D):
    """A pool of more than 2^31 elements, a row whose pages lie at both ends of it."""
    page, H_kv = 256, 8
    n = (1 << 31) // (page * H_kv * D) + 40
    kg = torch.empty(n, page, H_kv, D, dtype=dtype, device=DEV)
    vg = torch.empty(n, page, H_kv, D, dtype=dtype, device=DEV)
    g = torch.Generator().manual_seed(6)
    ids = [n - 1, 0, n - 2, 1, n - 17]
    pos = 5 * page - T
    k_all, v_all = randn(g, 5 * page, H_kv, D, dtype=dtype), randn(g, 5 * page, H_kv, D, dtype=dtype)
    for i, p in enumerate(ids):
        kg[p] = k_all[i * page:(i + 1) * page].to(DEV)
        vg[p] = v_all[i * page:(i + 1) * page].to(DEV)
    kg[n - 17, page - T:], vg[n - 17, page - T:] = 0, 0
    q = randn(g, 1, T, 16, D, dtype=dtype)
    y = _op()(q.to(DEV), kg, vg, k=k_all[None, pos:].to(DEV), v=v_all[None, pos:].to(DEV),
              block_table=i32([ids]), cache_seqlens=i32([pos]), causal=True).cpu()
    want, tol = attend(q[0], k_all, v_all, pos, -1)
    close(y[0], want, tol)
    assert same_bits(kg[n - 17], k_all[4 * page:])


@pytest.mark.parametrize("dtype,T", [(BF, 1), (BF, 40), (F32, 1), (F32, 40)])
@pytest.mark.parametrize("past", [-16, 16])
def test_pages_far_apart(dtype, T, past):
    """Pages 2 GiB apart, a little less and a little more, as in the views of one layer of a stacked pool."""
    page, H_kv, D = 16, 2, 128
    step = ((1 << 31) + past) // dtype.itemsize  # elements between pages
    flat = torch.empty(2 * step + page * H_kv * D * 2, dtype=dtype, device=DEV)
    shape, strides = (3, page, H_kv, D), (step, H_kv * D, D, 1)
    kg = torch.as_strided(flat, shape, strides)
    vg = torch.as_strided(flat, shape, strides, page * H_kv * D)
    g = torch.Generator().manual_seed(16)
    pos = 3 * page - T
    k_all, v_all = randn(g, 3 * page, H_kv, D, dtype=dtype), randn(g, 3 * page, H_kv, D, dtype=dtype)
    for i, p in enumerate((2, 0, 1)):
        kg[p], vg[p] = k_all[i * page:(i + 1) * page].to(DEV), v_all[i * page:(i + 1) * page].to(DEV)
    q = randn(g, 1, T, 8, D, dtype=dtype)
    y = _op()(q.to(DEV), kg, vg, block_table=i32([[2, 0, 1]]), cache_seqlens=i32([pos]), causal=True)
    want, tol = attend(q[0], k_all, v_all, pos, -1)
    close(y[0], want, tol)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H", [5, 8, 33, 40, 64])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_new_value_that_is_not_finite(dtype, H, value):
    """Heads in several blocks all see the token's own value, which its page does not hold before."""
    pool = Pool([20, 4], 16, 1, 128, dtype, stale=3.0)
    g = torch.Generator().manual_seed(18)
    q = randn(g, 2, 1, H, 128, dtype=dtype)
    k, v = randn(g, 2, 1, 1, 128, dtype=dtype), randn(g, 2, 1, 1, 128, dtype=dtype)
    v[0, 0, 0, 7] = value
    y = _call(pool, q, [19, 3], k, v)
    for b, p in enumerate((19, 3)):
        pool.k[pool.place(b, p)], pool.v[pool.place(b, p)] = k[b, 0], v[b, 0]
    other = [d for d in range(128) if d != 7]
    for b, p in enumerate((19, 3)):
        kk, vv = pool.rows(b, p + 1)
        want, tol = attend(q[b], kk, vv.nan_to_num(0.0, 0.0), p, -1)
        close(y[b][..., other], want[..., other], tol[..., other])
        if b == 1:
            close(y[b], want, tol)
    assert (y[0, ..., 7].isnan() if value != value else y[0, ..., 7] == value).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,H_kv", [(16, 1), (32, 1), (33, 1), (64, 1), (6, 6), (20, 5), (48, 12)])
def test_rows_at_the_edge_of_few_pairs(H, H_kv, dtype):
    """Rows of 31 to 66 pairs, uniform and packed, of one block of queries and of two."""
    G = H // H_kv
    near = sorted({max(1, 32 // G + i) for i in (-1, 0, 1)} | {1, 2})
    for T in near:
        run_attention([21, 300], [T, T], H, H_kv, 64, 16, dtype, seed=T)
    run_attention([21 * i for i in range(len(near))], near, H, H_kv, 128, 32, dtype, window=50, packed=True)


@pytest.mark.parametrize("H,H_kv,D", [(12, 12, 64), (8, 4, 32), (4, 1, 128), (6, 2, 256), (9, 1, 40)])
def test_single_tokens_of_many_keys_fp32(H, H_kv, D):
    """Cut into ranges, with a head to a wave and a head to a workgroup, with and without a window."""
    run_attention([4000, 0, 777, 16, 2047], [1] * 5, H, H_kv, D, 16, F32)
    run_attention([4000, 0, 777, 16, 2047], [1] * 5, H, H_kv, D, 64, F32, window=900)
    run_attention([300 + 13 * b for b in range(70)], [1] * 70, H, H_kv, D, 16, F32)
    run_attention([1500, 3, 900, 0], [1, 20, 1, 1], H, H_kv, D, 16, F32, pad=3)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (F32, 64)])
@pytest.mark.parametrize("longest", [1, 3, 40])
def test_tokens_past_max_seqlen_are_left_out(dtype, D, longest):
    """Rows longer than the call was told: their first tokens as in a call that was told right, the others
    neither read nor written, and the rows beside them whole."""
    new, pos = [20, 1, 70, 2], [30, 700, 10, 5]
    g = torch.Generator().manual_seed(20)
    pool = Pool([p + t for p, t in zip(pos, new)], 16, 2, D, dtype, stale=9.0)
    kp, vp = pool.k.clone(), pool.v.clone()
    q, k, v = (randn(g, sum(new), h, D, dtype=dtype) for h in (8, 2, 2))
    cu = [0, 20, 21, 91, 93]
    for b, (p, t) in enumerate(zip(pos, new)):
        for i in range(t):
            where = pool.place(b, p + i)
            kp[where], vp[where] = 9.0, 9.0
            here = i < longest
            pool.k[where] = k[cu[b] + i] if here else 9.0
            pool.v[where] = v[cu[b] + i] if here else 9.0
    kg, vg = kp.to(DEV), vp.to(DEV)
    y = _op()(q.to(DEV), kg, vg, k=k.to(DEV), v=v.to(DEV), block_table=pool.table.to(DEV),
              cache_seqlens=i32(pos), cu_seqlens=i32(cu), max_seqlen=longest, causal=True)
    torch.cuda.synchronize()
    assert same_bits(kg, pool.k) and same_bits(vg, pool.v)
    for b, (p, t) in enumerate(zip(pos, new)):
        n = min(t, longest)
        want, tol = attend(q[cu[b]:cu[b] + n], *pool.rows(b, p + n), p, -1)
        close(y[cu[b]:cu[b] + n], want, tol, f"row {b}")


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (F32, 64)])
def test_captured_calls_follow_their_inputs(dtype, D):
    """Two graphs out of one memory pool, of a mixed call and of single tokens: each replay, with eager calls
    and synchronizations in between, gives the bits of an eager call on what the buffers hold then."""
    g = torch.Generator().manual_seed(22)
    pool = Pool([1400, 60, 900], 16, 2, D, dtype, stale=0.0)
    kg, vg, table = pool.k.to(DEV), pool.v.to(DEV), pool.table.to(DEV)
    calls = []
    for new in ([1, 40, 5], [1, 1, 1]):
        n = sum(new)
        bufs = {"q": randn(g, n, 8, D, dtype=dtype).to(DEV), "k": randn(g, n, 2, D, dtype=dtype).to(DEV),
                "v": randn(g, n, 2, D, dtype=dtype).to(DEV), "pos": i32([0, 0, 0])}
        cu = i32([0, new[0], new[0] + new[1], n])
        calls.append((bufs, lambda kk, vv, b=bufs, cu=cu, m=max(new): _op()(
            b["q"], kk, vv, k=b["k"], v=b["v"], block_table=table, cache_seqlens=b["pos"], cu_seqlens=cu,
            max_seqlen=m, causal=True)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _, call in calls:
            call(kg, vg)
    torch.cuda.current_stream().wait_stream(side)
    share, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for _, call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side, pool=share):
            outs.append(call(kg, vg))
    for i in range(6):
        got, want = [], []
        ke, ve = kg.clone(), vg.clone()
        for bufs, call in calls:
            for name in ("q", "k", "v"):
                bufs[name].copy_(randn(g, *bufs[name].shape, dtype=dtype))
            bufs["pos"].copy_(torch.tensor([(i * 271 + 3) % 1390, i, (i * 97) % 850], dtype=torch.int32))
        for (bufs, call), graph, out in zip(calls, graphs, outs):
            graph.replay()
            got.append(out.clone())
            want.append(call(ke, ve))
            if i % 2:
                torch.cuda.synchronize()
        for a, b in zip(got + [kg, vg], want + [ke, ve]):
            assert same_bits(a, b), i


def _attention_args(**kw):
    z = lambda *shape, dtype=BF: torch.zeros(*shape, dtype=dtype, device=DEV)  # noqa: E731
    args = {"q": z(2, 1, 4, 64), "k_pages": z(4, 16, 2, 64), "v_pages": z(4, 16, 2, 64),
            "block_table": z(2, 2, dtype=torch.int32), "cache_seqlens": z(2, dtype=torch.int32)}
    args.update({n: x(z) if callable(x) else x for n, x in kw.items()})
    return args


@pytest.mark.parametrize("error,words,kw", [
    (ValueError, "q must be", {"q": lambda z: z(2, 4, 64)}),
    (ValueError, "block_table", {"block_table": lambda z: z(2, 2, dtype=torch.int64)}),
    (ValueError, "block_table", {"block_table": lambda z: z(2, 4, dtype=torch.int32)[:, ::2]}),
    (ValueError, "block_table", {"block_table": None}),
    (ValueError, "rows", {"block_table": lambda z: z(3, 2, dtype=torch.int32)}),
    (ValueError, "cache_seqlens", {"cache_seqlens": None}),
    (ValueError, "cache_seqlens", {"cache_seqlens": lambda z: z(3, dtype=torch.int32)}),
    (ValueError, "both k and v", {"k": lambda z: z(2, 1, 2, 64)}),
    (ValueError, "k/v must be", {"k": lambda z: z(2, 2, 2, 64), "v": lambda z: z(2, 2, 2, 64)}),
    (TypeError, "k is", {"k": lambda z: z(2, 1, 2, 64, dtype=F32), "v": lambda z: z(2, 1, 2, 64, dtype=F32)}),
    (TypeError, "k_pages is", {"k_pages": lambda z: z(4, 16, 2, 64, dtype=F32)}),
    (ValueError, "contiguous", {"k_pages": lambda z: z(4, 2, 16, 64).transpose(1, 2)}),
    (ValueError, "page stride", {"v_pages": lambda z: z(4, 2, 16, 2, 64)[:, 0]}),
    (ValueError, "power of two", {"k_pages": lambda z: z(4, 24, 2, 64), "v_pages": lambda z: z(4, 24, 2, 64)}),
    (ValueError, "power of two", {"k_pages": lambda z: z(4, 8, 2, 64), "v_pages": lambda z: z(4, 8, 2, 64)}),
    (ValueError, "multiple", {"q": lambda z: z(2, 1, 5, 64)}),
    (ValueError, "cu_seqlens", {"q": lambda z: z(2, 4, 64), "cu_seqlens": lambda z: z(2, dtype=torch.int32),
                                "max_seqlen": 1}),
    (ValueError, "max_seqlen", {"q": lambda z: z(2, 4, 64), "cu_seqlens": lambda z: z(3, dtype=torch.int32)}),
    (ValueError, "less than", {"q": lambda z: z(2, 3, 4, 64), "max_seqlen": 2}),
    (TypeError, "bfloat16 or float32", {"q": lambda z: z(2, 1, 4, 64, dtype=torch.float16)}),
    (RuntimeError, "64 query heads", {"q": lambda z: z(2, 1, 130, 64)}),
    (RuntimeError, "at most 256", {"q": lambda z: z(2, 1, 4, 264), "k_pages": lambda z: z(4, 16, 2, 264),
                                   "v_pages": lambda z: z(4, 16, 2, 264)}),
    (NotImplementedError, "forward-only", {"q": lambda z: z(2, 1, 4, 64).requires_grad_()}),
])
def test_attention_refuses_before_launching(error, words, kw):
    args = _attention_args(**kw)
    with pytest.raises(error, match=words):
        _op()(args.pop("q"), args.pop("k_pages"), args.pop("v_pages"), **args)


def test_same_bits_again_and_on_two_streams():
    """A call gives the same bits each time, also with another at work on another stream."""
    g = torch.Generator().manual_seed(8)
    cases = []
    for dtype, D, T in ((BF, 128, 1), (BF, 128, 100), (F32, 64, 1), (BF, 64, 30)):
        pool = Pool([1500 + T, 30 + T], 16, 2, D, dtype, stale=0.0)
        q = randn(g, 2, T, 8, D, dtype=dtype).to(DEV)
        kg, vg, table, pos = pool.k.to(DEV), pool.v.to(DEV), pool.table.to(DEV), i32([1500, 30])
        cases.append(lambda q=q, kg=kg, vg=vg, table=table, pos=pos: _op()(
            q, kg, vg, block_table=table, cache_seqlens=pos, causal=True))
    want = [c() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[] for _ in cases]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cases[i]())
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        for y in ys:
            assert torch.equal(w, y)


# -----------------------------------------------------------------------------------------------
# Pages and slots
# -----------------------------------------------------------------------------------------------
def _plan_state(lens, width, page, spare, seed=0):
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lens]
    order = torch.randperm(sum(held) + spare, generator=g).tolist()
    table = [[-1] * width for _ in lens]
    for b, h in enumerate(held):
        for i in range(h):
            table[b][i] = order.pop()
    return table, order + [-7] * sum(held), [len(order)]


def _check_plan(lens, new, width, page, spare, total=None, done=(), seed=0):
    from modelcore_amd.kernels.paged import paged_release, paged_reserve
    table, free, count = _plan_state(lens, width, page, spare, seed)
    dt = torch.tensor(table, dtype=torch.int32).reshape(len(lens), width).to(DEV)
    dl, df, dc = i32(lens), i32(free), i32(count)
    lens = list(lens)
    if done:
        paged_release(dt, dl, i32(list(done)), df, dc, page_size=page)
        release(table, lens, done, free, count, page)
        assert dt.tolist() == table and dl.tolist() == lens
        assert dc.tolist() == count and df.tolist()[:count[0]] == free[:count[0]]
    total = sum(new) if total is None else total
    plan = paged_reserve(dt, dl, i32(new), df, dc, total=total, page_size=page)
    slots, positions, cu, refused = reserve(table, lens, new, free, count, total, page)
    assert plan.slots.tolist() == slots and plan.positions.tolist() == positions
    assert plan.cu_seqlens.tolist() == cu and plan.refused.tolist() == [refused]
    assert dt.tolist() == table and dc.tolist() == count and dl.tolist() == lens
    assert plan.slots.dtype == torch.int64


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("rows", [1, 3, 64, 1023, 1025, 2500])
def test_reserve_single_tokens(rows, page):
    _check_plan([(b * 7) % 100 for b in range(rows)], [1] * rows, 8, page, rows + 5)


@pytest.mark.parametrize("hi", [3, 17, 700, 5000])
def test_reserve_mixed_lengths(hi):
    """Totals on both sides of one launch's tokens, rows without new tokens, rows that have ended."""
    lens = [(b * 37) % (hi + 1) for b in range(40)]
    new = [(b * 91) % (hi + 1) if b % 3 else 0 for b in range(40)]
    _check_plan(lens, new, 2 * hi // 16 + 3, 16, sum(new) // 16 + 41)
    _check_plan(lens, new, 2 * hi // 16 + 3, 16, sum(new) // 16 + 41, done=[3, 39, 0, 17])


def test_reserve_refuses_rows_one_by_one():
    _check_plan([0, 16, 5, 30, 0], [40, 1, 3, 40, 20], 6, 16, 4)   # the stack runs out
    _check_plan([0, 90, 5, 0], [40, 10, 3, 97], 6, 16, 40)        # a line of the table is full
    _check_plan([0, 10, 0], [1, 1, 1], 4, 16, 0)                  # nothing is free
    _check_plan([4, 20], [5, 20], 4, 16, 9, total=12)             # tokens past the total
    _check_plan([4, 20], [5, 20], 4, 16, 9, total=40)             # and a total past the tokens
    _check_plan([4, 20, 3], [0, 0, 0], 4, 16, 9, total=0)
    _check_plan([], [], 1, 16, 3, total=0)
    from modelcore_amd.kernels.paged import paged_reserve
    table, count = torch.full((3, 4), -1, dtype=torch.int32, device=DEV), i32([8])
    plan = paged_reserve(table, i32([-1, 0, 2 ** 31 - 1]), i32([3, -4, 2]), i32(list(range(8))), count,
                         total=5, page_size=16)
    assert plan.refused.tolist() == [3] and plan.slots.tolist() == [-1] * 5
    assert plan.cu_seqlens.tolist() == [0, 3, 3, 5] and count.tolist() == [8]
    assert (table == -1).all()


def test_release_rows_twice_and_outside():
    _check_plan([50, 3, 0, 64], [1, 1, 1, 1], 6, 16, 4, done=[0, 2])
    from modelcore_amd.kernels.paged import paged_release
    table, free, count = _plan_state([50, 20, 0, 64], 6, 16, 2)
    dt, dl, df, dc = i32(table), i32([50, 20, 0, 64]), i32(free), i32(count)
    paged_release(dt, dl, i32([1, 1, -3, 4, 2, 1000]), df, dc, page_size=16)
    assert dl.tolist() == [50, 0, 0, 64] and dc.tolist() == [count[0] + 2]
    assert df.tolist()[count[0]:count[0] + 2] == table[1][:2] and dt[1].tolist() == [-1] * 6
    paged_release(dt, dl, i32([]), df, dc, page_size=16)
    assert dc.tolist() == [count[0] + 2]


def test_rows_named_twice_give_their_pages_where_named_first():
    """Whichever wave comes first: the stack is the same every time, for names a few and a thousand apart."""
    from modelcore_amd.kernels.paged import paged_release
    n = 900
    lens = [16 + b % 40 for b in range(n)]
    g = torch.Generator().manual_seed(12)
    once = torch.randperm(n, generator=g).tolist()
    for names in (once[:70] + once[:70] + once[60:130], once + once[::-1] + once,
                  [x for b in once[:300] for x in (b, b, b)]):
        table, free, count = _plan_state(lens, 4, 16, 3)
        dt, dl, df, dc = i32(table), i32(lens), i32(free), i32(count)
        paged_release(dt, dl, i32(names), df, dc, page_size=16)
        held = list(lens)
        release(table, held, names, free, count, 16)
        assert dt.tolist() == table and dl.tolist() == held and dc.tolist() == count
        assert df.tolist()[:count[0]] == free[:count[0]]


@pytest.mark.parametrize("rows", [1024, 1025])
def test_reserve_more_tokens_than_one_launch_takes(rows):
    _check_plan([(7 * b) % 100 for b in range(rows)], [(0, 3, 11, 0, 1)[b % 5] * 2 for b in range(rows)], 10, 16,
                2 * rows)


def test_pages_change_hands_without_loss():
    """Forty rounds of rows that end and start anew: every page is free or held once."""
    from modelcore_amd.kernels.paged import paged_release, paged_reserve
    g = torch.Generator().manual_seed(2)
    n, width, page, pages = 70, 9, 16, 400
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    lens, free, count = i32([0] * n), i32(list(range(pages))), i32([pages])
    h_table, h_lens = [[-1] * width for _ in range(n)], [0] * n
    h_free, h_count = list(range(pages)), [pages]
    for _ in range(40):
        done = torch.randperm(n, generator=g)[:9].tolist()
        new = torch.randint(0, 40, (n,), generator=g).tolist()
        paged_release(table, lens, i32(done), free, count, page_size=page)
        release(h_table, h_lens, done, h_free, h_count, page)
        plan = paged_reserve(table, lens, i32(new), free, count, total=sum(new), page_size=page)
        slots, positions, _, refused = reserve(h_table, h_lens, new, h_free, h_count, sum(new), page)
        assert plan.slots.tolist() == slots and plan.refused.tolist() == [refused]
        at = 0
        for b, t in enumerate(new):  # rows that were given their pages move on
            if t and slots[at] >= 0:
                h_lens[b] += t
            at += t
        lens.copy_(i32(h_lens))
        held = [p for line in table.tolist() for p in line if p >= 0]
        assert sorted(held + free.tolist()[:h_count[0]]) == list(range(pages))
        assert table.tolist() == h_table and count.tolist() == h_count


# -----------------------------------------------------------------------------------------------
# The pre-attention step
# -----------------------------------------------------------------------------------------------
def _step(tokens, H, H_kv, D, dtype, page=16, n_pos=200, seed=0, with_kv=True):
    from modelcore_amd.kernels.qk_epilogue import default_eps, rope_norm_scale_append_paged
    g = torch.Generator().manual_seed(seed)
    n_pages = tokens // page + 4
    slots = torch.randperm(n_pages * page, generator=g)[:tokens]
    pos = torch.randint(0, n_pos, (tokens,), generator=g).int()
    if tokens > 4:
        slots[2], slots[3], pos[1], pos[4] = -1, n_pages * page, -1, n_pos
    cos, sin = randn(g, n_pos, D // 2, dtype=dtype), randn(g, n_pos, D // 2, dtype=dtype)
    qkv = randn(g, tokens, H + 2 * H_kv, D, dtype=dtype)
    kp, vp = randn(g, n_pages, page, H_kv, D, dtype=dtype), randn(g, n_pages, page, H_kv, D, dtype=dtype)
    kg, vg, dq = kp.to(DEV), vp.to(DEV), qkv.to(DEV)
    kv = (dq[:, H:H + H_kv], dq[:, H + H_kv:], kg, vg, slots.to(DEV)) if with_kv else ()
    q = rope_norm_scale_append_paged(dq[:, :H], cos.to(DEV), sin.to(DEV), pos.to(DEV), *kv, scale=1.2)
    ok = (pos >= 0) & (pos < n_pos)
    at = pos.clamp(0, n_pos - 1).long()
    # Angles of any size: fp32 all through, the terms of a rotation at most twice its result's norm, so
    # an element is off by its own rounding and by (D + 8) 2^-24 of the head's norm, scaled.
    want = rotated(qkv[:, :H + H_kv], cos[at], sin[at], default_eps(), 1.2)
    size = (cos[at].double().abs() + sin[at].double().abs()).amax(1)[:, None, None] * \
        qkv[:, :H + H_kv].double().square().sum(-1, keepdim=True).sqrt()
    raw = (want / 1.2).abs().amax()  # noqa: F841
    half = D // 2
    x = qkv[:, :H + H_kv].double()
    y = torch.cat([x[..., :half] * cos[at].double()[:, None] + x[..., half:] * sin[at].double()[:, None],
                   x[..., half:] * cos[at].double()[:, None] - x[..., :half] * sin[at].double()[:, None]], -1)
    rms = (y.square().mean(-1, keepdim=True) + default_eps()).sqrt()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (D + 8) * 2.0 ** -24 * (1.2 * 2 * size / rms + want.abs())
    close(q.cpu()[ok], want[:, :H][ok], tol[:, :H][ok], "q")
    assert q.cpu()[~ok].isnan().all()
    if not with_kv:
        return
    rows_k, rows_v = kp.view(-1, H_kv, D).clone(), vp.view(-1, H_kv, D).clone()
    got_k, got_v = kg.cpu().view(-1, H_kv, D), vg.cpu().view(-1, H_kv, D)
    for i in range(tokens):
        if bool(ok[i]) and 0 <= int(slots[i]) < n_pages * page:
            close(got_k[slots[i]], want[i, H:], tol[i, H:], f"k {i}")
            rows_k[slots[i]] = got_k[slots[i]]
            rows_v[slots[i]] = qkv[i, H + H_kv:]
    assert same_bits(got_k, rows_k) and same_bits(got_v, rows_v)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,H_kv,D", [(12, 12, 64), (32, 8, 128), (8, 2, 256), (3, 1, 96), (4, 4, 32), (2, 1, 16),
                                      (5, 5, 24), (1, 1, 2), (6, 2, 200), (7, 7, 250)])
def test_step(H, H_kv, D, dtype):
    _step(37, H, H_kv, D, dtype, seed=D)
    _step(1, H, H_kv, D, dtype, seed=D + 1)
    _step(9, H, H_kv, D, dtype, seed=D + 2, with_kv=False)


def test_step_of_many_tokens():
    _step(3000, 4, 2, 64, BF, page=64)


def test_step_copies_values_bit_for_bit():
    """Every bf16 there is, signalling NaNs among them, goes into the pages as it is."""
    from modelcore_amd.kernels.qk_epilogue import rope_norm_scale_append_paged
    v = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(BF).view(512, 1, 128)
    k = torch.ones(512, 1, 128, dtype=BF)
    kp, vp = torch.zeros(32, 16, 1, 128, dtype=BF, device=DEV), torch.zeros(32, 16, 1, 128, dtype=BF, device=DEV)
    cos, sin = torch.ones(4, 64, dtype=BF, device=DEV), torch.zeros(4, 64, dtype=BF, device=DEV)
    rope_norm_scale_append_paged(k.to(DEV), cos, sin, i32([1] * 512), k.to(DEV), v.to(DEV), kp, vp,
                                 torch.arange(512, device=DEV))
    assert same_bits(vp.view(512, 1, 128), v)
