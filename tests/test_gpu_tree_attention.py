"""Attention of drafted trees over a paged cache, on the GPU against a plain form in 64 bits."""
import random

import pytest
import torch

import _tree
from _paged import Pool
from modelcore_amd import _ext
from modelcore_amd.kernels import flash_attn as fa
from modelcore_amd.kernels.flash_attn import flash_attn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def op(*a, **kw):
    return flash_attn.flash_attn_paged_tree_with_kvcache(*a, **kw)


def same_bits(a, b):
    view = {BF: torch.int16, F32: torch.int32}[a.dtype]
    return torch.equal(a.cpu().contiguous().view(view), b.cpu().contiguous().view(view))


class Call:
    """Rows at `pos` with trees of bits[b][i] (node numbers that node i of row b may see)."""

    def __init__(self, pos, bits, H, H_kv, D, page, dtype, window=-1, words=None, append=True, seed=0, stale=NAN,
                 pad=0, packed=None, max_pages=None):
        g = torch.Generator().manual_seed(seed + 1)
        new = [len(x) for x in bits]
        self.pos, self.bits, self.window, self.new = pos, bits, window, new
        self.H, self.D = H, D
        self.pool = pool = Pool([p + t for p, t in zip(pos, new)], page, H_kv, D, dtype, seed=seed, stale=stale,
                                max_pages=max_pages)
        n = sum(new) + pad
        self.q = torch.randn(n, H, D, generator=g).to(dtype)
        self.k, self.v = (torch.randn(n, H_kv, D, generator=g).to(dtype) for _ in range(2))
        words = words or max(1, -(-max(new) // 64))
        masks = [_tree.words_of(nodes, words) for row in bits for nodes in row] + [[-1] * words] * pad
        self.masks = torch.tensor(masks, dtype=torch.int64, device=DEV).view(n, words)
        self.packed = packed if packed is not None else len(set(new)) > 1 or pad > 0
        self.append = append
        cu = [0]
        for t in new:
            cu.append(cu[-1] + t)
        self.cu = cu

    def place_new(self):
        """The new tokens' keys and values in the pool on the CPU; what it holds there before the call."""
        kp, vp = self.pool.k.clone(), self.pool.v.clone()
        for b, (p, t) in enumerate(zip(self.pos, self.new)):
            for i in range(t):
                where = self.pool.place(b, p + i)
                if self.append:
                    kp[where], vp[where] = NAN, NAN
                    self.pool.k[where], self.pool.v[where] = self.k[self.cu[b] + i], self.v[self.cu[b] + i]
        return kp.to(DEV), vp.to(DEV)

    def run(self, check_pages=True):
        kg, vg = self.place_new()
        n = len(self.q)
        shape = (n,) if self.packed else (len(self.pos), self.new[0])
        kw = {"cu_seqlens": i32(self.cu), "max_seqlen": max(self.new)} if self.packed else {}
        if self.append:
            kw.update(k=self.k.to(DEV).view(*shape, *self.k.shape[1:]), v=self.v.to(DEV).view(*shape, *self.v.shape[1:]))
        y = op(self.q.to(DEV).view(*shape, self.H, self.D), kg, vg, tree_masks=self.masks.view(*shape, -1),
               block_table=self.pool.table.to(DEV), cache_seqlens=i32(self.pos), window_size=(self.window, 0), **kw)
        torch.cuda.synchronize()
        if check_pages:
            assert same_bits(kg, self.pool.k) and same_bits(vg, self.pool.v), "the pages"
        return y.view(n, self.H, self.D).cpu()

    def check(self, y=None, rows=None):
        y = self.run() if y is None else y
        for b, (p, t) in enumerate(zip(self.pos, self.new)):
            if t == 0 or (rows is not None and b not in rows):
                continue
            kk, vv = self.pool.rows(b, p + t)
            for i in range(t):
                seen = _tree.seen_keys(p, i, self.bits[b][i], self.window)
                want, tol = _tree.attend(self.q[self.cu[b] + i], kk, vv, seen)
                off = (y[self.cu[b] + i].double() - want).abs()
                bad = ~(off <= tol)
                bad &= ~(want.isnan() & y[self.cu[b] + i].isnan())
                assert not bad.any(), f"row {b} node {i}: {int(bad.sum())} off, worst {float((off - tol)[bad].max()):.3e} past"


def trees(rng, sizes):
    return [_tree.ancestors(_tree.random_parents(rng, n)) for n in sizes]


HEADS = [(1, 1, 64), (12, 12, 64), (16, 4, 128), (32, 8, 128), (6, 2, 96), (8, 8, 256), (5, 1, 40), (24, 2, 128),
         (64, 1, 128), (3, 3, 32), (4, 2, 8), (20, 2, 192)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,H_kv,D", HEADS)
def test_trees(H, H_kv, D, dtype):
    rng = random.Random(H * 1000 + D)
    Call([0, 37, 128, 1], trees(rng, [9, 1, 33, 4]), H, H_kv, D, 32, dtype).check()


@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 16, 31, 32, 33, 63, 64, 65, 70, 128, 129, 200])
def test_sizes(T):
    """Few pairs and many, trees that end on and beside a word, in rows of any place within tiles and pages."""
    rng = random.Random(T)
    Call([0, 61, 130], trees(rng, [T] * 3), 8, 2, 128, 16, BF).check()
    Call([5, 64], trees(rng, [T] * 2), 4, 4, 64, 64, F32).check()


def test_the_widest_tree():
    rng = random.Random(1)
    call = Call([100, 3], trees(rng, [1024, 700]), 2, 1, 64, 64, BF)
    call.check()
    Call([40], [[[i] if i < 5 else [i - 5, i] for i in range(1024)]], 1, 1, 128, 128, BF, window=3).check()


@pytest.mark.parametrize("window", [0, 1, 2, 5, 15, 16, 40, 100])
@pytest.mark.parametrize("page", [16, 64])
def test_windows(page, window):
    """Windows that end among the ancestors, at the row's last tokens and far before them."""
    rng = random.Random(window)
    Call([0, 31, 95, 257, 300], trees(rng, [12] * 5), 8, 2, 128, page, BF, window).check()
    chain = [list(range(i + 1)) for i in range(70)]
    Call([0, 33, 200], [chain, chain[:9], chain[:64]], 4, 1, 128, page, BF, window).check()
    Call([5, 90], [chain[:40], chain[:3]], 4, 2, 64, page, F32, window).check()
    Call([5, 90], [chain[:40], chain[:3]], 4, 2, 96, page, BF, window).check()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("window", [-1, 0, 3])
@pytest.mark.parametrize("D", [64, 128])
def test_any_bits(D, window, dtype):
    """Masks that are no ancestors: nodes without a bit, which stand before the row's next position and, in a row
    without tokens, see nothing; bits past the node's own, which do not count; nodes that miss themselves."""
    rng = random.Random(D + window)
    for sizes in ([3, 5], [40, 30, 20], [100]):
        bits = [[[] if i in (0, n - 2) else sorted(rng.sample(range(n), rng.randrange(n))) for i in range(n)]
                for n in sizes]
        Call([0, 50, 7][:len(sizes)], bits, 4, 1, D, 16, dtype, window).check()


def test_a_node_that_sees_nothing_is_zero():
    for T in (1, 3, 40):
        call = Call([0, 0], [[[]] * T, [[0]] * T], 4, 1, 128, 16, BF)
        y = call.run()
        assert bool((y[:T] == 0).all())
        call.check(y)


def test_a_chain_is_a_sequence():
    """The tree of one chain sees what the operator of sequences sees."""
    for T, H, H_kv, D, dtype in ((5, 8, 2, 128, BF), (64, 32, 8, 128, BF), (40, 12, 12, 64, F32)):
        call = Call([100, 333], [[list(range(i + 1)) for i in range(T)]] * 2, H, H_kv, D, 16, dtype)
        y = call.run()
        call.check(y)
        kg, vg = call.pool.k.to(DEV), call.pool.v.to(DEV)
        x = flash_attn.flash_attn_paged_with_kvcache(call.q.to(DEV).view(2, T, H, D), kg, vg, block_table=call.pool.table.to(DEV),
                                                     cache_seqlens=i32(call.pos))
        call.check(x.view(-1, H, D).cpu())


def test_layouts_and_long_rows():
    """Rows without nodes, tokens past the last row's, keys cut into ranges, pages already written."""
    rng = random.Random(4)
    Call([3000, 40, 2047], trees(rng, [16, 0, 5]), 16, 4, 128, 16, BF, pad=4).check()
    Call([4100], trees(rng, [64]), 32, 8, 128, 64, BF, max_pages=200).check()
    Call([2500, 1800], trees(rng, [30, 30]), 4, 2, 64, 32, BF, append=False).check()
    Call([2500], trees(rng, [20]), 4, 4, 64, 32, F32).check()
    Call([1500, 900], trees(rng, [20, 3]), 4, 2, 256, 32, BF, window=800).check()


def test_tokens_past_the_last_row_are_left():
    rng = random.Random(9)
    call = Call([30], trees(rng, [5]), 4, 2, 128, 16, BF, pad=3)
    kg, vg = call.place_new()
    out = []
    real = torch.empty_like

    def marked(t, **kw):
        y = real(t, **kw)
        if t.shape == call.q.shape:
            out.append(y.fill_(7.0))
        return y

    torch.empty_like = marked
    try:
        y = op(call.q.to(DEV), kg, vg, k=call.k.to(DEV), v=call.v.to(DEV), tree_masks=call.masks,
               block_table=call.pool.table.to(DEV), cache_seqlens=i32([30]), cu_seqlens=i32(call.cu), max_seqlen=5)
    finally:
        torch.empty_like = real
    assert out and bool((y[5:] == 7.0).all())
    call.check(y.cpu())


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("T,H,H_kv,D,dtype", [(6, 8, 2, 128, BF), (40, 8, 1, 128, BF), (70, 8, 2, 64, BF), (9, 4, 4, 64, F32),
                                              (50, 4, 2, 128, F32)])
def test_what_is_hidden_does_not_reach_a_node(T, H, H_kv, D, dtype, bad):
    """Infinities and NaN in the keys and values of nodes reach those below them and nobody else."""
    rng = random.Random(T)
    parents = [-1] + [rng.randrange(max(0, i - 4), i) for i in range(1, T)]
    seen = _tree.ancestors(parents)
    for which in ("k", "v"):
        call = Call([70, 20], [seen, seen], H, H_kv, D, 16, dtype)
        hit = T - 3
        getattr(call, which)[hit] = bad  # of row 0
        y = call.run()
        for i in range(T):
            if hit in seen[i]:
                assert not bool(torch.isfinite(y[i]).all()), i
                if which == "v" and bad == bad:
                    want = torch.full_like(y[i], bad)
                    assert torch.equal(y[i], want), i
            else:
                assert bool(torch.isfinite(y[i]).all()), i
        call.bits[0] = [s if hit not in s else [] for s in seen]
        keep = [i for i in range(T) if hit not in seen[i]]
        kk, vv = call.pool.rows(0, 70 + T)
        for i in keep:
            want, tol = _tree.attend(call.q[i], kk, vv, _tree.seen_keys(70, i, seen[i], -1))
            assert bool(((y[i].double() - want).abs() <= tol).all()), i
        call.check(y, rows=[1])


def test_rows_that_do_not_fit_and_pages_outside_the_pool():
    rng = random.Random(2)
    for T, H, H_kv, D, dtype in ((5, 8, 2, 128, BF), (40, 8, 1, 128, BF), (40, 4, 2, 64, F32), (1, 4, 2, 64, F32)):
        call = Call([40, 60, 90], trees(rng, [T] * 3), H, H_kv, D, 16, dtype)
        kg, vg = call.place_new()
        table = call.pool.table.clone()
        table[1, 1] = 10 ** 6  # tokens 16 .. 31 of row 1
        pos = i32([40, 60, table.shape[1] * 16 - T + 1])
        y = op(call.q.to(DEV).view(3, T, H, D), kg, vg, k=call.k.to(DEV).view(3, T, H_kv, D), v=call.v.to(DEV).view(3, T, H_kv, D),
               tree_masks=call.masks.view(3, T, -1), block_table=table.to(DEV), cache_seqlens=pos)
        y = y.view(-1, H, D).cpu()
        assert bool(y[T:].isnan().all())
        call.check(y, rows=[0])
        # Behind a window that hides the lost page, the row is as it should be.
        y = op(call.q.to(DEV).view(3, T, H, D), kg, vg, k=call.k.to(DEV).view(3, T, H_kv, D), v=call.v.to(DEV).view(3, T, H_kv, D),
               tree_masks=call.masks.view(3, T, -1), block_table=table.to(DEV), cache_seqlens=i32([40, 60, 90]), window_size=(20, 0))
        call.window = 20
        call.check(y.view(-1, H, D).cpu())


def test_checked_mode_names_what_is_wrong():
    call = Call([40], [[[0], [0, 1]]], 4, 2, 64, 16, BF)
    kg, vg = call.place_new()
    kw = dict(tree_masks=call.masks.view(1, 2, 1), cache_seqlens=i32([40]))
    q = call.q.to(DEV).view(1, 2, 4, 64)
    table = call.pool.table.clone()
    fa.set_checked(True)
    try:
        op(q, kg, vg, block_table=table.to(DEV), **kw)
        table[0, 1] = -1
        with pytest.raises(IndexError, match="tree_with_kvcache: page -1"):
            op(q, kg, vg, block_table=table.to(DEV), **kw)
        with pytest.raises(IndexError, match="fall"):
            op(q, kg, vg, block_table=table[:, :2].contiguous().to(DEV), **kw)
    finally:
        fa.set_checked(False)


def test_strided_tables_masks_and_other_streams():
    """A block table and masks that are views, queries that are, and a stream of the caller's."""
    rng = random.Random(6)
    call = Call([33, 70], trees(rng, [9, 9]), 8, 2, 128, 16, BF)
    kg, vg = call.place_new()
    table = torch.full((2, call.pool.table.shape[1] + 5), 77, dtype=torch.int32, device=DEV)
    table[:, :-5] = call.pool.table.to(DEV)
    masks = torch.stack([call.masks.view(2, 9, 1), ~call.masks.view(2, 9, 1)], -1)[..., 0]
    q = torch.cat([call.q.to(DEV).view(2, 9, 8, 128)] * 2, -1)[..., :128]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = op(q, kg, vg, k=call.k.to(DEV).view(2, 9, 2, 128), v=call.v.to(DEV).view(2, 9, 2, 128), tree_masks=masks,
               block_table=table[:, :-5], cache_seqlens=i32([33, 70]))
    side.synchronize()
    call.check(y.view(-1, 8, 128).cpu())
    assert same_bits(kg, call.pool.k) and same_bits(vg, call.pool.v)


def test_captured_and_replayed():
    """A captured call follows the tables, masks and lengths that it is replayed on."""
    rng = random.Random(8)
    calls = [Call([300, 1000], trees(rng, [20, 20]), 16, 4, 128, 16, BF, seed=s, max_pages=80) for s in range(3)]
    calls += [Call([500, 20], trees(rng, [20, 20]), 16, 4, 128, 16, BF, seed=5, max_pages=80)]
    n_pages = max(c.pool.n_pages for c in calls)
    pools = [torch.zeros(n_pages, 16, 4, 128, dtype=BF, device=DEV) for _ in range(2)]
    first = calls[0]
    args = dict(q=first.q.to(DEV), k=first.k.to(DEV), v=first.v.to(DEV), masks=first.masks.clone(),
                table=first.pool.table.to(DEV), pos=i32(first.pos))

    def body():
        return op(args["q"].view(2, 20, 16, 128), *pools, k=args["k"].view(2, 20, 4, 128), v=args["v"].view(2, 20, 4, 128),
                  tree_masks=args["masks"].view(2, 20, 1), block_table=args["table"], cache_seqlens=args["pos"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = body()
    for call in (*calls, calls[0]):
        kg, vg = call.place_new()
        pools[0][:len(kg)].copy_(kg), pools[1][:len(vg)].copy_(vg)
        for name, x in (("q", call.q), ("k", call.k), ("v", call.v), ("masks", call.masks), ("table", call.pool.table),
                        ("pos", i32(call.pos))):
            args[name].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        call.check(out.view(-1, 16, 128).cpu())


def test_the_same_call_gives_the_same_bits():
    rng = random.Random(3)
    call = Call([3000, 500, 20], trees(rng, [30, 16, 3]), 16, 4, 128, 16, BF)
    y = call.run()
    for _ in range(3):
        assert same_bits(call.run(), y)


@pytest.mark.parametrize("seed", range(12))
def test_at_random(seed):
    rng = random.Random(100 + seed)
    H, H_kv, D = rng.choice(HEADS)
    rows = rng.randrange(1, 6)
    sizes = [rng.choice([0, 1, rng.randrange(1, 12), rng.randrange(1, 90)]) for _ in range(rows)]
    if max(sizes) == 0:
        sizes[0] = 1
    pos = [rng.choice([0, rng.randrange(40), rng.randrange(700)]) for _ in range(rows)]
    Call(pos, trees(rng, sizes), H, H_kv, D, rng.choice([16, 32, 128]), rng.choice([BF, BF, F32]),
         rng.choice([-1, -1, rng.randrange(60)]), seed=seed, pad=rng.choice([0, 2])).check()


@pytest.mark.parametrize("rows,T,H,H_kv,D,page,dtype", [
    (70, 20, 8, 2, 64, 16, BF), (150, 9, 8, 1, 128, 32, BF), (70, 9, 4, 2, 64, 16, F32),  # more rows than a wave has lanes
    (24, 40, 64, 32, 32, 16, BF), (9, 70, 64, 32, 64, 64, BF),  # more blocks than a KV head has workgroups
    (2, 40, 600, 600, 8, 16, BF), (2, 3, 520, 520, 8, 16, F32)])  # more KV heads than workgroups that fill the chip
def test_many_rows_blocks_and_heads(rows, T, H, H_kv, D, page, dtype):
    rng = random.Random(rows)
    sizes = [rng.choice([T, rng.randrange(1, T + 1)]) for _ in range(rows)]
    pos = [rng.choice([0, rng.randrange(30), rng.randrange(500 if rows < 30 and H_kv < 100 else 120)]) for _ in range(rows)]
    Call(pos, trees(rng, sizes), H, H_kv, D, page, dtype, max_pages=2048 // page).check()


@pytest.mark.parametrize("window", [-1, 0, 7, 63, 64, 200, 900])
@pytest.mark.parametrize("T,H,H_kv,D,dtype", [(60, 8, 2, 128, BF), (60, 4, 2, 256, BF), (30, 8, 4, 96, BF), (60, 4, 2, 64, F32)])
def test_windows_of_wide_trees_over_ranges(T, H, H_kv, D, dtype, window):
    """Windows that begin in any range of a cut row, and before the first key of a tile."""
    rng = random.Random(window)
    chain = [list(range(i + 1)) for i in range(T)]
    bits = [chain, *trees(rng, [T, T // 2]), chain]
    Call([0, 255, 1000, 1290], bits, H, H_kv, D, 64, dtype, window, max_pages=64).check()


@pytest.mark.parametrize("T,H,H_kv,D,dtype", [(3, 8, 2, 128, BF), (16, 16, 4, 128, BF), (40, 16, 4, 64, BF), (20, 4, 4, 64, F32)])
def test_without_scratch(T, H, H_kv, D, dtype):
    """No scratch, or too little of it, cuts no row; the outputs are of the same kind."""
    rng = random.Random(T)
    call = Call([900, 100], trees(rng, [T, T]), H, H_kv, D, 16, dtype, max_pages=128)
    lib, code = _ext.lib(), _ext.dtype_code(dtype)
    table, pos = call.pool.table.to(DEV), i32(call.pos)
    q, k, v = (t.to(DEV) for t in (call.q, call.k, call.v))
    need = lib.mcamd_paged_tree_scratch_bytes(2, 2 * T, T, H, H_kv, D, 128, 16, -1, code)
    assert need > 0
    for nbytes in (0, need - 1):
        kg, vg = call.place_new()
        y = torch.full_like(q, NAN)
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=DEV)
        st = lib.mcamd_flash_attn_paged_tree_with_kvcache(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), kg.data_ptr(), vg.data_ptr(), table.data_ptr(), 128, pos.data_ptr(), None,
            call.masks.data_ptr(), call.masks.shape[-1], y.data_ptr(), 2, 2 * T, T, H, H_kv, D, call.pool.n_pages, 16,
            16 * H_kv * D, 128, -1, code, ws.data_ptr() if nbytes else None, nbytes, _ext.stream_handle(y.device))
        _ext.check(st, "tree attention")
        torch.cuda.synchronize()
        call.check(y.cpu())
        assert same_bits(kg, call.pool.k) and same_bits(vg, call.pool.v)


def test_two_streams_at_once():
    """Calls that run beside each other on two streams have their own scratch."""
    rng = random.Random(12)
    calls = [Call([2500, 700], trees(rng, [16, 16]), 16, 4, 128, 16, BF, seed=s) for s in range(2)]
    ready = []
    for c in calls:
        kg, vg = c.place_new()
        ready.append((c.q.to(DEV).view(2, 16, 16, 128), kg, vg, dict(
            k=c.k.to(DEV).view(2, 16, 4, 128), v=c.v.to(DEV).view(2, 16, 4, 128), tree_masks=c.masks.view(2, 16, 1),
            block_table=c.pool.table.to(DEV), cache_seqlens=i32(c.pos))))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    out = [[], []]
    for _ in range(10):
        for i, (q, kg, vg, kw) in enumerate(ready):
            with torch.cuda.stream(streams[i]):
                out[i].append(op(q, kg, vg, **kw))
    torch.cuda.synchronize()
    for c, ys in zip(calls, out):
        c.check(ys[0].view(-1, 16, 128).cpu())
        assert all(same_bits(y, ys[0]) for y in ys)
