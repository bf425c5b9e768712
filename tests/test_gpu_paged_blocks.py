"""Paged attention whose blocks are cut in two, for each kernel that does it, and bf16 rows whose weights are
two terms, against the 64-bit form with the bound that counts the terms."""
import pytest
import torch

from _paged import Pool
from _paged_blocks import Rules, attend, close, rounds_weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Call:
    """Packed rows of (tokens, position), their pools and queries; `lost` rows lie outside their lines."""

    def __init__(self, rows, H, H_kv, D, dtype, page=16, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.H, self.H_kv, self.D, self.dtype, self.page = rows, H, H_kv, D, dtype, page
        self.pool = Pool([s + t for t, s in rows], page, H_kv, D, dtype, seed=seed, stale=1.0)
        n = sum(t for t, _ in rows)
        self.q, self.k, self.v = (torch.randn(n, h, D, generator=g).to(dtype) for h in (H, H_kv, H_kv))
        self.cu = [0]
        for t, _ in rows:
            self.cu.append(self.cu[-1] + t)

    def rules(self, rows=None):
        return Rules(rows or self.rows, self.H, self.H_kv, self.D, self.dtype,
                     self.pool.table.shape[1] * self.page,
                     cus=torch.cuda.get_device_properties(0).multi_processor_count)

    def run(self, append, pos=None):
        from modelcore_amd.kernels.flash_attn import flash_attn
        kp, vp = self.pool.k.clone(), self.pool.v.clone()
        for b, (t, s) in enumerate(self.rows):
            for i in range(t):
                where = self.pool.place(b, s + i)
                kp[where], vp[where] = (7, 7) if append else (self.k[self.cu[b] + i], self.v[self.cu[b] + i])
        self.kg, self.vg = kp.to(DEV), vp.to(DEV)
        kw = {"k": self.k.to(DEV), "v": self.v.to(DEV)} if append else {}
        return flash_attn.flash_attn_paged_with_kvcache(
            self.q.to(DEV), self.kg, self.vg, block_table=self.pool.table.to(DEV),
            cache_seqlens=i32([s for _, s in self.rows] if pos is None else pos), cu_seqlens=i32(self.cu),
            max_seqlen=max(t for t, _ in self.rows), causal=True, **kw).cpu()

    def row(self, b):
        """K and V of row b, its new tokens included."""
        t, s = self.rows[b]
        k, v = self.pool.rows(b, s + t)
        k, v = k.clone(), v.clone()
        k[s:], v[s:] = self.k[self.cu[b]:self.cu[b + 1]], self.v[self.cu[b]:self.cu[b + 1]]
        return k, v

    def check(self, y, but=()):
        for b, (t, s) in enumerate(self.rows):
            if t == 0 or b in but:
                continue
            a, e = self.cu[b], self.cu[b + 1]
            want, tol = attend(self.q[a:e], *self.row(b), s)
            close(y[a:e], want, tol, f"row {b}: {t} at {s}")


def rows_that_halve(H, H_kv, D, dtype, tokens, deep, kernel=None, ks=None, singles=0):
    """Rows of `tokens` new tokens, dealt in turn, at positions up to `deep`, as many as leave room for some of
    their blocks to be cut in two, and single tokens between them."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    longs = []
    for n in range(1, 400):
        longs.append((tokens[n % len(tokens)], deep - (n * 137) % (deep // 2 + 1) if n % 3 else n % 20))
        rows = list(longs)
        for i in range(singles):
            rows.insert((i * 5) % (len(rows) + 1), (1, (i * 31) % deep))
        width = max(-(-(s + t) // 16) for t, s in rows) + 1  # of the table that Pool makes
        r = Rules(rows, H, H_kv, D, dtype, 16 * width, cus=cus)
        blocks = sum(r.blocks_of(t) for t, _ in rows)
        if r.slots and 0.55 * r.slots < blocks * H_kv < 0.95 * r.slots and (ks is None or r.ks == ks):
            return rows
    raise AssertionError("no such rows")


KINDS = [  # H, H_kv, D, dtype, tokens of long rows, deepest position, the kernel and its waves on the keys
    (32, 32, 128, BF, [40, 33, 64, 50], 1100, "ping-pong", None),
    (64, 16, 128, BF, [100, 37, 150], 900, "ping-pong", None),     # G = 4, blocks that end inside a token's heads
    (80, 16, 128, BF, [120, 60], 900, "ping-pong", None),          # G = 5
    (2, 2, 128, BF, [40, 33, 37], 800, "ping-pong", None),         # more than 64 rows
    (64, 32, 64, BF, [40, 30, 22], 900, "tiled", 1),
    (64, 32, 64, BF, [32, 32, 31], 900, "tiled", 4),
    (16, 8, 256, BF, [20, 70], 500, "tiled", 1),
    (48, 24, 40, BF, [40, 100], 1500, "tiled", 1),
    (32, 32, 64, F32, [40, 8, 130], 700, "tiled", 1),
    (32, 32, 64, F32, [64, 33], 700, "tiled", 4),
    (48, 16, 128, F32, [40, 9], 300, "tiled", 1),                  # G = 3
    (8, 4, 64, F32, [10, 3, 7], 300, "tiled", 1),                  # more than 64 rows
    (16, 8, 256, F32, [20, 5], 200, "tiled", 1),
]


@pytest.mark.parametrize("append", [True, False])
@pytest.mark.parametrize("H,H_kv,D,dtype,tokens,deep,kernel,ks", KINDS)
def test_blocks_that_are_halved(H, H_kv, D, dtype, tokens, deep, kernel, ks, append):
    """The deepest blocks of each kernel in two ranges, alone and beside single tokens; the replayed rule says
    that some are."""
    for singles, seed in ((0, 0), (9, 1)):
        if ks == 4 and singles:
            continue  # more rows turn to blocks of 128 pairs
        call = Call(rows_that_halve(H, H_kv, D, dtype, tokens, deep, kernel, ks, singles), H, H_kv, D, dtype, seed=seed)
        rules = call.rules()
        assert rules.kernel == kernel and (ks is None or rules.ks == ks)
        assert rules.check() > 0
        y = call.run(append)
        call.check(y)
        assert torch.equal(y, call.run(append))


@pytest.mark.parametrize("H,H_kv,D,dtype,tokens,deep,kernel,ks", [KINDS[0], KINDS[1], KINDS[4], KINDS[8]])
def test_halved_blocks_and_rows_outside_their_lines(H, H_kv, D, dtype, tokens, deep, kernel, ks):
    """Rows that do not fit count as blocks without keys: NaN, with the others as they should be."""
    rows = rows_that_halve(H, H_kv, D, dtype, tokens, deep, kernel, ks)
    call = Call(rows, H, H_kv, D, dtype)
    room = call.pool.table.shape[1] * 16
    out = sorted({1 % len(rows), len(rows) - 1})
    for lost in (2 ** 31 - 1, -1, -2 ** 31, room - min(t for t, _ in rows) + 1):
        pos = [lost if b in out else s for b, (_, s) in enumerate(rows)]
        assert call.rules([(t, p) for (t, _), p in zip(rows, pos)]).check() > 0
        y = call.run(False, pos)
        call.check(y, but=out)
        for b in out:
            assert y[call.cu[b]:call.cu[b + 1]].isnan().all()


def test_halved_blocks_in_a_captured_call():
    """The rows' positions move between replays, and with them which blocks are cut."""
    from modelcore_amd.kernels.flash_attn import flash_attn
    H, H_kv, D = 32, 32, 128
    call = Call(rows_that_halve(H, H_kv, D, BF, [40, 33, 64, 50], 1100), H, H_kv, D, BF)
    call.run(False)
    q, pos, cu, table = call.q.to(DEV), i32([0] * len(call.rows)), i32(call.cu), call.pool.table.to(DEV)
    room = [s for _, s in call.rows]

    def run():
        return flash_attn.flash_attn_paged_with_kvcache(q, call.kg, call.vg, block_table=table, cache_seqlens=pos,
                                                        cu_seqlens=cu, max_seqlen=64, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = run()
    halved = set()
    for i in range(5):
        at = [s if (b + i) % 5 else s // 3 for b, s in enumerate(room)]
        rules = call.rules([(t, p) for (t, _), p in zip(call.rows, at)])
        assert rules.check() > 0
        halved.add(tuple(x[:2] for x in rules.replay()[0] if x and x[2] == 1))
        pos.copy_(torch.tensor(at, dtype=torch.int32))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, run())
    assert len(halved) > 1


@pytest.mark.parametrize("H,H_kv,D,rows", [
    (16, 4, 128, [(1, 300), (1, 0), (8, 900), (5, 17)]),                # the streaming kernel, of one range and cut
    (16, 4, 128, [(1, 16000)]),
    (16, 4, 64, [(1, 700), (8, 30), (1, 4000)]),
    (64, 1, 128, [(1, 500), (1, 40)]),                                  # two blocks of pairs
    (4, 4, 256, [(1, 900), (32, 100)]),
    (10, 2, 96, [(6, 400), (1, 77)]),
    (8, 2, 64, [(67, 500), (40, 0), (130, 200)]),                       # the tiled one, whole
    (8, 2, 64, [(150, 1900)]),                                          # cut
    (6, 2, 96, [(70, 300), (1, 9), (33, 800)]),
    (4, 1, 256, [(200, 700), (20, 5)]),
    (12, 4, 40, [(90, 250)]),
])
def test_weights_in_two_terms(H, H_kv, D, rows):
    """bf16 rows of the streaming and the tiled kernels: closer than one rounding of the weights would be."""
    assert not any(rounds_weights(t, H // H_kv, D, BF) for t, _ in rows)
    call = Call(rows, H, H_kv, D, BF, seed=5)
    call.check(call.run(True))


@pytest.mark.parametrize("T", [1, 30, 300])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (F32, 64)])
def test_queries_before_a_lost_page(dtype, D, T):
    """A page outside the pool: queries that see none of its keys are what they should be."""
    call = Call([(T, 40), (T, 40)], 4, 2, D, dtype, seed=9)
    first = (40 + T // 2) // 16 * 16
    ok = max(0, first - 40)
    table = call.pool.table.clone()
    table[0, first // 16] = 2 ** 31 - 1
    from modelcore_amd.kernels.flash_attn import flash_attn
    call.run(True)  # the pages, whole
    y = flash_attn.flash_attn_paged_with_kvcache(
        call.q.to(DEV), call.kg, call.vg, block_table=table.to(DEV), cache_seqlens=i32([40, 40]),
        cu_seqlens=i32(call.cu), max_seqlen=T, causal=True).cpu()
    want, tol = attend(call.q[:T], *call.row(0), 40)
    close(y[:ok], want[:ok], tol[:ok])
    assert y[ok:T].isnan().all()
    want, tol = attend(call.q[T:], *call.row(1), 40)
    close(y[T:], want, tol)
