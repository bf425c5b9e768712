"""The paged attention's rules on the host: what a call's long rows are cut into, by the same sums as the
device's, and a 64-bit form whose bound counts what each kernel rounds.

The replay is for tests that need blocks cut in a certain way: it tells them whether their rows are, so
that a retuned constant cannot leave them without their subject."""
import math

import torch

MIN_RANGE_KEYS = 256   # of the ping-pong kernel's ranges
RANGE_US = 3.0         # of the tiled kernel's
SHORT_US = 30.0
MAX_SPLITS = 32


class Rules:
    """A packed call's long rows: (tokens, position) of every row, room in positions of a table line."""

    def __init__(self, rows, H, H_kv, D, dtype, room, window=-1, cus=256):
        self.rows, self.H_kv, self.G, self.room, self.cus = rows, H_kv, H // H_kv, room, cus
        self.total, self.t_new = sum(t for t, _ in rows), max(t for t, _ in rows)
        self.bf, self.D, self.window = dtype == torch.bfloat16, D, window
        self.skip = 32 if self.bf else 1
        self.kernel = "ping-pong" if self.bf and D == 128 else "tiled"
        if self.kernel == "ping-pong":
            self.pairs, self.kt = 256 // self.G * self.G, 64
            self.min_tiles = MIN_RANGE_KEYS // self.kt
            self.slots = self._slots(self.pairs, 1, MIN_RANGE_KEYS)
        else:
            self._tiled()
        self.halve = 2 * self.min_tiles * self.kt if window < 0 else 0

    def _few(self, t):
        return t == 1 or t * self.G <= self.skip

    def blocks_of(self, t):
        return 0 if self._few(t) else -(-t * self.G // self.pairs)

    def _keys(self):
        return self.room if self.window < 0 else min(self.room, self.window + 256 + 64)

    def _slots(self, pairs, per_cu, min_keys):
        least = self.total * self.G // pairs * self.H_kv
        return per_cu * self.cus if least <= per_cu * self.cus and self._keys() >= 2 * min_keys else 0

    def _tiled(self):
        def plan(ks):
            pairs, kt = 128 // ks, 128 if ks == 4 else 64 if self.bf and self.D <= 128 else 32
            us = self.D * ((0.027 if self.bf else 0.085) if ks == 4 else (0.012 if self.bf else 0.035))
            min_tiles = max(1, int(RANGE_US / us))
            shortest = max(self.skip // self.G, 1) + 1
            bound = self.total * self.G // pairs + min(self.total // shortest, len(self.rows))
            return ks, pairs, kt, us, min_tiles, bound, self._slots(pairs, 2 if self.D <= 128 else 1, min_tiles * kt)
        whole, four = plan(1), plan(4)
        fills = whole[5] * self.H_kv >= self.cus
        few = self.t_new * self.G <= 64
        brief = self._keys() / four[2] * four[3] <= SHORT_US
        take = four if self.D <= 128 and not fills and (few or brief or whole[6] == 0) else whole
        self.ks, self.pairs, self.kt, _, self.min_tiles, _, self.slots = take

    def _depth(self, t, s0, qt=None):
        if not 0 <= s0 <= self.room - t:
            return 0
        return s0 + (t if qt is None else min((qt + 1) * self.pairs // self.G, t))

    def _deeper(self, t, s0, blocks, keys):
        if blocks == 0 or self._depth(t, s0) <= keys:
            return 0
        shallow = -(-max(keys - s0 + 1, 0) * self.G // self.pairs) - 1
        return blocks - max(shallow, 0)

    def replay(self):
        """What workgroup i of a KV head does, for all of them: (row, block, range, number of the second range
        or -1), or None; and how many blocks are cut in two."""
        mine = [self.blocks_of(t) for t, _ in self.rows]
        n = sum(mine)
        lanes = 64 if len(self.rows) <= 64 else 256
        grid = max(self.slots // self.H_kv, n) + 2
        if n == 0:
            return [], 0
        if self.slots >= 2 * n * self.H_kv:
            return None, 0  # cut at will
        spare = 0
        if self.halve > 0 and len(self.rows) <= lanes and self.slots:
            spare = max(0, int((self.slots - n * self.H_kv) / self.H_kv))
        cut, halves, keys = [0] * len(mine), 0, 0
        if spare:
            deep = max(self._depth(t, s) for (t, s), m in zip(self.rows, mine) if m)

            def count(k):
                return [self._deeper(t, s, m, k) for (t, s), m in zip(self.rows, mine)]
            under = max(deep // 2, self.halve - 1)
            keys = max(deep, under)
            for _ in range(5):
                if keys - under <= 1:
                    break
                mid = (under + keys) // 2
                if sum(count(mid)) <= spare:
                    keys = mid
                else:
                    under = mid
            cut = count(keys)
            halves = sum(cut)
        order = [(b, qt) for qt in range(max(mine)) for b in range(len(mine)) if mine[b] > qt]
        order.sort(key=lambda x: -x[1])
        done = []
        for i in range(grid):
            if i < n:
                b, qt = order[i]
                t, s0 = self.rows[b]
                half = -1
                if spare and self._depth(t, s0, qt) > keys:
                    half = n + sum(cut[:b]) + mine[b] - 1 - qt
                done.append((b, qt, 0, half))
            elif i - n < halves:
                nth, b = i - n, 0
                while nth >= cut[b]:
                    nth -= cut[b]
                    b += 1
                done.append((b, mine[b] - 1 - nth, 1, i))
            else:
                done.append(None)
        return done, halves

    def check(self):
        """Every block once, second ranges where their firsts expect them, none past the room; returns how
        many blocks are cut in two."""
        done, halves = self.replay()
        if done is None:
            return 0
        firsts = [x for x in done if x and x[2] == 0]
        seconds = {x[3]: x[:2] for x in done if x and x[2] == 1}
        assert sorted(x[:2] for x in firsts) == sorted(
            (b, qt) for b, (t, _) in enumerate(self.rows) for qt in range(self.blocks_of(t)))
        assert {x[3]: x[:2] for x in firsts if x[3] >= 0} == seconds and len(seconds) == halves
        assert all((i + 1) * self.H_kv <= self.slots for i in seconds)
        return halves


def rounds_weights(T, G, D, dtype):
    """Whether a row's weights are rounded to one bf16 term before they meet V."""
    return dtype == torch.bfloat16 and D == 128 and T > 1 and T * G > 32


def attend(q, k, v, pos, window=-1):
    """q (T, H, D) at positions pos .. against keys k, v (pos + T, H_kv, D): the outputs in 64 bits and how
    far each may be off, as the tests' other bound has it but for the weights: rounded once (2^-8) in
    the rows of rounds_weights(), two terms in the other bf16 rows, w = hi + lo, of which hi is off by at
    most 2^-8 w, so that lo, rounded to the same 2^-8 of itself, leaves 2^-16 w; not at all in fp32."""
    T, H, D = q.shape
    G = H // k.shape[1]
    n = pos + T
    u, step = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    w_off = 0.0 if q.dtype == torch.float32 else u if rounds_weights(T, G, D, q.dtype) else u * u
    qh = q.double().transpose(0, 1)
    kk = k[:n].double().repeat_interleave(G, 1).permute(1, 2, 0).contiguous()
    vv = v[:n].double().repeat_interleave(G, 1).transpose(0, 1).contiguous()
    gap = (pos + torch.arange(T))[:, None] - torch.arange(n)[None]
    seen = (gap >= 0) & ((gap <= window) if window >= 0 else torch.ones(1, dtype=torch.bool))
    scale = 1 / math.sqrt(D)
    w = torch.softmax((qh @ kk * scale).masked_fill(~seen, float("-inf")), -1)
    out, mean = w @ vv, w @ vv.abs()
    size = (qh.abs() @ kk.abs() * scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
    d = (D + 4) * step * size + 8 * step * (1 + size)
    rel = 2 * d + w_off + (seen.sum(-1)[None, :, None] + 64) * step
    tol = torch.expm1(rel) * mean + u * out.abs() * (1 + torch.expm1(rel))
    return out.transpose(0, 1), tol.transpose(0, 1)


def close(got, want, tol, what=""):
    off = (got.detach().cpu().double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((off - tol)[bad].max()):.3e} past"
