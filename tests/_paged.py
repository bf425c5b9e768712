"""The paged cache's operators in 64 bits and plain Python, for the tests: pages and slots from a list,
attention row by row with a bound on what the kernels' roundings may add."""
import math

import torch


class Pool:
    """Pools of pages and a block table of rows that hold `lens` tokens, their pages dealt at random,
    all on the CPU; what no row holds is `stale`."""

    def __init__(self, lens, page, H_kv, D, dtype, max_pages=None, spare=3, seed=0, stale=float("nan")):
        g = torch.Generator().manual_seed(seed)
        held = [-(-n // page) for n in lens]
        self.n_pages = sum(held) + spare
        self.page, self.lens = page, list(lens)
        order = torch.randperm(self.n_pages, generator=g).tolist()
        self.table = torch.full((len(lens), max_pages or max(held + [1]) + 1), -1, dtype=torch.int32)
        for b, h in enumerate(held):
            for i in range(h):
                self.table[b, i] = order.pop()
        self.k = torch.full((self.n_pages, page, H_kv, D), stale, dtype=dtype)
        self.v = self.k.clone()
        for b, n in enumerate(lens):
            for t in range(n):
                p, o = self.place(b, t)
                self.k[p, o] = torch.randn(H_kv, D, generator=g).to(dtype)
                self.v[p, o] = torch.randn(H_kv, D, generator=g).to(dtype)

    def place(self, b, t):
        return int(self.table[b, t // self.page]), t % self.page

    def rows(self, b, n):
        """K and V of row b's first n tokens, (n, H_kv, D)."""
        at = [self.place(b, t) for t in range(n)]
        p, o = torch.tensor([x for x, _ in at]), torch.tensor([x for _, x in at])
        return self.k[p, o], self.v[p, o]


def attend(q, k, v, pos, window):
    """q (T, H, D) at positions pos .. against keys k, v (pos + T, H_kv, D): the outputs in 64 bits and,
    per output element, how far the kernels may be off.

    A score's terms are products of D pairs, which no kernel rounds to fewer than 32 bits: its sum is off by
    at most d = (D + 4) 2^-24 sum |q k| scale. exp2 of it adds a few units of its argument's last place. A
    weight is so off by a factor within exp(+-d'), its sum alike; the weights of the bf16 / 128 kernel for
    long rows are rounded once more (2^-8) before they meet V, and the sums over n keys, the
    ranges' merge and the final division take fewer than (n + 64) steps of 2^-24. Outputs are weighted
    means, so all of this is at most (2 d' + ..) sum w |v|, and the last rounding half a step of the
    result."""
    T, H, D = q.shape
    G = H // k.shape[1]
    q64, k64, v64 = q.double(), k.double(), v.double()
    out, tol = torch.empty(T, H, D, dtype=torch.float64), torch.empty(T, H, D, dtype=torch.float64)
    scale = 1 / math.sqrt(D)
    u = torch.finfo(q.dtype).eps / 2
    for t in range(T):
        p = pos + t
        lo = max(0, p - window) if window >= 0 else 0
        kk = k64[lo:p + 1].repeat_interleave(G, 1)  # (n, H, D)
        vv = v64[lo:p + 1].repeat_interleave(G, 1)
        s = torch.einsum("hd,nhd->hn", q64[t], kk) * scale
        size = torch.einsum("hd,nhd->hn", q64[t].abs(), kk.abs()).amax(1) * scale
        w = torch.softmax(s, 1)
        out[t] = torch.einsum("hn,nhd->hd", w, vv)
        mean = torch.einsum("hn,nhd->hd", w, vv.abs())
        n = p + 1 - lo
        step = 2.0 ** -24
        d = (D + 4) * step * size + 8 * step * (1 + size)
        rel = 2 * d + (u if q.dtype == torch.bfloat16 else 0) + (n + 64) * step
        tol[t] = torch.expm1(rel)[:, None] * mean + u * out[t].abs() * (1 + torch.expm1(rel)[:, None])
    return out, tol


def reserve(table, lens, new, free, count, total, page):
    """paged_reserve on Python lists, in place; returns slots, positions, cu, refused."""
    slots, positions, cu, refused = [], [], [0], 0
    width, asked, start = len(table[0]) if table else 0, 0, 0
    given = 0
    for b, (n, t) in enumerate(zip(lens, new)):
        fresh = min(max(t, 0), total - start)
        have, need = -(-max(n, 0) // page), -(-(max(n, 0) + fresh) // page)
        fits = n >= 0 and t >= 0 and need <= width
        take = need - have if fits else 0
        asked += take
        ok = fits and (take == 0 or asked <= count[0])
        if ok:
            for i in range(take):
                table[b][have + i] = free[count[0] - 1 - (asked - take) - i]
            given += take
        refused += not ok
        for i in range(fresh):
            p = n + i
            positions.append(p if ok else -1)
            slots.append(table[b][p // page] * page + p % page if ok else -1)
        start += fresh
        cu.append(start)
    count[0] -= given
    slots += [-1] * (total - start)
    positions += [-1] * (total - start)
    return slots, positions, cu, refused


def release(table, lens, rows, free, count, page):
    for b in rows:
        if not 0 <= b < len(lens):
            continue
        for i in range(min(-(-max(lens[b], 0) // page), len(table[b]))):
            if count[0] < len(free):
                free[count[0]] = table[b][i]
                count[0] += 1
            table[b][i] = -1
        lens[b] = 0


def rotated(x, cos, sin, eps, scale):
    """The pre-attention step of x (n, heads, D) in 64 bits, cos and sin (n, D / 2) of its tokens."""
    half = x.shape[-1] // 2
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    a, b = x[..., :half], x[..., half:]
    y = torch.cat([a * c + b * s, b * c - a * s], -1)
    return y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * scale
