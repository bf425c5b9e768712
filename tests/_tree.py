"""Decoding with drafted trees in plain Python and 64 bits, for the tests."""
import math
import random

import torch


def random_parents(rng, n, roots=0.0):
    """A tree of n nodes whose parents are drawn at random from the nodes before each."""
    return [-1 if i == 0 or rng.random() < roots else rng.randrange(i) for i in range(n)]


def ancestors(parents):
    """Per node its ancestors and itself, ascending; None for one whose chain does not go down to -1."""
    out = []
    for i in range(len(parents)):
        seen, a = [], i
        while a >= 0:
            seen.append(a)
            if parents[a] >= a or parents[a] < -1:
                seen = None
                break
            a = parents[a]
        out.append(None if seen is None else seen[::-1])
    return out


def words_of(nodes, words):
    """A list of node numbers as `words` signed 64-bit words."""
    m = sum(1 << j for j in nodes)
    line = [(m >> (64 * w)) & ((1 << 64) - 1) for w in range(words)]
    return [x - (1 << 64) if x >> 63 else x for x in line]


def plan(parents, lens, held, words):
    """Positions and masks of the rows' nodes, one row after another."""
    positions, masks, at = [], [], 0
    for n, s in zip(lens, held):
        for i, seen in enumerate(ancestors(parents[at:at + n])):
            ok = seen is not None and s >= 0 and i < 64 * words and s + len(seen) - 1 < 2 ** 31
            positions.append(s + len(seen) - 1 if ok else -1)
            masks.append(words_of(seen, words) if ok else [0] * words)
        at += n
    return positions, masks


def seen_keys(s0, node, bits, window):
    """Keys that node `node` of a row of s0 tokens sees, `bits` its mask's node numbers."""
    mine = sorted(j for j in bits if j <= node)
    pos = s0 + len(mine) - 1
    if window < 0:
        return list(range(s0)) + [s0 + j for j in mine]
    return list(range(min(max(0, pos - window), s0), s0)) + [s0 + j for j in mine[-(window + 1):]]


def attend(q, k, v, seen):
    """q (H, D) over the keys `seen` of k, v (n, H_kv, D): the output in 64 bits and how far the kernels may
    be off, by the reasoning of _paged.attend."""
    H, D = q.shape
    if not seen:
        return torch.zeros(H, D, dtype=torch.float64), torch.zeros(H, D, dtype=torch.float64)
    G, n = H // k.shape[1], len(seen)
    u, step = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    kk, vv = (t[seen].double().repeat_interleave(G, 1) for t in (k, v))
    scale = 1 / math.sqrt(D)
    s = torch.einsum("hd,nhd->hn", q.double(), kk) * scale
    size = torch.einsum("hd,nhd->hn", q.double().abs(), kk.abs()).amax(1) * scale
    w = torch.softmax(s, 1)
    out = torch.einsum("hn,nhd->hd", w, vv)
    mean = torch.einsum("hn,nhd->hd", w, vv.abs())
    d = (D + 4) * step * size + 8 * step * (1 + size)
    rel = 2 * d + (u if q.dtype == torch.bfloat16 else 0) + (n + 64) * step
    more = torch.expm1(rel)[:, None]
    return out, more * mean + u * out.abs() * (1 + more)


class Margin:
    """The nearest that a test came to its border, relative to what it compares."""

    def __init__(self):
        self.least = math.inf

    def less(self, x, y):
        if x != 0 or y != 0:  # nothing against nothing is not near but the same, on every side
            self.least = min(self.least, abs(x - y) / max(abs(x), abs(y)))
        return x < y


def verify(logits, tokens, parents, numbers, temperature, probs=None):
    """One row's walk, on lists: (kept, tokens, margin)."""
    near = Margin()
    n = len(tokens)
    if n == 0:
        return [], [], near.least
    V = len(logits[0])

    def distribution(row):
        x = [-math.inf if math.isnan(y) else y for y in row]
        top = max(x)
        if top == -math.inf:
            return None
        if top == math.inf:
            w = [1.0 if y == top else 0.0 for y in x]
        else:
            w = [math.exp((y - top) / temperature) for y in x]
        total = math.fsum(w)
        return [y / total for y in w]

    def first_best(row):
        x = [-math.inf if math.isnan(y) else y for y in row]
        return x.index(max(x)) if max(x) > -math.inf else None

    kept, out, node = [0], [], 0
    while True:
        greedy = temperature == 0
        best = first_best(logits[node])
        p = None if greedy else distribution(logits[node])
        q = probs[node] if probs is not None and not greedy else None
        a, gone, found = 0.0, set(), None
        rest = None if p is None else list(p)
        for i in range(node + 1, n):
            x = tokens[i]
            if parents[i] != node or not 0 <= x < V or best is None:
                continue
            if greedy:
                if x == best:
                    found = i
                    break
                continue
            left = math.fsum(rest) if q is not None and a > 0 or gone else 1.0
            if near.less(numbers[i] * left * (q[x] if q is not None else 1.0), rest[x]):
                found = i
                break
            if q is not None:
                a += left
                rest = [max(y - a * z, 0.0) for y, z in zip(p, q)]
            else:
                gone.add(x)
                rest[x] = 0.0
        if found is None:
            break
        node = found
        kept.append(node)
        out.append(tokens[node])
    if best is None:
        out.append(0)
    elif greedy:
        out.append(best)
    else:
        if math.fsum(rest) <= 0:
            rest = p
        want = numbers[0] * math.fsum(rest)
        upto = 0.0
        for i, w in enumerate(rest):
            upto += w
            # An empty weight leaves the border where the one before it had it.
            if w > 0 and near.less(want, upto):
                out.append(i)
                break
        else:
            out.append(max(i for i, w in enumerate(rest) if w > 0))
    return kept, out, near.least


def keep(pools, table, held, new, kept, counts, free, count, page):
    """paged_keep on lists, pools as dicts {(page, token): value}, all in place."""
    n_pages = len(free)
    for b, (s, t) in enumerate(zip(held, new)):
        t = max(t, 0)
        if s < 0 or s + t > len(table[b]) * page:
            continue
        c = max(0, min(counts[b], len(kept[b]), t))
        if t == 0 or not 0 <= table[b][(s + t - 1) // page] < n_pages:
            c = 0
        for j in range(c):
            i = kept[b][j]
            if not j < i < t:
                continue
            src, dst = table[b][(s + i) // page], table[b][(s + j) // page]
            if 0 <= src < n_pages and 0 <= dst < n_pages:
                for pool in pools:
                    pool[dst, (s + j) % page] = pool[src, (s + i) % page]
        for i in range(-(-(s + c) // page), -(-(s + t) // page)):
            if 0 <= table[b][i] < n_pages and count[0] < n_pages:
                free[count[0]] = table[b][i]
                count[0] += 1
            table[b][i] = -1
        held[b] = s + c
