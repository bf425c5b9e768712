"""What decoding with drafted tokens is timed on: the plan of the drafted trees, the attention of a tree
over a paged cache, the verification of the drafts and the cache's part in accepting them, as a serving
program calls them, each also in a plain form of elementary torch operations.

A row's drafted tokens are nodes: node 0, the root, is the last token that was accepted, every other node
a guess that follows its parent, a node before it. One forward runs all nodes of all rows, packed one
after another: node i of a row that holds s tokens is written behind them, at s + i, rotated to the
position s + its depth, and attends the row's tokens, its ancestors and itself. The logits of every node
then decide, with one random number a node, how far the drafts go: from the root down to the first node
none of whose children is accepted, whose own draw is one more token. The accepted nodes' keys and values
move up behind the row's tokens, and pages that no token is left in are given back.

``listed`` gives the named cases, ``draw`` more of the same kinds over the same ranges. The sizes are
those of the framework's own workloads: the 12-layer 768-wide quickstart model (12 heads of 64, fp32),
the mixed-window stack (12 query / 4 KV heads of 128, window 1024), the decode microbenchmark (32 rows,
16 / 4 heads of 128, up to 8192 keys) and the sampling model (32 layers, 32 / 8 heads of 128, 64 rows, a
vocabulary of 32768). Lengths of ragged rows are evenly spaced and dealt to the rows by the seed, so that
the work of a case does not depend on it. Pages are dealt at random, as in a pool that has served for a
while.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_K_SCALE = 1.2  # the models scale q and k by this after the norm


def _device():
    return torch.device("cuda", 0)


# -----------------------------------------------------------------------------------------------
# Cases
# -----------------------------------------------------------------------------------------------
# Trees. "lanes": `width` continuations of the root side by side (one: a chain), each a chain of its own;
# "spread": every node has `width` children, until the nodes are used up.
def _parents(n, shape, width):
    if shape == "lanes":
        return [-1 if i == 0 else max(0, i - width) for i in range(n)]
    return [-1 if i == 0 else (i - 1) // width for i in range(n)]


def _plan(name, rows, t_lo, t_hi, shape, width):
    """Positions and ancestors of t_lo to t_hi nodes for each of `rows` rows."""
    return {"name": name, "kind": "plan", "rows": rows, "t_lo": t_lo, "t_hi": t_hi, "shape": shape,
            "width": width}


def _attn(name, heads, kv_heads, dim, dtype, page, rows, lo, hi, t_lo, t_hi, shape, width, t_max, window=-1):
    """The attention of `rows` rows of t_lo to t_hi nodes behind lo to hi tokens, with its append."""
    return {"name": name, "kind": "attn", "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page": page, "rows": rows, "lo": lo, "hi": hi, "t_lo": t_lo, "t_hi": t_hi, "shape": shape,
            "width": width, "t_max": t_max, "window": window}


def _verify(name, rows, nodes, shape, width, vocab, temperature, drawn):
    """How far the drafts of `rows` rows go. drawn: they were drawn from a draft model's probabilities,
    which the verification takes; else they are guesses."""
    return {"name": name, "kind": "verify", "rows": rows, "nodes": nodes, "shape": shape, "width": width,
            "vocab": vocab, "temperature": temperature, "drawn": drawn}


def _keep(name, slots, kv_heads, dim, dtype, page, rows, lo, hi, nodes, width):
    """`rows` rows of lo to hi tokens keep a path of one to `width` of their nodes (lanes; of a chain, one to
    all), in every one of `slots` KV slots."""
    return {"name": name, "kind": "keep", "slots": slots, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page": page, "rows": rows, "lo": lo, "hi": hi, "nodes": nodes, "width": width}


def listed():
    return [
        # One user's chain of eight drafted tokens: all launch latency.
        _plan("plan_one", 1, 8, 8, "lanes", 1),
        # A full server with the widest trees, 64 rows of 64 nodes.
        _plan("plan_64x64", 64, 64, 64, "spread", 4),
        # The smallest forward: the quickstart's two rows, three guesses and what may follow each, in fp32.
        _attn("tree_quickstart_fp32", 12, 12, 64, "fp32", 16, 2, 79, 79, 7, 7, "lanes", 3, 96),
        # One user after a long prompt with a wide tree: the most keys of a row, 256 pairs for each of them.
        _attn("tree_one_row_16k", 32, 8, 128, "bf16", 64, 1, 16384, 16384, 64, 64, "spread", 4, 32768),
        # The decode microbenchmark's rows with trees of sixteen: the most cache read.
        _attn("tree_gqa16x4_8k", 16, 4, 128, "bf16", 16, 32, 512, 8191, 16, 16, "spread", 2, 16384),
        # A server whose rows draft chains, as many tokens as each has lately had accepted.
        _attn("chains_60_rows", 32, 8, 128, "bf16", 16, 60, 128, 8191, 1, 8, "lanes", 1, 16384),
        # Trees of different sizes through the mixed-window stack's local layers.
        _attn("tree_w1024", 12, 4, 128, "bf16", 32, 8, 300, 4001, 9, 61, "spread", 3, 4352, window=1024),
        # Greedy decoding of one row's chain of five.
        _verify("verify_greedy_one", 1, 6, "lanes", 1, 32768, 0.0, False),
        # The sampling model's 64 rows, chains of four drawn from a draft model.
        _verify("verify_chains_64", 64, 5, "lanes", 1, 32768, 1.0, True),
        # 32 rows with trees of guesses: the most logits.
        _verify("verify_trees_32x32", 32, 32, "spread", 4, 32768, 0.8, False),
        # The quickstart's two rows, of whose nodes one path is kept.
        _keep("keep_quickstart_fp32", 12, 12, 64, "fp32", 16, 2, 79, 79, 7, 3),
        # The sampling model's 64 rows: paths of up to four nodes in 32 layers.
        _keep("keep_64_rows", 32, 8, 128, "bf16", 16, 64, 40, 200, 17, 4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# Head groupings (query heads, KV heads) of the framework's workloads and tests.
_HEADS = [(12, 12), (12, 4), (16, 4), (32, 8), (16, 2), (8, 8)]
_PAGES = [16, 16, 32, 64, 128, 256]


def draw(rng):
    kind = rng.choice(["attn"] * 6 + ["verify"] * 4 + ["keep"] * 2 + ["plan"])
    shape = rng.choice(["lanes", "spread"])
    width = rng.choice([1, rng.randint(1, 6)])
    page = rng.choice(_PAGES)
    if kind == "plan":
        t_hi = _log_int(rng, 1, 64 if rng.random() < 0.7 else 200)
        return _plan("drawn", _log_int(rng, 1, min(256, 4096 // t_hi)), rng.choice([t_hi, (t_hi + 7) // 8]), t_hi,
                     shape, width)
    if kind == "verify":
        vocab = rng.choice([32768, _log_int(rng, 100, 130000)])
        drawn = rng.random() < 0.5
        temperature = rng.choice([1.0, round(rng.uniform(0.3, 1.5), 3)] if drawn else [0.0, 1.0, round(rng.uniform(0.3, 1.5), 3)])
        # At most the logits of the largest listed case.
        most = (32 * 32 * 32768 // (2 if drawn else 1)) // vocab
        nodes = _log_int(rng, 1, min(64, most))
        return _verify("drawn", _log_int(rng, 1, max(1, min(128, most // nodes))), nodes, shape, width, vocab, temperature, drawn)
    heads, kv_heads = rng.choice(_HEADS)
    dim = rng.choice([64, 64, 128, 128, 128, 96, 256])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    size = 2 if dtype == "bf16" else 4
    if kind == "keep":
        nodes = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, 300)
        slots = rng.choice([1, 12, 24, 32])
        token = 2 * slots * kv_heads * dim * size
        rows = _log_int(rng, 1, max(1, min(128, int(1.2e9 // (token * (hi + nodes + page))))))
        return _keep("drawn", slots, kv_heads, dim, dtype, page, rows, rng.choice([hi, hi // 4]), hi, nodes, min(width, nodes))
    window = rng.choice([-1, -1, -1, rng.randint(0, 2048)])
    t_hi = _log_int(rng, 1, 64 if rng.random() < 0.8 else 200)
    hi = _log_int(rng, 1, 16384)
    # At most the microbenchmark's cache bytes (285 MB), and of the arithmetic what takes about as long as one
    # row's wide tree.
    limit = 1.8e10 if dtype == "bf16" and dim == 128 else 6e9 if dtype == "bf16" else 2e9
    while 4 * heads * dim * t_hi * (hi + t_hi) > limit and t_hi > 1:
        t_hi //= 2
    cost = max(2 * (hi + t_hi) * kv_heads * dim * size / 2.8e8, 4 * heads * dim * t_hi * (hi + t_hi) / limit)
    rows = _log_int(rng, 1, max(1, min(64, int(1 // cost) if cost < 1 else 1)))
    return _attn("drawn", heads, kv_heads, dim, dtype, page, rows, rng.choice([hi, hi // 16, 0]), hi,
                 rng.choice([t_hi, (t_hi + 7) // 8]), t_hi, shape, width,
                 hi + t_hi + rng.choice([0, rng.randint(0, 300), 8192]), window)


# -----------------------------------------------------------------------------------------------
# Inputs
# -----------------------------------------------------------------------------------------------
def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)] if n > 1 else [hi] * n


def _sequences(case):
    """(tokens held, nodes) of every row of an attention case: longer rows have fewer nodes."""
    return list(zip(_spread(case["lo"], case["hi"], case["rows"]),
                    _spread(case["t_lo"], case["t_hi"], case["rows"])[::-1]))


def _dealt(values, seed):
    order = torch.randperm(len(values), generator=torch.Generator().manual_seed(seed)).tolist()
    return [values[i] for i in order]


def _normal(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device=_device()) * scale).to(dtype)


def _pages_of(n, page):
    return -(-n // page)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=_device())


def _offsets(lens):
    cu = [0]
    for t in lens:
        cu.append(cu[-1] + t)
    return cu


def _dealt_table(held, max_pages, spare, seed):
    """A block table of rows that hold `held` pages each, its pages dealt at random from a pool with
    `spare` more, entries without a page -1; and the pages that are left."""
    n = sum(held) + spare
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(held), max_pages), -1, dtype=torch.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    return table.to(_device()), order[at:], n


def _masks(parents, words):
    """Every node's ancestors and itself as bits, 64 a word."""
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    low = (1 << 64) - 1
    at = [[m >> (64 * w) & low for w in range(words)] for m in seen]
    return [[x - (1 << 64) if x >> 63 else x for x in line] for line in at]


def _path_lengths(case):
    """Nodes that each row keeps."""
    most = case["nodes"] if case["width"] == 1 else min(case["width"], 1 + (case["nodes"] - 1) // case["width"])
    return _spread(1, max(1, most), case["rows"])


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["kind"] == "verify":
        return _prepare_verify(case, seed, g)
    if case["kind"] == "plan":
        lens = _dealt(_spread(case["t_lo"], case["t_hi"], case["rows"]), seed)
        parents = [p for n in lens for p in _parents(n, case["shape"], case["width"])]
        held = torch.randint(0, 8192, (case["rows"],), generator=g, device=dev, dtype=torch.int32)
        return {"kind": "plan", "parents": _i32(parents), "cu": _i32(_offsets(lens)), "held": held,
                "longest": max(lens), "total": len(parents)}
    page, rows = case["page"], case["rows"]
    dt = DTYPES[case["dtype"]]
    Hk, D = case["kv_heads"], case["dim"]
    if case["kind"] == "keep":
        held = _dealt(_spread(case["lo"], case["hi"], rows), seed)
        n = case["nodes"]
        counts = _dealt(_path_lengths(case), seed + 1)
        # One lane of each tree; of several, one whose nodes lie behind all places that they move to, so that
        # a second pass finds them where the first did.
        lane = torch.randint(0, 1 << 20, (rows,), generator=torch.Generator().manual_seed(seed)).tolist()
        w = case["width"]
        kept = torch.full((rows, n), -1, dtype=torch.int32)
        for b, c in enumerate(counts):
            first = c - 1 + lane[b] % (w - c + 1) if w > 1 else 0
            for j in range(c):
                kept[b, j] = 0 if j == 0 else 1 + first + (j - 1) * w
        table, left, n_pages = _dealt_table([_pages_of(p + n, page) for p in held],
                                            _pages_of(max(held) + n, page) + 1, 8, seed)
        free = torch.full((n_pages,), -1, dtype=torch.int32)
        free[:len(left)] = left
        return {"kind": "keep", "page": page, "table": table, "held": _i32(held), "new": _i32([n] * rows),
                "kept": kept.to(dev), "counts": _i32(counts), "free": free.to(dev), "count": _i32([len(left)]),
                "k_pages": _normal(g, case["slots"], n_pages, page, Hk, D, dtype=dt),
                "v_pages": _normal(g, case["slots"], n_pages, page, Hk, D, dtype=dt)}
    H = case["heads"]
    held, lens = zip(*_dealt(_sequences(case), seed))
    words = _pages_of(max(lens), 64)
    masks = [m for n in lens for m in _masks(_parents(n, case["shape"], case["width"]), words)]
    table, _, n_pages = _dealt_table([_pages_of(p + t, page) for p, t in zip(held, lens)],
                                     _pages_of(case["t_max"], page), 64, seed)
    n = sum(lens)
    s = {"kind": "attn", "page": page, "window": case["window"], "table": table, "pos": _i32(held),
         "lens": lens, "held": held, "masks": torch.tensor(masks, dtype=torch.int64, device=dev),
         "k_pages": _normal(g, n_pages, page, Hk, D, dtype=dt, scale=_K_SCALE),
         "v_pages": _normal(g, n_pages, page, Hk, D, dtype=dt),
         "q": _normal(g, n, H, D, dtype=dt, scale=_K_SCALE),
         "k": _normal(g, n, Hk, D, dtype=dt, scale=_K_SCALE), "v": _normal(g, n, Hk, D, dtype=dt)}
    if len(set(lens)) > 1:  # rows of different numbers of nodes, packed
        s["cu"], s["longest"] = _i32(_offsets(lens)), max(lens)
    else:
        for name in ("q", "k", "v", "masks"):
            s[name] = s[name].view(len(lens), lens[0], *s[name].shape[1:])
    return s


def _prepare_verify(case, seed, g):
    """Logits with a few likely tokens, as a model's are, and drafts by a model that mostly agrees with them."""
    dev = _device()
    rows, n, V = case["rows"], case["nodes"], case["vocab"]
    parents = torch.tensor(_parents(n, case["shape"], case["width"]), device=dev)
    logits = torch.randn(rows, n, V, generator=g, device=dev) * 2.5
    near = logits + torch.randn(rows, n, V, generator=g, device=dev) * 0.4
    if case["temperature"] > 0:
        near = near / case["temperature"]
    tokens = torch.randint(0, V, (rows, n), generator=g, device=dev)
    s = {"kind": "verify", "temperature": case["temperature"], "longest": n}
    up = parents.clamp(min=0)
    if case["drawn"]:
        probs = torch.softmax(near, -1)
        # A child is drawn from its parent's probabilities: the least of exponential numbers over them.
        for i in range(1, n):
            e = -torch.log1p(-torch.rand(rows, V, generator=g, device=dev))
            tokens[:, i] = (e / probs[:, up[i]]).argmin(-1)
        s["probs"] = probs.view(rows * n, V)
    elif n > 1:
        # A node's children are the likeliest tokens after it, the first of them the likeliest.
        rank = torch.arange(n, device=dev) - torch.searchsorted(up, up)
        rank = (rank - (up == 0).long()).clamp(0, V - 1)  # node 0 stands among the root's own children
        best = near.topk(min(V, int(rank.max()) + 1), -1).indices
        tokens[:, 1:] = best[:, up[1:], rank[1:].clamp(max=best.shape[-1] - 1)]
    s.update(logits=logits.view(rows * n, V), tokens=tokens.view(-1),
             parents=parents.to(torch.int32).repeat(rows), cu=_i32([n * b for b in range(rows + 1)]),
             numbers=torch.rand(rows * n, generator=g, device=dev))
    return s


# -----------------------------------------------------------------------------------------------
# One pass
# -----------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    if s["kind"] == "plan":
        from modelcore_amd.kernels.paged import paged_tree
        plan = paged_tree(s["parents"], s["cu"], s["held"], max_seqlen=s["longest"])
        return [plan.positions, plan.masks]
    if s["kind"] == "verify":
        from modelcore_amd.sampling import verify_drafts
        done = verify_drafts(s["logits"], s["tokens"], s["parents"], s["cu"], s["numbers"],
                             temperature=s["temperature"], draft_probs=s.get("probs"), max_seqlen=s["longest"])
        return [done.kept, done.counts, done.tokens]
    if s["kind"] == "keep":
        from modelcore_amd.kernels.paged import paged_keep
        # The tables move with every step of a server; here each pass starts from the same ones.
        table, held, free, count = (s[n].clone() for n in ("table", "held", "free", "count"))
        paged_keep(s["k_pages"], s["v_pages"], table, held, s["new"], s["kept"], s["counts"], free, count)
        return [s["k_pages"], s["v_pages"], table, held, free, count]
    from modelcore_amd.kernels.flash_attn import flash_attn
    packed = {"cu_seqlens": s["cu"], "max_seqlen": s["longest"]} if "cu" in s else {}
    y = flash_attn.flash_attn_paged_tree_with_kvcache(
        s["q"], s["k_pages"], s["v_pages"], k=s["k"], v=s["v"], tree_masks=s["masks"], block_table=s["table"],
        cache_seqlens=s["pos"], window_size=(s["window"], 0), **packed)
    return [y, s["k_pages"], s["v_pages"]]


def _plan_plain(s):
    """Every node climbs to its root, all of them a step at a time."""
    parents, dev = s["parents"].long(), s["parents"].device
    cu, n = s["cu"].long(), s["total"]
    row = torch.repeat_interleave(torch.arange(len(cu) - 1, device=dev), cu[1:] - cu[:-1], output_size=n)
    begin = cu[row]
    at = torch.arange(n, device=dev) - begin
    words = _pages_of(s["longest"], 64)
    masks = torch.zeros(n, words, dtype=torch.int64, device=dev)
    depth = torch.full((n,), -1, dtype=torch.int64, device=dev)
    node, word = at, torch.arange(words, device=dev)[None, :]
    for _ in range(s["longest"]):
        bit = torch.ones_like(node) << (node & 63)
        masks |= torch.where((node[:, None] >= 0) & (node[:, None] >> 6 == word), bit[:, None], 0)
        depth += node >= 0
        node = torch.where(node >= 0, parents[begin + node.clamp(min=0)], -1)
    return [(s["held"].long()[row] + depth).to(torch.int32), masks]


def _verify_plain(s):
    """A node after the other: children come behind their parents, so the walk down the trees passes every
    node once. Probabilities and their sums are in 64 bits: a draw falls between neighbours of 32768."""
    cu, t = s["cu"].long(), s["temperature"]
    rows, longest = len(cu) - 1, s["longest"]
    dev = cu.device
    logits, tokens, parents = s["logits"], s["tokens"], s["parents"].long()
    n_of = cu[1:] - cu[:-1]
    if t == 0.0:
        best = logits.argmax(-1)
    else:
        x = logits.double() / t
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p /= p.sum(-1, keepdim=True)
    probs = s.get("probs")
    u = s["numbers"].double()
    each = torch.arange(rows, device=dev)
    node = torch.zeros(rows, dtype=torch.int64, device=dev)  # where each row's walk is
    kept = torch.full((rows, longest), -1, dtype=torch.int64, device=dev)
    kept[:, 0] = torch.where(n_of > 0, 0, -1)
    count = (n_of > 0).long()
    less = torch.zeros(rows, dtype=torch.float64, device=dev)  # of the draft's probabilities, taken off
    left = torch.ones(rows, dtype=torch.float64, device=dev)   # what is left of the target's
    gone = None if t == 0.0 or probs is not None else torch.zeros(rows, logits.shape[1], dtype=torch.bool, device=dev)
    for i in range(1, longest):
        at = (cu[:-1] + i).clamp(max=len(tokens) - 1)
        tried = (i < n_of) & (parents[at] == node)
        here, token = cu[:-1] + node, tokens[at]
        here = here.clamp(max=len(tokens) - 1)
        if t == 0.0:
            taken = tried & (best[here] == token)
        elif probs is not None:
            q = probs[here, token].double()
            taken = tried & (u[at] * left * q < (p[here, token] - less * q).clamp(min=0))
            refused = tried & ~taken
            less = torch.where(taken, 0.0, torch.where(refused, less + left, less))
            after = (p[here] - less[:, None] * probs[here].double()).clamp(min=0).sum(-1)
            left = torch.where(taken, 1.0, torch.where(refused, after, left))
        else:
            mine = torch.where(gone[each, token], 0.0, p[here, token])
            taken = tried & (u[at] * left < mine)
            refused = tried & ~taken
            left = torch.where(taken, 1.0, torch.where(refused, left - mine, left))
            gone[taken] = False
            gone[each, token] |= refused
        node = torch.where(taken, i, node)
        kept[each, count.clamp(max=longest - 1)] = torch.where(taken, i, kept[each, count.clamp(max=longest - 1)])
        count += taken
    here = (cu[:-1] + node).clamp(max=len(tokens) - 1)
    if t == 0.0:
        last = best[here]
    else:
        w = p[here]
        if probs is not None:
            rest = (w - less[:, None] * probs[here].double()).clamp(min=0)
        else:
            rest = torch.where(gone, 0.0, w)
        w = torch.where((rest.sum(-1) > 0)[:, None], rest, w)
        upto = torch.cumsum(w, -1)
        last = (upto <= (u[cu[:-1].clamp(max=len(u) - 1)] * upto[:, -1])[:, None]).sum(-1)
    out = torch.full((rows, longest), -1, dtype=torch.int64, device=dev)
    if longest > 1:
        behind = kept[:, 1:]
        out[:, :-1] = torch.where(behind >= 0, tokens[(cu[:-1, None] + behind).clamp(0, len(tokens) - 1)], -1)
    there = n_of > 0
    out[each[there], count[there] - 1] = last[there]
    return [kept.to(torch.int32), count.to(torch.int32), out]


def _keep_plain(s):
    page = s["page"]
    table, held, free, count = (s[n].clone() for n in ("table", "held", "free", "count"))
    k, v = (s[n].flatten(1, 2) for n in ("k_pages", "v_pages"))
    length, kept, n = held.long(), s["kept"].long(), s["counts"].long()
    j = torch.arange(kept.shape[1], device=table.device)[None, :]
    moved = ((j < n[:, None]) & (kept != j)).nonzero()
    b, j = moved[:, 0], moved[:, 1]

    def slot(b, at):
        return table[b, at // page].long() * page + at % page

    src, dst = slot(b, length[b] + kept[b, j]), slot(b, length[b] + j)
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    # Pages past the tokens that are kept go back, the rows' in order.
    had, has = (length + s["new"].long() + page - 1) // page, (length + n + page - 1) // page
    cols = torch.arange(table.shape[1], device=table.device)[None, :]
    back = (cols >= has[:, None]) & (cols < had[:, None])
    at = count.long() + torch.cumsum(back.flatten(), 0).view(back.shape) - 1
    free[at[back]] = table[back]
    table[back] = -1
    count += back.sum()
    held += s["counts"]
    return [s["k_pages"], s["v_pages"], table, held, free, count]


def _run_plain(s):
    if s["kind"] == "plan":
        return _plan_plain(s)
    if s["kind"] == "verify":
        return _verify_plain(s)
    if s["kind"] == "keep":
        return _keep_plain(s)
    page, window = s["page"], s["window"]
    shape = s["q"].shape
    q, k, v = (s[n].reshape(-1, *s[n].shape[-2:]) for n in ("q", "k", "v"))
    masks = s["masks"].reshape(len(q), -1)
    H, D = q.shape[1:]
    Hk = k.shape[1]
    G, dev = H // Hk, q.device
    lens, held = torch.tensor(s["lens"], device=dev), s["pos"].long()
    rows, T, L = len(s["lens"]), max(s["lens"]), max(p + t for p, t in zip(s["held"], s["lens"]))
    begin = torch.cumsum(lens, 0) - lens
    node, where = torch.arange(T, device=dev), torch.arange(L, device=dev)
    there = node[None, :] < lens[:, None]
    at = torch.where(there, begin[:, None] + node, 0)  # (rows, T): the packed nodes, padded
    pages = s["table"].long()[:, where // page].clamp(min=0)
    slots = pages * page + where % page
    k_rows, v_rows = s["k_pages"].flatten(0, 1), s["v_pages"].flatten(0, 1)
    row, i = there.nonzero(as_tuple=True)
    new = slots[row, held[row] + i]
    k_rows[new], v_rows[new] = k[at[row, i]], v[at[row, i]]
    # Who sees whom: (rows, T, T) among the nodes, then (rows, T, L) among all keys.
    above = (masks[at][:, :, node // 64] >> (node % 64) & 1).bool()
    nearer = above.flip(-1).cumsum(-1).flip(-1)  # that ancestor and those between it and the node
    depth = nearer[..., 0] - 1
    if window >= 0:
        above = above & (nearer <= window + 1)
    j = where[None, :] - held[:, None]
    seen = torch.gather(above, 2, j.clamp(0, T - 1)[:, None, :].expand(-1, T, -1)) & (j < T)[:, None, :]
    behind = j[:, None, :] < 0
    if window >= 0:
        behind = behind & (held[:, None, None] + depth[..., None] - where <= window)
    seen = torch.where((j < 0)[:, None, :], behind, seen)
    kt = k_rows[slots].float().permute(0, 2, 3, 1).contiguous()  # (rows, H_kv, D, keys)
    vt = v_rows[slots].float().permute(0, 2, 1, 3).contiguous()
    qt = q[at].float().view(rows, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(rows, Hk, G * T, D)
    score = (qt @ kt).view(rows, Hk, G, T, L) * D ** -0.5
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    score -= score.amax(-1, keepdim=True)
    weight = score.exp_().view(rows, Hk, G * T, L)
    weight = weight.nan_to_num_(0.0)  # of the padding, which may see nothing
    y = (weight @ vt) / weight.sum(-1, keepdim=True)
    y = y.view(rows, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(rows, T, H, D)
    return [y[there].to(q.dtype).view(shape), s["k_pages"], s["v_pages"]]


# -----------------------------------------------------------------------------------------------
# What a pass cannot do without
# -----------------------------------------------------------------------------------------------
def _depths(parents):
    depth = []
    for p in parents:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return depth


def work(case):
    rows = case["rows"]
    if case["kind"] == "plan":
        lens = _spread(case["t_lo"], case["t_hi"], rows)
        # Parents and lengths in; a position and a node's words of bits out.
        return {"bytes": sum(lens) * (8 + 8 * _pages_of(max(lens), 64)) + 8 * rows, "flops": 0}
    if case["kind"] == "verify":
        nodes = rows * case["nodes"]
        # The logits, and of the draft's probabilities those of each draft and of a row's last node.
        n = 4 * nodes * case["vocab"] + 24 * nodes
        return {"bytes": n + (4 * nodes + 4 * rows * case["vocab"] if case["drawn"] else 0),
                "flops": 0 if case["temperature"] == 0.0 else 4 * nodes * case["vocab"]}
    Hk, D = case["kv_heads"], case["dim"]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "keep":
        counts = _path_lengths(case)
        moved = sum(c - 1 for c in counts) if case["width"] > 1 else 0
        return {"bytes": 4 * moved * case["slots"] * Hk * D * size + 16 * rows + 4 * sum(counts), "flops": 0}
    H, window = case["heads"], case["window"]
    pairs = old = named = total = 0
    for p, n in _sequences(case):
        total += n
        depth = _depths(_parents(n, case["shape"], case["width"]))
        for d in depth:
            pairs += p + d + 1 if window < 0 else min(p + d, window) + 1
        old += p if window < 0 else min(p, window)
        named += _pages_of(p + n, case["page"])
    moved = 2 * total * H * D + 2 * Hk * D * (old + 2 * total)  # q, out; K/V read, new ones in and out
    return {"bytes": moved * size + 4 * named + 8 * total, "flops": 4 * H * D * pairs}


# -----------------------------------------------------------------------------------------------
# The same in 64 bits
# -----------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] in ("plan", "verify"):
        return None  # whole numbers
    s = prepare(case, seed)
    page = case["page"]
    k_pool, v_pool = s["k_pages"].double(), s["v_pages"].double()
    if case["kind"] == "keep":
        table, held, kept = s["table"].tolist(), s["held"].tolist(), s["kept"].tolist()
        for b, c in enumerate(s["counts"].tolist()):
            for j in range(c):  # in order, each node's place read before a later one is written there
                (to, to_at), (of, of_at) = (divmod(held[b] + i, page) for i in (j, kept[b][j]))
                for pool in (k_pool, v_pool):
                    pool[:, table[b][to], to_at] = pool[:, table[b][of], of_at].clone()
        return [k_pool, v_pool, None, None, None, None]
    window = case["window"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = (s[n].reshape(-1, *s[n].shape[-2:]).double() for n in ("q", "k", "v"))
    y = torch.empty_like(q)
    begin = 0
    for b, (p0, T) in enumerate(zip(s["held"], s["lens"])):
        parents = _parents(T, case["shape"], case["width"])
        pages = s["table"][b, :_pages_of(p0 + T, page)].long()
        new = torch.arange(p0, p0 + T, device=q.device)
        k_pool[pages[new // page], new % page] = k[begin:begin + T]
        v_pool[pages[new // page], new % page] = v[begin:begin + T]
        keys = k_pool[pages].reshape(-1, Hk, D)[:p0 + T]
        values = v_pool[pages].reshape(-1, Hk, D)[:p0 + T]
        seen = torch.zeros(T, p0 + T, dtype=torch.bool)
        depth = _depths(parents)
        for i in range(T):
            first = max(0, p0 + depth[i] - window) if window >= 0 else 0
            seen[i, min(first, p0):p0] = True
            a = i
            while a >= 0 and p0 + depth[a] >= first:
                seen[i, p0 + a] = True
                a = parents[a]
        seen = seen.to(q.device)
        for h in range(H):
            score = q[begin:begin + T, h].contiguous() @ keys[:, h * Hk // H].t().contiguous() / math.sqrt(D)
            weight = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
            y[begin:begin + T, h] = weight @ values[:, h * Hk // H].contiguous()
        begin += T
    return [y.view(s["q"].shape), k_pool, v_pool]
