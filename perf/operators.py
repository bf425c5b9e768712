"""What the paged KV cache is timed on: its page plan, its pre-attention step and its attention, as
a serving program calls them, each also in a plain form of elementary torch operations.

A paged cache keeps K and V in a pool of pages, (n_pages, page_size, H_kv, D) per KV slot, and per
request a row of a block table that names its pages. Once per forward a program reserves the pages
of the new tokens and gets their slots (page * page_size + offset) and positions; then every layer
rotates, norms and scales q and k, writes k and v to the slots and attends through the table.

``listed`` gives the named cases, ``draw`` more of the same kinds over the same ranges. The sizes
are those of the framework's own workloads: the 12-layer 768-wide quickstart model (12 heads of
64, fp32), the mixed-window stack (12 query / 4 KV heads of 128, window 1024), the decode
microbenchmark (32 rows, 16 / 4 heads of 128, up to 8192 keys), the chunked prefill (8 rows,
512-token chunks, 32 / 8 heads of 128) and the sampling model (32 / 8 heads of 128). Lengths of
ragged rows are evenly spaced and dealt to the rows by the seed, so that the work of a case does not
depend on it. Pages are dealt at random, as in a pool that has served for a while.
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
def _attn(name, heads, kv_heads, dim, dtype, page, t_max, ones=0, lo=0, hi=0, chunks=0, t_lo=0,
          t_hi=0, c_lo=0, c_hi=0, window=-1):
    """An attention call with its append: `ones` rows of one new token at positions spaced over
    [lo, hi], and `chunks` rows of t_lo to t_hi new tokens at positions spaced over [c_lo, c_hi]."""
    return {"name": name, "kind": "attn", "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "page": page, "t_max": t_max, "ones": ones, "lo": lo, "hi": hi,
            "chunks": chunks, "t_lo": t_lo, "t_hi": t_hi, "c_lo": c_lo, "c_hi": c_hi,
            "window": window}


def _step(name, tokens, each, heads, kv_heads, dim, dtype, page, n_pos):
    """The pre-attention step of `tokens` new tokens, `each` of them per request."""
    return {"name": name, "kind": "step", "tokens": tokens, "each": each, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "n_pos": n_pos}


def _plan(name, rows, lo, hi, t_lo, t_hi, page, t_max, done=0):
    """Pages, slots and positions of t_lo to t_hi new tokens for each of `rows` requests that hold
    lo to hi; `done` of the requests have ended, give their pages back and start anew."""
    return {"name": name, "kind": "plan", "rows": rows, "lo": lo, "hi": hi, "t_lo": t_lo,
            "t_hi": t_hi, "page": page, "t_max": t_max, "done": done}


def listed():
    return [
        # A decode step of 64 running requests: one token each, a page for every sixteenth of them.
        _plan("plan_decode_64", 64, 512, 8192, 1, 1, 16, 16384),
        # A server admitting work: 512 requests, a quarter of which have ended and start anew, read
        # 37 to 4001 tokens each (a million slots).
        _plan("plan_prompts_512", 512, 0, 2000, 37, 4001, 64, 8192, done=128),
        # The step before the attention in a decode step of 64 requests of the sampling model.
        _step("step_decode_64", 64, 1, 32, 8, 128, "bf16", 16, 16384),
        # The same over the 4096 tokens of a chunk of eight prompts in the chunked prefill.
        _step("step_chunk_8x512", 4096, 512, 32, 8, 128, "bf16", 64, 16384),
        # The smallest call: one token for each of the quickstart's two rows, at the end of its
        # 16-token prompt and 64 new tokens, in its own fp32. All launch latency.
        _attn("decode_quickstart_fp32", 12, 12, 64, "fp32", 16, 96, ones=2, lo=79, hi=79),
        # The decode microbenchmark from pages: the largest decode, bound by reading the cache.
        _attn("decode_gqa16x4_8k", 16, 4, 128, "bf16", 16, 16384, ones=32, lo=512, hi=8191),
        # One user's generation after a long prompt: a single row, 16K keys.
        _attn("decode_one_row_16k", 32, 8, 128, "bf16", 64, 32768, ones=1, lo=16384, hi=16384),
        # A chunk in the middle of the chunked prefill of eight 16K prompts: the most arithmetic.
        _attn("chunk_gqa32x8_8k", 32, 8, 128, "bf16", 64, 16384, chunks=8, t_lo=512, t_hi=512,
              c_lo=8192, c_hi=8192),
        # The next message of one conversation: a hundred new tokens after 8000 cached ones.
        _attn("chat_turn_8k", 32, 8, 128, "bf16", 16, 16384, chunks=1, t_lo=100, t_hi=100,
              c_lo=8000, c_hi=8000),
        # A server's step: 60 requests that decode, and four prompts of which this step reads a
        # chunk, in one call.
        _attn("mixed_60_and_4", 32, 8, 128, "bf16", 16, 16384, ones=60, lo=128, hi=8191, chunks=4,
              t_lo=300, t_hi=512, c_lo=0, c_hi=3000),
        # Eight prompts of different lengths through the mixed-window stack's local layers.
        _attn("prompts_w1024", 12, 4, 128, "bf16", 32, 4352, chunks=8, t_lo=37, t_hi=4001,
              window=1024),
        # The quickstart model reading two prompts of its own length in fp32.
        _attn("prompts_quickstart_fp32", 12, 12, 64, "fp32", 16, 576, chunks=2, t_lo=512, t_hi=512),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# Head groupings (query heads, KV heads) of the framework's workloads and tests.
_HEADS = [(12, 12), (12, 4), (16, 4), (32, 8), (16, 2), (8, 8)]
_PAGES = [16, 16, 32, 64, 128, 256]


def draw(rng):
    kind = rng.choice(["decode"] * 4 + ["chunk"] * 4 + ["mixed"] * 4 + ["step"] * 2 + ["plan"] * 2)
    page = rng.choice(_PAGES)
    if kind == "plan":
        rows = _log_int(rng, 1, 512)
        hi = _log_int(rng, 1, 8192)
        t_hi = rng.choice([1, _log_int(rng, 1, 4001)])
        return _plan("drawn", rows, rng.choice([0, hi // 8, hi]), hi, rng.choice([t_hi, (t_hi + 7) // 8]),
                     t_hi, page, hi + t_hi + rng.randint(0, 3000), rng.choice([0, rows // 4, rows]))
    heads, kv_heads = rng.choice(_HEADS)
    dim = rng.choice([64, 64, 128, 128, 128, 96, 256])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if kind == "step":
        return _step("drawn", _log_int(rng, 1, 4096 if dtype == "bf16" and dim <= 128 else 1000),
                     rng.choice([1, _log_int(rng, 1, 2048)]), heads, kv_heads, dim, dtype, page,
                     rng.randint(4200, 16384))
    window = rng.choice([-1, -1, -1, rng.randint(0, 2048)])
    size = 2 if dtype == "bf16" else 4
    ones = chunks = lo = hi = t_lo = t_hi = c_lo = c_hi = 0
    if kind in ("decode", "mixed"):
        # At most the microbenchmark's cache bytes (285 MB) for the single tokens of a call.
        hi = _log_int(rng, 1, 16384)
        lo = rng.choice([hi, hi // 16])
        ones = _log_int(rng, 1, max(1, min(64, int(2.8e8 // (2 * (hi + 1) * kv_heads * dim * size)))))
    if kind in ("chunk", "mixed"):
        t_hi = _log_int(rng, 2, 2048)
        c_hi = rng.choice([0, _log_int(rng, 16, 8192)])
        # The listed cases bound the work: a chunk of eight 16K prompts on the 128-wide bf16 heads;
        # of the others what takes about as long.
        limit = 2.5e11 if dtype == "bf16" and dim == 128 else 2.5e10 if dtype == "bf16" else 8e9
        one = 4 * heads * dim * t_hi * (c_hi + t_hi / 2)
        while one > limit and t_hi > 2:
            t_hi //= 2
            one = 4 * heads * dim * t_hi * (c_hi + t_hi / 2)
        t_lo, c_lo = rng.choice([t_hi, (t_hi + 7) // 8]), rng.choice([c_hi, c_hi // 4, 0])
        chunks = _log_int(rng, 1, max(1, min(16, int(limit // one))))
    t_max = max(hi + 1, c_hi + t_hi) + rng.choice([0, rng.randint(0, 300), 8192])
    return _attn("drawn", heads, kv_heads, dim, dtype, page, t_max, ones, lo, hi, chunks, t_lo, t_hi,
                 c_lo, c_hi, window)


# -----------------------------------------------------------------------------------------------
# Inputs
# -----------------------------------------------------------------------------------------------
def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)] if n > 1 else [hi] * n


def _dealt(values, seed):
    order = torch.randperm(len(values), generator=torch.Generator().manual_seed(seed)).tolist()
    return [values[i] for i in order]


def _normal(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device=_device()) * scale).to(dtype)


def _pages_of(n, page):
    return -(-n // page)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=_device())


def _sequences(case):
    """(position, new tokens) of every row of an attention case."""
    return ([(p, 1) for p in _spread(case["lo"], case["hi"], case["ones"])] +
            list(zip(_spread(case["c_lo"], case["c_hi"], case["chunks"]),
                     _spread(case["t_lo"], case["t_hi"], case["chunks"])[::-1])))


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


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)
    page = case["page"]
    if case["kind"] == "plan":
        lens = _dealt(_spread(case["lo"], case["hi"], case["rows"]), seed)
        new = _dealt(_spread(case["t_lo"], case["t_hi"], case["rows"]), seed + 1)
        done = sorted(_dealt(list(range(case["rows"])), seed + 2)[:case["done"]])
        held = [_pages_of(n, page) for n in lens]
        # Pages enough, whichever rows the new tokens fall to.
        table, left, n_pages = _dealt_table(held, _pages_of(case["t_max"], page),
                                            sum(_pages_of(t, page) + 1 for t in new), seed)
        free = torch.full((n_pages,), -1, dtype=torch.int32)
        free[:len(left)] = left
        return {"kind": "plan", "table": table, "lens": _i32(lens), "new": _i32(new),
                "done": _i32(done), "free": free.to(dev), "count": _i32([len(left)]),
                "total": sum(new), "page": page}
    dt = DTYPES[case["dtype"]]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "step":
        # The tokens of each request follow one another, in pages of its own.
        n, each, n_pos = case["tokens"], case["each"], case["n_pos"]
        pos, slots = [], []
        requests = -(-n // each)
        n_pages = 2 * requests * (_pages_of(each, page) + 1)
        order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        for i, p0 in enumerate(_dealt(_spread(0, n_pos - each, requests), seed + 1)):
            mine = {}
            for p in range(p0, p0 + min(each, n - i * each)):
                if p // page not in mine:
                    mine[p // page] = order.pop()
                pos.append(p)
                slots.append(mine[p // page] * page + p % page)
        half = D // 2
        freq = 100000.0 ** (-torch.arange(0, half, dtype=torch.float64, device=dev) / half)
        angle = torch.arange(n_pos, dtype=torch.float64, device=dev)[:, None] * freq[None, :]
        # q, k and v are the columns of one stacked projection's output.
        qkv = _normal(g, n, H + 2 * Hk, D, dtype=dt)
        return {"kind": "step", "q": qkv[:, :H], "k": qkv[:, H:H + Hk], "v": qkv[:, H + Hk:],
                "cos": angle.cos().to(dt)[None, :, None, :], "sin": angle.sin().to(dt)[None, :, None, :],
                "pos": _i32(pos), "slots": torch.tensor(slots, dtype=torch.int64, device=dev),
                "k_pages": torch.zeros(n_pages, page, Hk, D, dtype=dt, device=dev),
                "v_pages": torch.zeros(n_pages, page, Hk, D, dtype=dt, device=dev)}
    seqs = _dealt(_sequences(case), seed)
    table, left, n_pages = _dealt_table([_pages_of(p + t, page) for p, t in seqs],
                                        _pages_of(case["t_max"], page), 64, seed)
    lens = [t for _, t in seqs]
    cu = [0]
    for t in lens:
        cu.append(cu[-1] + t)
    n = cu[-1]
    s = {"kind": "attn", "seqs": seqs, "cu_host": cu, "page": page, "window": case["window"],
         "table": table, "pos": _i32([p for p, _ in seqs]),
         "k_pages": _normal(g, n_pages, page, Hk, D, dtype=dt, scale=_K_SCALE),
         "v_pages": _normal(g, n_pages, page, Hk, D, dtype=dt),
         "q": _normal(g, n, H, D, dtype=dt, scale=_K_SCALE),
         "k": _normal(g, n, Hk, D, dtype=dt, scale=_K_SCALE), "v": _normal(g, n, Hk, D, dtype=dt)}
    if len(set(lens)) > 1:  # rows of different lengths, packed
        s["cu"], s["longest"] = _i32(cu), max(lens)
    else:
        for name in ("q", "k", "v"):
            s[name] = s[name].view(len(lens), lens[0], *s[name].shape[1:])
    return s


# -----------------------------------------------------------------------------------------------
# One pass
# -----------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    if s["kind"] == "plan":
        from modelcore_amd.kernels.paged import paged_release, paged_reserve
        # The tables move with every step of a server; here each pass starts from the same ones.
        table, lens, free, count = (s[n].clone() for n in ("table", "lens", "free", "count"))
        if s["done"].numel():
            paged_release(table, lens, s["done"], free, count, page_size=s["page"])
        plan = paged_reserve(table, lens, s["new"], free, count, total=s["total"],
                             page_size=s["page"])
        return [plan.slots, plan.positions, plan.cu_seqlens, plan.refused, table, lens, free, count]
    if s["kind"] == "step":
        from modelcore_amd.kernels.qk_epilogue import rope_norm_scale_append_paged
        q = rope_norm_scale_append_paged(s["q"], s["cos"], s["sin"], s["pos"], s["k"], s["v"],
                                         s["k_pages"], s["v_pages"], s["slots"])
        return [q, s["k_pages"], s["v_pages"]]
    from modelcore_amd.kernels.flash_attn import flash_attn
    packed = {"cu_seqlens": s["cu"], "max_seqlen": s["longest"]} if "cu" in s else {}
    y = flash_attn.flash_attn_paged_with_kvcache(
        s["q"], s["k_pages"], s["v_pages"], k=s["k"], v=s["v"], block_table=s["table"],
        cache_seqlens=s["pos"], causal=True, window_size=(s["window"], 0), **packed)
    return [y, s["k_pages"], s["v_pages"]]


def _release(table, lens, done, free, count, page):
    """The rows `done` give their pages back: onto the stack of free pages, in order."""
    cols = torch.arange(table.shape[1], device=table.device)[None, :]
    held = (lens[done].long() + page - 1) // page
    off = torch.cumsum(held, 0) - held
    there = cols < held[:, None]
    at = (count.long() + off)[:, None] + cols
    free[at[there]] = table[done][there]
    table[done] = torch.where(there, -1, table[done])
    count += held.sum()
    lens[done] = 0


def _reserve(table, lens, new, free, count, total, page):
    """Pages off the stack for the rows in order, then every new token's slot and position."""
    dev = table.device
    length, fresh = lens.long(), new.long()
    have, need = (length + page - 1) // page, (length + fresh + page - 1) // page
    fits = need <= table.shape[1]
    take = torch.where(fits, need - have, 0)
    upto = torch.cumsum(take, 0)
    ok = fits & ((take == 0) | (upto <= count.long()))
    cols = torch.arange(table.shape[1], device=dev)[None, :]
    mine = (cols >= have[:, None]) & (cols < need[:, None]) & ok[:, None]
    rank = (upto - take)[:, None] + cols - have[:, None]
    table[mine] = free[(count.long() - 1 - rank)[mine]]
    cu = torch.zeros(len(new) + 1, dtype=torch.int32, device=dev)
    cu[1:] = torch.cumsum(fresh, 0)
    row = torch.repeat_interleave(torch.arange(len(new), device=dev), fresh, output_size=total)
    pos = length[row] + torch.arange(total, device=dev) - cu[row].long()
    in_row = ok[row]
    slots = table[row, torch.where(in_row, pos // page, 0)].long() * page + pos % page
    refused = (~ok).sum(0, keepdim=True).to(torch.int32)
    count -= torch.where(ok, take, 0).sum()
    return (torch.where(in_row, slots, -1), torch.where(in_row, pos, -1).to(torch.int32), cu, refused)


def _rotated(x, cos, sin):
    """x rotated by each token's angles, RMS-normed over its last dim and scaled."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    r = torch.cat([a * cos + b * sin, b * cos - a * sin], -1)
    eps = torch.finfo(torch.float32).eps
    return r * torch.rsqrt((r * r).mean(-1, keepdim=True) + eps) * _K_SCALE


def _run_plain(s):
    page = s.get("page")
    if s["kind"] == "plan":
        table, lens, free, count = (s[n].clone() for n in ("table", "lens", "free", "count"))
        if s["done"].numel():
            _release(table, lens, s["done"].long(), free, count, page)
        slots, pos, cu, refused = _reserve(table, lens, s["new"], free, count, s["total"], page)
        return [slots, pos, cu, refused, table, lens, free, count]
    k_rows, v_rows = s["k_pages"].flatten(0, 1), s["v_pages"].flatten(0, 1)
    if s["kind"] == "step":
        pos = s["pos"].long()
        cos, sin = s["cos"][0, pos].float(), s["sin"][0, pos].float()
        k_rows[s["slots"]] = _rotated(s["k"].float(), cos, sin).to(k_rows.dtype)
        v_rows[s["slots"]] = s["v"]
        return [_rotated(s["q"].float(), cos, sin).to(s["q"].dtype), s["k_pages"], s["v_pages"]]
    q, k, v = (s[n].reshape(-1, *s[n].shape[-2:]) for n in ("q", "k", "v"))
    H, D = q.shape[1:]
    Hk = k.shape[1]
    G = H // Hk
    out = torch.empty_like(q)
    window = s["window"]
    for b, (p0, T) in enumerate(s["seqs"]):
        at = slice(s["cu_host"][b], s["cu_host"][b] + T)
        L = p0 + T
        where = torch.arange(L, device=q.device)
        rows = s["table"][b].long()[where // page] * page + where % page
        k_rows[rows[p0:]], v_rows[rows[p0:]] = k[at], v[at]
        lo = max(0, p0 - window) if window >= 0 else 0
        kt = k_rows[rows[lo:]].float().permute(1, 2, 0).contiguous()  # (H_kv, D, keys)
        vt = v_rows[rows[lo:]].float().transpose(0, 1).contiguous()
        qt = q[at].float().view(T, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * T, D)
        score = (qt @ kt).view(Hk, G, T, L - lo) * D ** -0.5
        gap = where[p0:, None] - where[None, lo:]
        hidden = gap < 0
        if window >= 0:
            hidden = hidden | (gap > window)
        score.masked_fill_(hidden, float("-inf"))
        score -= score.amax(-1, keepdim=True)
        score.exp_()
        weight = score.view(Hk, G * T, L - lo)
        y = (weight @ vt) / weight.sum(-1, keepdim=True)
        out[at] = y.view(Hk, G, T, D).permute(2, 0, 1, 3).reshape(T, H, D).to(out.dtype)
    return [out.view(s["q"].shape), s["k_pages"], s["v_pages"]]


# -----------------------------------------------------------------------------------------------
# What a pass cannot do without
# -----------------------------------------------------------------------------------------------
def _pairs(pos, T, window):
    """(query, key) pairs of T tokens from position pos on, and the keys they read in all."""
    if window < 0:
        return T * pos + T * (T + 1) // 2, pos + T
    full = max(0, min(T, window - pos + 1))  # queries that still see key 0
    return (full * pos + full * (full + 1) // 2 + (T - full) * (window + 1),
            pos + T - max(0, pos - window))


def work(case):
    if case["kind"] == "plan":
        page, n = case["page"], case["rows"]
        lens, new = _spread(case["lo"], case["hi"], n), _spread(case["t_lo"], case["t_hi"], n)
        total = sum(new)
        # Lengths in, cu_seqlens out, the pages that change hands, a slot and a position per token.
        moved = _pages_of(total, page) + sum(_pages_of(x, page) for x in lens) * case["done"] // n
        return {"bytes": 12 * n + 8 * moved + 12 * total, "flops": 0}
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "step":
        row = (H + 2 * Hk) * D
        # Of the tables the rows of the tokens' positions.
        return {"bytes": case["tokens"] * ((2 * row + D) * size + 12),
                "flops": case["tokens"] * (H + Hk) * D * 6}
    seqs = _sequences(case)
    total = sum(t for _, t in seqs)
    seen = [_pairs(p, t, case["window"]) for p, t in seqs]
    old = sum(keys for _, keys in seen) - total  # cached keys read; the new ones come as k, v
    rows = 2 * total * H * D + 2 * Hk * D * (old + 2 * total)  # q, out; K/V read, new ones written
    named = sum(_pages_of(keys, case["page"]) for _, keys in seen)
    return {"bytes": rows * size + 4 * named, "flops": 4 * H * D * sum(p for p, _ in seen)}


# -----------------------------------------------------------------------------------------------
# The same in 64 bits
# -----------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    k_pool, v_pool = s["k_pages"].double(), s["v_pages"].double()
    page = case["page"]
    if case["kind"] == "step":
        eps = torch.finfo(torch.float32).eps
        angle = torch.complex(s["cos"][0, :, 0].double(), -s["sin"][0, :, 0].double())[s["pos"].long()]

        def turned(x):
            """The two halves of a head as the parts of complex numbers, turned by -theta."""
            half = x.shape[-1] // 2
            z = torch.complex(x[..., :half].double().contiguous(), x[..., half:].double().contiguous())
            z = z * angle[:, None, :]
            y = torch.cat([z.real, z.imag], -1)
            return _K_SCALE * y / torch.sqrt(y.square().sum(-1, keepdim=True) / x.shape[-1] + eps)

        at = (s["slots"] // page, s["slots"] % page)
        k_pool[at], v_pool[at] = turned(s["k"]), s["v"].double()
        return [turned(s["q"]), k_pool, v_pool]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = (s[n].reshape(-1, *s[n].shape[-2:]).double() for n in ("q", "k", "v"))
    y = torch.empty_like(q)
    at = 0
    for b, (p0, T) in enumerate(s["seqs"]):
        held = s["table"][b, :_pages_of(p0 + T, page)].long()
        new = torch.arange(p0, p0 + T, device=q.device)
        k_pool[held[new // page], new % page] = k[at:at + T]
        v_pool[held[new // page], new % page] = v[at:at + T]
        keys = k_pool[held].reshape(-1, Hk, D)[:p0 + T]
        values = v_pool[held].reshape(-1, Hk, D)[:p0 + T]
        cols = torch.arange(p0 + T, device=q.device)
        seen = cols[None, :] <= new[:, None]
        if case["window"] >= 0:
            seen &= cols[None, :] >= new[:, None] - case["window"]
        for h in range(H):
            score = q[at:at + T, h].contiguous() @ keys[:, h * Hk // H].t().contiguous() / math.sqrt(D)
            weight = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
            y[at:at + T, h] = weight @ values[:, h * Hk // H].contiguous()
        at += T
    return [y.view(s["q"].shape), k_pool, v_pool]
