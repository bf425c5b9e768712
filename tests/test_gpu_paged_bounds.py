"""The paged attention at the ends of what its header allows: bounds, scratch, positions, KV heads."""
import pytest
import torch

from _paged import Pool
from _paged_blocks import attend, close
from modelcore_amd import _ext
from modelcore_amd.kernels.flash_attn import flash_attn

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("longest", [71, (1 << 31) - 1, 1 << 31, (1 << 32) + 2, (1 << 63) - 1])
def test_rows_shorter_than_any_bound(dtype, D, longest):
    """max_seqlen is an upper bound: the outputs are those of the exact one."""
    g = torch.Generator().manual_seed(3)
    new, pos = [40, 1, 30], [30, 700, 10]
    pool = Pool([p + t for p, t in zip(pos, new)], 16, 2, D, dtype, stale=0.0)
    k, v, table = pool.k.to(DEV), pool.v.to(DEV), pool.table.to(DEV)
    q = torch.randn(71, 8, D, generator=g).to(dtype).to(DEV)
    cu, at = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 40, 41, 71], pos))
    want = flash_attn.flash_attn_paged_with_kvcache(q, k, v, block_table=table, cache_seqlens=at, cu_seqlens=cu,
                                                    max_seqlen=71, causal=True)
    lib, code = _ext.lib(), _ext.dtype_code(dtype)
    sizes = (3, 71, longest, 8, 2, D)
    nbytes = lib.mcamd_paged_scratch_bytes(*sizes, table.shape[1], 16, -1, code)
    scratch = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=DEV)
    out = torch.full_like(q, 7)
    assert lib.mcamd_flash_attn_paged_with_kvcache(
        q.data_ptr(), None, None, k.data_ptr(), v.data_ptr(), table.data_ptr(), table.stride(0), at.data_ptr(),
        cu.data_ptr(), out.data_ptr(), *sizes, pool.n_pages, 16, k.stride(0), table.shape[1], -1, 1, code,
        scratch.data_ptr() if nbytes else None, nbytes, _ext.stream_handle(q.device)) == _ext.OK
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("rows", [[(1, 5000)], [(1, 3000), (1, 10), (70, 2000), (3, 900)], [(150, 1900)]])
@pytest.mark.parametrize("short", [None, 0, 16])
def test_less_scratch_than_keys_are_cut_with(dtype, D, rows, short):
    """None of it, or a little too few bytes: every row is whole, and right."""
    g = torch.Generator().manual_seed(4)
    pool = Pool([p + t for t, p in rows], 16, 2, D, dtype, stale=0.0)
    k, v, table = pool.k.to(DEV), pool.v.to(DEV), pool.table.to(DEV)
    n, cu = sum(t for t, _ in rows), [0]
    for t, _ in rows:
        cu.append(cu[-1] + t)
    q = torch.randn(n, 8, D, generator=g).to(dtype)
    cus, at = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (cu, [p for _, p in rows]))
    lib, code = _ext.lib(), _ext.dtype_code(dtype)
    sizes = (len(rows), n, max(t for t, _ in rows), 8, 2, D)
    nbytes = lib.mcamd_paged_scratch_bytes(*sizes, table.shape[1], 16, -1, code)
    assert nbytes > 16
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    dq, out = q.to(DEV), torch.full((n, 8, D), 7, dtype=dtype, device=DEV)
    assert lib.mcamd_flash_attn_paged_with_kvcache(
        dq.data_ptr(), None, None, k.data_ptr(), v.data_ptr(), table.data_ptr(), table.stride(0), at.data_ptr(),
        cus.data_ptr(), out.data_ptr(), *sizes, pool.n_pages, 16, k.stride(0), table.shape[1], -1, 1, code,
        None if short is None else scratch.data_ptr(), 0 if short is None else nbytes - short,
        _ext.stream_handle(dq.device)) == _ext.OK
    for b, (t, p) in enumerate(rows):
        want, tol = attend(q[cu[b]:cu[b + 1]], *pool.rows(b, p + t), p)
        close(out[cu[b]:cu[b + 1]], want, tol, f"row {b}")


@pytest.mark.parametrize("dtype,T,D,log2", [(torch.bfloat16, 1, 64, 29), (torch.float32, 1, 32, 28),
                                            (torch.bfloat16, 40, 128, 26), (torch.float32, 40, 32, 25)])
@pytest.mark.parametrize("where", [0, 0.5, 1])
def test_one_key_among_hundreds_of_millions(dtype, T, D, log2, where):
    """A row of up to half a billion positions on pages that repeat: the one key that is like the queries, at
    the row's start, in its middle or the last that the first query sees, gives its value."""
    n, page, pool = 1 << log2, 16, 96
    g = torch.Generator().manual_seed(7)
    k = torch.zeros(pool, page, 1, D, dtype=dtype, device=DEV)
    v = torch.randn(pool, page, 1, D, generator=g).to(dtype).to(DEV)
    table = (torch.arange(n // page + 4, device=DEV) % (pool - 1)).int()[None]
    at = int(where * (n - 1))
    table[0, at // page] = pool - 1  # a page of its own, but for the row's end
    like = torch.ones(D, dtype=dtype)
    k[pool - 1, at % page, 0] = like.to(DEV)
    q = (like * (200 / D ** 0.5)).expand(1, T, 2, D).to(DEV)  # 200 more than the other keys' scores
    y = flash_attn.flash_attn_paged_with_kvcache(
        q, k, v, block_table=table, cache_seqlens=torch.tensor([n - 1], dtype=torch.int32, device=DEV), causal=True)
    # The others weigh at most 2^30 exp(-199).
    want = v[pool - 1, at % page, 0].double().cpu().expand(1, T, 2, D)
    close(y, want, torch.finfo(dtype).eps * want.abs() + 2.0 ** -24)


@pytest.mark.parametrize("dtype,H,H_kv,D", [(torch.bfloat16, 200, 200, 64), (torch.bfloat16, 600, 300, 16),
                                            (torch.float32, 200, 200, 32), (torch.bfloat16, 130, 130, 128)])
def test_hundreds_of_kv_heads(dtype, H, H_kv, D):
    """More KV heads than the workgroups a call aims at have to share."""
    rows = [(1, 700), (40, 100), (1, 0), (3, 300)]
    g = torch.Generator().manual_seed(8)
    pool = Pool([p + t for t, p in rows], 16, H_kv, D, dtype, stale=0.0)
    cu = [0, 1, 41, 42, 45]
    q = torch.randn(45, H, D, generator=g).to(dtype)
    y = flash_attn.flash_attn_paged_with_kvcache(
        q.to(DEV), pool.k.to(DEV), pool.v.to(DEV), block_table=pool.table.to(DEV),
        cache_seqlens=torch.tensor([p for _, p in rows], dtype=torch.int32, device=DEV),
        cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV), max_seqlen=40, causal=True)
    for b, (t, p) in enumerate(rows):
        want, tol = attend(q[cu[b]:cu[b + 1]], *pool.rows(b, p + t), p)
        close(y[cu[b]:cu[b + 1]], want, tol, f"row {b}")
