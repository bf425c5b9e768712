"""The paged attention's C entry with bounds that no tensor has, as its header allows them."""
import pytest
import torch

from _paged import Pool
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
