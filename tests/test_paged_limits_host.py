"""Sizes at the ends of 64 bits at the paged operators' C entry points: refused on the host, or taken for
what they say. Nothing here is launched."""
import pytest

from modelcore_amd import _ext
from test_paged_host import FAKE, attention

TOP = (1 << 63) - 1


@pytest.mark.parametrize("page", [1 << 31, 1 << 62, (1 << 62) + 1, TOP, -16, -(1 << 63)])
def test_page_sizes_end_the_search_for_their_power(page):
    lib = _ext.lib()
    assert attention(page=page, page_stride=TOP) == _ext.EINVAL and b"power of two" in lib.mcamd_last_error()
    assert lib.mcamd_paged_reserve(FAKE, 8, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 8, 20, page,
                                   5, None) == _ext.EINVAL
    assert lib.mcamd_paged_release(FAKE, 8, FAKE, FAKE, 1, 2, FAKE, FAKE, 8, 20, page, None) == _ext.EINVAL
    assert lib.mcamd_qk_rope_norm_append_paged(
        FAKE, 1024, FAKE, 256, FAKE, 256, FAKE, FAKE, 64, FAKE, FAKE, FAKE, FAKE, FAKE, 3, 8, 2, 128, 4, page, TOP,
        1e-6, 1.2, _ext.BF16, None) == _ext.EINVAL
    assert lib.mcamd_paged_scratch_bytes(2, 7, 5, 8, 2, 128, 8, page, -1, _ext.BF16) == 0


@pytest.mark.parametrize("kw", [
    dict(n_pages=1 << 60), dict(n_pages=TOP), dict(max_pages=TOP, table_stride=TOP),
    dict(n_pages=1 << 59, page=32), dict(H=1 << 40, H_kv=1 << 40, page_stride=TOP),
    dict(D=1 << 60, page_stride=TOP), dict(cu=None, n_rows=2, longest=(1 << 63) - 2, total=-4),
    dict(cu=None, n_rows=1 << 15, longest=1 << 49, total=0), dict(total=TOP, H=1, H_kv=1)])
def test_products_that_leave_64_bits_are_refused(kw):
    assert attention(**kw) in (_ext.EINVAL, _ext.EUNSUPPORTED), kw


@pytest.mark.parametrize("n_pages,page", [(1 << 60, 16), (1 << 62, 64), (TOP, 1 << 30)])
def test_pools_that_leave_64_bits_are_refused(n_pages, page):
    lib = _ext.lib()
    assert lib.mcamd_paged_reserve(FAKE, 8, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 8, n_pages, page,
                                   5, None) == _ext.EUNSUPPORTED
    assert lib.mcamd_paged_release(FAKE, 8, FAKE, FAKE, 1, 2, FAKE, FAKE, 8, n_pages, page, None) == _ext.EUNSUPPORTED
    assert lib.mcamd_qk_rope_norm_append_paged(
        FAKE, 1024, FAKE, 256, FAKE, 256, FAKE, FAKE, 64, FAKE, FAKE, FAKE, FAKE, FAKE, 3, 8, 2, 128, n_pages, page,
        TOP, 1e-6, 1.2, _ext.BF16, None) == _ext.EUNSUPPORTED


@pytest.mark.parametrize("total,H,H_kv,q_tok", [(0x7fffffff, 1 << 29, 1, TOP), (0x7fffffff, 1, 1 << 28, TOP),
                                                (5, 1 << 62, 1 << 61, TOP), (1 << 20, 2000, 50, 2000 * 128)])
def test_steps_of_more_heads_than_a_grid_are_refused(total, H, H_kv, q_tok):
    assert _ext.lib().mcamd_qk_rope_norm_append_paged(
        FAKE, q_tok, FAKE, TOP, FAKE, TOP, FAKE, FAKE, 64, FAKE, FAKE, FAKE, FAKE, FAKE, total, H, H_kv, 128, 4, 16,
        TOP, 1e-6, 1.2, _ext.BF16, None) == _ext.EUNSUPPORTED


@pytest.mark.parametrize("dtype", [_ext.BF16, _ext.F32])
@pytest.mark.parametrize("D", [64, 128])
def test_a_bound_on_rows_past_their_tokens_is_one_by_them(dtype, D):
    """max_seqlen says "at most": past a call's tokens it changes nothing, past 31 bits too."""
    def scratch(longest, total=20):
        return _ext.lib().mcamd_paged_scratch_bytes(3, total, longest, 8, 8, D, 4000, 16, -1, dtype)
    want = scratch(20)
    assert want > 0
    for longest in (21, 1000, (1 << 31) - 1, 1 << 31, (1 << 32) + 1, TOP):
        assert scratch(longest) == want, longest
    assert attention(longest=TOP, total=0) == _ext.OK


def test_page_sizes_end_in_python_too():
    from modelcore_amd.kernels.paged import check_page_size
    assert check_page_size(1 << 30) == 1 << 30
    for n in (1 << 31, 1 << 62):
        with pytest.raises(ValueError, match="power of two"):
            check_page_size(n)
