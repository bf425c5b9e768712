"""Strides at the ends of 64 bits at the C entry of what a paged cache keeps of drafted trees: refused on the host.
Nothing here is launched."""
import pytest

from modelcore_amd import _ext

FAKE = 1 << 20  # never dereferenced: the checks fail first
TOP = (1 << 63) - 16


def keep(slots, slot_stride, n_pages, page_stride, n_rows=2):
    return _ext.lib().mcamd_paged_keep(FAKE, FAKE, slots, slot_stride, FAKE, 8, FAKE, FAKE, FAKE, 4, FAKE, FAKE, FAKE, n_rows, 8,
                                       n_pages, 16, page_stride, 256, _ext.BF16, None)


@pytest.mark.parametrize("n_pages,page_stride,slot_stride", [
    (20, 1 << 62, 20 * 16 * 256), (20, 1 << 62, TOP), (3, 1 << 62, TOP), (5, 1 << 62, 16 * 256), (20, TOP, TOP), ((1 << 27) - 1, 1 << 37, 1 << 40),
    (2, 16 * 256, 2 * 16 * 256 - 16), (2, 1 << 20, (1 << 20) + 16 * 256 - 16)])
def test_slots_that_a_pools_pages_do_not_fit(n_pages, page_stride, slot_stride):
    assert keep(2, slot_stride, n_pages, page_stride) == _ext.EINVAL
    assert b"slot_stride" in _ext.lib().mcamd_last_error()


@pytest.mark.parametrize("n_pages,page_stride,slot_stride", [
    (2, 16 * 256, 2 * 16 * 256), (2, 1 << 20, (1 << 20) + 16 * 256), (1, TOP, 16 * 256), (20, 1 << 40, 20 << 40)])
def test_slots_that_they_fit(n_pages, page_stride, slot_stride):
    assert keep(2, slot_stride, n_pages, page_stride, n_rows=0) == _ext.OK
