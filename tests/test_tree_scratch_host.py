"""Which calls over drafted trees have scratch to cut their keys with, on the host."""
import pytest

from modelcore_amd import _ext


@pytest.mark.parametrize("dtype", [_ext.BF16, _ext.F32])
@pytest.mark.parametrize("window", [0, 10, 100, 191])
def test_wide_trees_behind_narrow_windows(window, dtype):
    """A block's keys are the window's and its row's nodes: a thousand of those are worth ranges, however narrow the
    window; a few are not."""
    of = lambda T: _ext.lib().mcamd_paged_tree_scratch_bytes(2, 2 * T, T, 8, 2, 64, 4096, 16, window, dtype)  # noqa: E731
    assert of(1024) > 0
    assert of(40) == 0 or dtype == _ext.F32
