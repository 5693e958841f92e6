"""MXFP4 products without a GPU: sizes at the ends of what the C entry points take."""
import pytest

from mslk_amd import _lib

SOMEWHERE = 1 << 20   # a pointer that is not followed
L = _lib.lib()


@pytest.mark.parametrize("groups", [(1 << 30) + 1, (1 << 31) - 64, (1 << 31) - 1])
def test_more_groups_than_a_loop_over_them_can_count_are_refused(groups):
    """Kernels take 64 groups at a time: the number behind the last 64 has to be an int, too."""
    assert L.mslk_amd_mxfp4_grouped_mm(*[SOMEWHERE] * 5, groups, 0, SOMEWHERE, 0, 100, 1, 512, SOMEWHERE, 1 << 62, None) != 0
    assert "2^30 groups" in L.mslk_amd_last_error().decode()
