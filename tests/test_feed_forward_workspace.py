"""Workspaces of the feed-forward operators, laid out without a GPU."""

import ctypes

import pytest


@pytest.mark.parametrize("m", [1, 31, 32, 33, 1000, 65536, 10 ** 6])
@pytest.mark.parametrize("n", [1, 255, 256, 257, 7168, 200_000])
def test_slabs_are_the_kernels(m, n):
    """The bias gradient's partial sums: as many slabs as the C side asks for, each inside the workspace."""
    from dsv4_b200 import _native as N
    from dsv4_b200 import feed_forward as F
    count = ctypes.c_int64(0)
    N.call("dsv4_b200_act_backward_slabs", m, n, ctypes.byref(count))
    slabs, (size, (dz, partial, restored)) = F._dense_workspace(m, n, 40, True, True, True)
    assert slabs == count.value >= 1
    assert dz == 0 and partial >= m * n * 2 and restored >= partial + slabs * n * 4
    assert 2 * size >= restored + m * 40 * 2
    assert F._dense_workspace(m, n, 40, False, False, False) == (0, (0, (None, None, None)))
