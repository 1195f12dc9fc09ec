"""Entry points of dense layers as a binding calls them: sizes and refusals, which come back before anything is launched."""
import ctypes

import pytest

from difflogic_b200 import _native as N


@pytest.mark.parametrize("rows, cols", [(40, 1), (40, 7), (100, 784), (1001, 783)])
def test_planes_laid_out_apart_are_the_forward_passs(rows, cols):
    lib, sizes = N.lib(), (ctypes.c_int64 * 3)()
    lib.dl_dense_forward_sizes(16, cols, 0, 16, rows, cols, 56, 0, 0, sizes)
    assert (lib.dl_dense_planes_bytes(rows, cols, 0), lib.dl_dense_planes_bytes(56, cols, 0)) == (sizes[0], sizes[1])
    lib.dl_dense_forward_sizes(16, rows, 1, 16, rows, cols, 56, 0, 0, sizes)
    assert lib.dl_dense_planes_bytes(cols, rows, 0) == sizes[0]
    assert lib.dl_dense_planes_bytes(0, 4, 0) == lib.dl_dense_planes_bytes(4, 0, 0) == 0


def test_laying_out_refuses():
    lib, bad = N.lib(), N.DL_ERR_INVALID_ARG
    for args in ((None, 4, 4, 4, 0, 16), (16, 4, 4, 4, 0, None), (16, 4, 4, 4, 0, 8), (16, 4, 4, 3, 0, 16), (16, 0, 4, 4, 0, 16), (16, 4, 0, 4, 0, 16),
                 (16, 4, 4, 4, 3, 16)):
        assert lib.dl_dense_lay_out(*args, None) == bad
