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


@pytest.mark.parametrize("rows, cols, k", [(300, 500, 4000), (64, 64, 20000), (1000, 1000, 1000)])
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_a_workspace_fits_its_call_whoever_sets_switches_between(rows, cols, k, kind):
    """The question for a workspace and the call plan by their arguments alone, of which the switches are one."""
    lib = N.lib()

    def sizes(kind):
        dense = (ctypes.c_int64 * 3)()
        lib.dl_dense_forward_sizes(16, k, 0, 16, rows, k, cols, 0, kind, dense)
        return (list(dense), lib.dl_dense_backward_workspace_bytes(16, 0, 1, 16, k, 0, 16, 1, 1, rows, k, cols, kind),
                lib.dl_orthogonalize_workspace_bytes(2, rows, cols, kind))

    def muon():
        return lib.dl_muon_workspace_bytes((ctypes.c_int64 * 5)(16, 16, 16, rows, cols), 1)

    assert lib.dl_matmul_choice() == 0
    plain, plain_muon, seen = sizes(kind), muon(), set()
    for columns in (64, 128, 256, 0):
        for splits in (1, 7, 64, 0):
            with N.tuning(N.TUNE_MATMUL_COLUMNS, columns), N.tuning(N.TUNE_MATMUL_SPLITS, splits):
                assert sizes(kind) == plain and muon() == plain_muon
                choice = lib.dl_matmul_choice()
                asked = sizes(kind | choice)
            assert (choice == 0) == (columns == splits == 0) and sizes(kind | choice) == asked
            seen.add(str(asked))
    assert len(seen) > 1      # the switches do what they say


@pytest.mark.parametrize("columns, splits", [(100, 0), (1, 1), (1023, 4095), (-1, -1), (0, -5), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_switches_that_say_nothing(columns, splits):
    lib = N.lib()
    with N.tuning(N.TUNE_MATMUL_COLUMNS, columns), N.tuning(N.TUNE_MATMUL_SPLITS, splits):
        kind = lib.dl_matmul_choice()
        dense = (ctypes.c_int64 * 3)()
        lib.dl_dense_forward_sizes(16, 500, 0, 16, 100, 500, 70, 0, kind, dense)
        assert 0 <= dense[2] <= 64 << 20 and lib.dl_orthogonalize_workspace_bytes(1, 100, 70, kind) > 0
